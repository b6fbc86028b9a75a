// kvcache.cu -- rows written into and read back from a slot-addressed KV cache (sm_100a).
//
// A cache holds, for every slot and KV head, one K row and one V row of `dim` elements: bf16 or
// fp16 as given, or e4m3 codes with one fp32 scale per (slot, head).  The scale rule is the one of
// the FP8 retrieval head's rows (layers/fp8/coarse.py:41-55 _scale, _quantize; fp8.cu
// quantize_kernel): s = amax|x| / 448 (1 for an all-zero row and for a row with a NaN), code =
// e4m3(x / s), IEEE division, round to nearest even.
//
//   write_kernel  one group of lanes per (token, head) row, 16 elements per lane
//   read_kernel   the inverse: code * s in fp32, rounded once to the output type
//
// A row is read once and written once.  A lane holds 16 elements because 16 codes are one 16-byte
// access of the cache: the widest there is, and rows of 128 elements then need 8 lanes, so a warp
// moves 4 rows at a time.  Measured with 8 heads of 128, e4m3, bf16 rows: 131072 tokens read in
// 145 us (5.6 TB/s, bound by memory); 32749 written in 51.4 us (4.0 TB/s, bound by issue: 318
// instructions for the 16 elements of a lane, schedulers 70% busy.  The next row's loads ahead of this
// one's arithmetic took the same time; arithmetic on pairs took fewer instructions but more
// registers, 53 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dsv_common.cuh"
#include "dsv_kernels.h"

namespace dsv {
namespace kvc {

constexpr int kThreads = 256;

struct V16 {
    float x[16];
};

template <typename A, typename B> struct same { static constexpr bool value = false; };
template <typename A> struct same<A, A> { static constexpr bool value = true; };

__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, __nv_bfloat16) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 consecutive elements as they lie in memory
template <typename T>
struct Raw {
    static constexpr int kVecs = (int)sizeof(T);  // 16 elements = sizeof(T) vectors of 16 bytes
    uint4 w[kVecs];
};

template <typename T>
__device__ __forceinline__ Raw<T> load16(const T* p) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < Raw<T>::kVecs; ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return r;
}

template <typename T>
__device__ __forceinline__ void store16(T* p, const Raw<T>& r) {
#pragma unroll
    for (int i = 0; i < Raw<T>::kVecs; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

template <typename T>
__device__ __forceinline__ V16 unpack16(const Raw<T>& r) {
    V16 v;
#pragma unroll
    for (int i = 0; i < Raw<T>::kVecs; ++i) {
        const uint32_t w[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4)
                v.x[4 * i + j] = __uint_as_float(w[j]);
            else
                unpack2(w[j], v.x[8 * i + 2 * j], v.x[8 * i + 2 * j + 1], T());
        }
    }
    return v;
}

template <typename T>
__device__ __forceinline__ Raw<T> pack16(const V16& v) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < Raw<T>::kVecs; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4)
                w[j] = __float_as_uint(v.x[4 * i + j]);
            else
                w[j] = pack2(v.x[8 * i + 2 * j], v.x[8 * i + 2 * j + 1], T());
        }
        r.w[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}

__device__ __forceinline__ V16 decode16(const uint4& c, float s) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    V16 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint16_t two = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        v.x[2 * i] = __fmul_rn(f.x, s);
        v.x[2 * i + 1] = __fmul_rn(f.y, s);
    }
    return v;
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
}

// The codes of x / s, IEEE quotients rounded to e4m3.  In a row of finite values a quotient takes a
// product with r = 1 / s and two corrections by its exact residual (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990: with r rounded correctly, the
// first leaves a quotient off by less than a step, the second rounds that one correctly; fp32 rows need
// both, for bf16 ones the first is correct already, over all pairs of mantissas).  s
// within 2^-60 and 2^100 keeps r normal and the residuals of all quotients from 2^-42 on exact (they
// are multiples of 2^-47 s y); smaller ones are far below half of the smallest code, 2^-10.  The residual is taken as q s - x, so that -0
// stays -0.
__device__ __forceinline__ void encode(const V16& v, float s, bool finite, uint32_t (&w)[4]) {
    float y[16];
    if (finite && s > 8.6737e-19f && s < 1.2676e30f) {
        const float r = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            y[i] = __fmul_rn(v.x[i], r);
            y[i] = __fmaf_rn(-__fmaf_rn(y[i], s, -v.x[i]), r, y[i]);
            y[i] = __fmaf_rn(-__fmaf_rn(y[i], s, -v.x[i]), r, y[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = __fdiv_rn(v.x[i], s);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = codes4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
}

__device__ __forceinline__ long long slot_at(const void* slots, int is64, long long n) {
    return is64 ? __ldg(static_cast<const long long*>(slots) + n)
                : (long long)__ldg(static_cast<const int*>(slots) + n);
}

// TIN: type of the rows; kQuant: the cache holds e4m3 codes, else TIN
template <typename TIN, bool kQuant>
__global__ void __launch_bounds__(kThreads) write_kernel(KvRowsArgs a) {
    const int lanes = a.lanes;                      // lanes of a row's group (a power of two)
    const int sub = threadIdx.x & (lanes - 1);
    const int e0 = sub * 16;
    const bool live = e0 < a.c.dim;
    const uint32_t per_block = kThreads / lanes;
    const uint32_t rows = (uint32_t)(a.tokens * a.c.heads);
    const bool is_v = blockIdx.y != 0;
    const TIN* x = static_cast<const TIN*>(is_v ? a.v : a.k);
    const long long ts = is_v ? a.v_token_stride : a.k_token_stride;
    const long long hs = is_v ? a.v_head_stride : a.k_head_stride;
    for (uint32_t base = blockIdx.x * per_block; base < rows; base += gridDim.x * per_block) {
        const uint32_t r = base + threadIdx.x / lanes;
        const bool in = r < rows;
        const uint32_t n = in ? r / a.c.heads : 0, h = in ? r - n * a.c.heads : 0;
        const long long slot = in ? slot_at(a.slots, a.slots64, n) : -1;
        const bool ok = slot >= 0 && slot < a.c.slots;
        if (in && slot >= a.c.slots && sub == 0 && a.err) atomicOr(a.err, 1u);
        Raw<TIN> raw = {};
        if (ok && live) raw = load16(x + n * ts + h * hs + e0);
        const long long at = slot * a.c.slot_stride + h * a.c.head_stride + e0;
        if constexpr (kQuant) {
            const V16 v = unpack16(raw);
            float m = 0.f;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float t = fabsf(v.x[i]);
                nan |= t != t;
                m = fmaxf(m, t);
            }
            // a NaN in the row: its maximum counts as NaN, which is not > 0, so the scale is 1
            if (nan) m = __int_as_float(0x7fffffff);
            uint32_t mb = __float_as_uint(m);  // ordered as the values are, NaN above all
            for (int o = lanes >> 1; o > 0; o >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
            const float amax = __uint_as_float(mb);
            const float s = amax > 0.f ? __fdiv_rn(amax, 448.0f) : 1.0f;
            if (ok && live) {
                uint32_t w[4];
                encode(v, s, amax < INFINITY, w);
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + at) =
                    make_uint4(w[0], w[1], w[2], w[3]);
                if (sub == 0) (is_v ? a.c.v_scale : a.c.k_scale)[slot * a.c.scale_stride + h] = s;
            }
        } else if (ok && live) {
            store16(static_cast<TIN*>(is_v ? a.c.v : a.c.k) + at, raw);  // bits as they are
        }
    }
}

// TC: type of the cache (uint8_t: e4m3 codes with scales); TOUT: type of the rows
template <typename TC, typename TOUT>
__global__ void __launch_bounds__(kThreads) read_kernel(KvRowsArgs a) {
    const int lanes = a.lanes;
    const int sub = threadIdx.x & (lanes - 1);
    const int e0 = sub * 16;
    const bool live = e0 < a.c.dim;
    const uint32_t per_block = kThreads / lanes;
    const uint32_t rows = (uint32_t)(a.tokens * a.c.heads);
    const bool is_v = blockIdx.y != 0;
    const TC* src = static_cast<const TC*>(is_v ? a.c.v : a.c.k);
    const float* scale = is_v ? a.c.v_scale : a.c.k_scale;
    TOUT* out = static_cast<TOUT*>(const_cast<void*>(is_v ? a.v : a.k));
    for (uint32_t base = blockIdx.x * per_block; base < rows; base += gridDim.x * per_block) {
        const uint32_t r = base + threadIdx.x / lanes;
        if (r >= rows || !live) continue;
        const uint32_t n = r / a.c.heads, h = r - n * a.c.heads;
        const long long slot = slot_at(a.slots, a.slots64, n);
        const bool ok = slot >= 0 && slot < a.c.slots;
        if (slot >= a.c.slots && sub == 0 && a.err) atomicOr(a.err, 1u);
        Raw<TOUT> v = {};
        if (ok) {
            const Raw<TC> raw = load16(src + slot * a.c.slot_stride + h * a.c.head_stride + e0);
            if constexpr (sizeof(TC) == 1)
                v = pack16<TOUT>(decode16(raw.w[0], __ldg(scale + slot * a.c.scale_stride + h)));
            else if constexpr (same<TC, TOUT>::value)
                v = raw;  // bits as they are
            else
                v = pack16<TOUT>(unpack16(raw));
        }
        store16(out + (long long)r * a.c.dim + e0, v);
    }
}

int lanes_for(int dim) {
    int l = 1;
    while (l * 16 < dim) l *= 2;
    return l;
}

dim3 grid_for(long long rows, int lanes) {
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const long long per_block = kThreads / lanes, blocks = (rows + per_block - 1) / per_block;
    const long long cap = (long long)sms * 8;
    return dim3((unsigned)(blocks < cap ? blocks : cap), 2);
}

}  // namespace kvc

int launch_kv_write(KvRowsArgs a, int dtype, cudaStream_t st) {
    a.lanes = kvc::lanes_for(a.c.dim);
    const dim3 grid = kvc::grid_for(a.tokens * a.c.heads, a.lanes);
    const bool quant = a.c.dtype == kE4m3;
    if (dtype == kBf16 && quant)
        kvc::write_kernel<__nv_bfloat16, true><<<grid, kvc::kThreads, 0, st>>>(a);
    else if (dtype == kF16 && quant)
        kvc::write_kernel<__half, true><<<grid, kvc::kThreads, 0, st>>>(a);
    else if (dtype == kF32 && quant)
        kvc::write_kernel<float, true><<<grid, kvc::kThreads, 0, st>>>(a);
    else if (dtype == kBf16 && a.c.dtype == kBf16)
        kvc::write_kernel<__nv_bfloat16, false><<<grid, kvc::kThreads, 0, st>>>(a);
    else if (dtype == kF16 && a.c.dtype == kF16)
        kvc::write_kernel<__half, false><<<grid, kvc::kThreads, 0, st>>>(a);
    else
        return kBadDtype;
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

int launch_kv_read(KvRowsArgs a, int dtype, cudaStream_t st) {
    a.lanes = kvc::lanes_for(a.c.dim);
    const dim3 grid = kvc::grid_for(a.tokens * a.c.heads, a.lanes);
    const int key = a.c.dtype * 4 + dtype;
    switch (key) {
        case kBf16 * 4 + kBf16: kvc::read_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kBf16 * 4 + kF16: kvc::read_kernel<__nv_bfloat16, __half><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kBf16 * 4 + kF32: kvc::read_kernel<__nv_bfloat16, float><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kF16 * 4 + kBf16: kvc::read_kernel<__half, __nv_bfloat16><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kF16 * 4 + kF16: kvc::read_kernel<__half, __half><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kF16 * 4 + kF32: kvc::read_kernel<__half, float><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kE4m3 * 4 + kBf16: kvc::read_kernel<uint8_t, __nv_bfloat16><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kE4m3 * 4 + kF16: kvc::read_kernel<uint8_t, __half><<<grid, kvc::kThreads, 0, st>>>(a); break;
        case kE4m3 * 4 + kF32: kvc::read_kernel<uint8_t, float><<<grid, kvc::kThreads, 0, st>>>(a); break;
        default: return kBadDtype;
    }
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace dsv
