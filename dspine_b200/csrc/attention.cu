// attention.cu -- attention of drafted tokens over a slot-addressed, paged KV cache (sm_100a).
//
// Request b has t_b drafted tokens (rows of q) and lens[b] cached ones, the drafted among them as
// its last t_b: drafted token j is cached at position p0 + j, p0 = lens[b] - t_b.  Its row i sees
// the keys before p0 and the drafted tokens j that bit j of mask[i] names (without a mask: a
// chain, j <= i):
//     out = sum_j softmax_j(scale q . k_j) v_j,   lse = log sum_j exp(scale q . k_j).
// A row that sees nothing gets zeros and -inf.  Position p lives in slot
// table[b][p / page_size] * page_size + p % page_size; a page outside the cache makes its
// positions unseen and sets bit 1 of the error word.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dsv_common.cuh"
#include "dsv_kernels.h"

namespace dsv {
namespace attn {

constexpr int kThreads = 128;
constexpr int kMaxDim = 128;

__device__ __forceinline__ float elem(const void* p, long long i, int dtype) {
    if (dtype == kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[i]);
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(p)[i], __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
}

__device__ __forceinline__ void rows_of(const TreeAttnArgs& a, int b, long long& lo, long long& hi) {
    if (a.indptr) {
        lo = a.indptr[b];
        hi = a.indptr[b + 1];
        lo = lo < 0 ? 0 : (lo > a.rows ? a.rows : lo);
        hi = hi < lo ? lo : (hi > a.rows ? a.rows : hi);
    } else {
        lo = (long long)b * a.width;
        hi = lo + a.width;
    }
}

// one block per (query head, request); its rows one after the other, 128 keys at a time
__global__ void __launch_bounds__(kThreads) rows_kernel(TreeAttnArgs a, int dtype) {
    __shared__ float q[kMaxDim], p[kThreads], red[kThreads / 32];
    __shared__ long long at[kThreads];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int hq = blockIdx.x, b = blockIdx.y, h = hq / a.group, dim = a.c.dim;
    const bool scaled = a.c.dtype == kE4m3;
    long long lo, hi;
    rows_of(a, b, lo, hi);
    const long long cap = (long long)a.max_pages * a.page_size;
    long long len = a.lens[b] < 0 ? 0 : a.lens[b];
    if (len > cap) {
        len = cap;
        if (tid == 0 && a.err) atomicOr(a.err, 2u);
    }
    const long long p0 = len - (hi - lo), pages = a.c.slots / a.page_size;
    for (long long r = lo; r < hi; ++r) {
        const int i = (int)(r - lo);
        __syncthreads();
        if (tid < dim) q[tid] = elem(a.q, r * a.q_token_stride + hq * a.q_head_stride + tid, dtype);
        const uint64_t bits = a.mask ? (uint64_t)a.mask[r] : 0;
        float m = -INFINITY, l = 0.f, o = 0.f;
        for (long long base = 0; base < len; base += kThreads) {
            __syncthreads();
            const long long pos = base + tid, j = pos - p0;
            long long slot = -1;
            if (pos < len && (j < 0 || (a.mask ? (j < 64 && ((bits >> j) & 1)) : j <= i))) {
                const long long page = a.table[b * a.table_stride + pos / a.page_size];
                if (page >= 0 && page < pages)
                    slot = page * a.page_size + pos % a.page_size;
                else if (a.err)
                    atomicOr(a.err, 2u);
            }
            float s = -INFINITY;
            if (slot >= 0) {
                s = 0.f;
                const long long k = slot * a.c.slot_stride + h * a.c.head_stride;
                for (int d = 0; d < dim; ++d) s = fmaf(q[d], elem(a.c.k, k + d, a.c.dtype), s);
                s *= a.scale * (scaled ? a.c.k_scale[slot * a.c.scale_stride + h] : 1.0f);
            }
            float t = s;
            for (int k = 16; k > 0; k >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, k));
            if (lane == 0) red[wid] = t;
            __syncthreads();
            const float mn = fmaxf(fmaxf(m, fmaxf(red[0], red[1])), fmaxf(red[2], red[3]));
            const float ref = mn == -INFINITY ? 0.f : mn;
            at[tid] = slot;
            p[tid] = slot >= 0 ? expf(s - ref) : 0.f;
            __syncthreads();
            const float f = expf(m - ref);
            l *= f;
            o *= f;
            for (int k = 0; k < kThreads; ++k) {
                const long long sk = at[k];
                if (sk < 0) continue;
                l += p[k];
                if (tid < dim)
                    o = fmaf(p[k] * (scaled ? a.c.v_scale[sk * a.c.scale_stride + h] : 1.0f),
                             elem(a.c.v, sk * a.c.slot_stride + h * a.c.head_stride + tid, a.c.dtype), o);
            }
            m = mn;
        }
        if (tid < dim) {
            const float x = l == 0.f ? 0.f : o / l;
            const long long w = r * a.out_token_stride + hq * a.out_head_stride + tid;
            if (dtype == kBf16)
                static_cast<__nv_bfloat16*>(a.out)[w] = __float2bfloat16_rn(x);
            else
                static_cast<__half*>(a.out)[w] = __float2half_rn(x);
        }
        if (tid == 0 && a.lse) a.lse[r * a.q_heads + hq] = l == 0.f ? -INFINITY : m + logf(l);
    }
}

}  // namespace attn

size_t tree_attn_workspace_bytes(int, int, int, int) { return 0; }

int launch_tree_attn(const TreeAttnArgs& a, int dtype, cudaStream_t st) {
    attn::rows_kernel<<<dim3(a.q_heads, a.batch), attn::kThreads, 0, st>>>(a, dtype);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace dsv
