// attention.cu -- attention of drafted tokens over a slot-addressed, paged KV cache (sm_100a:
// tcgen05 + TMEM).
//
// Request b has t_b drafted tokens (rows of q) and lens[b] cached ones, the drafted among them as
// its last t_b: drafted token j is cached at position p0 + j, p0 = lens[b] - t_b.  Its row i sees
// the keys before p0 and the drafted tokens j that bit j of mask[i] names (without a mask: a
// chain, j <= i):
//     out = sum_j softmax_j(scale q . k_j) v_j,   lse = log sum_j exp(scale q . k_j).
// A row that sees nothing gets zeros and -inf.  Position p lives in slot
// table[b][p / page_size] * page_size + p % page_size; a page outside the cache makes its
// positions unseen and sets bit 1 of the error word.
//
//   attn_kernel     persistent, one CTA per SM.  The rows of one (request, KV head), t_b tokens x
//                   `group` query heads, are the M = 128 rows of the matrix instructions, so a key
//                   is read once for all of them.  The tiles of 64 keys of all (request, KV head,
//                   row block) items form one line that is cut into equal pieces, one per CTA:
//                   every SM streams the same number of tiles however ragged the lengths are.
//                     warps 0-7    two softmax warpgroups, one TMEM lane (row) per thread, its
//                                  scores of a tile in registers
//                     warps 8, 9   MMA issuers: scores (and TMEM allocation), accumulation
//                     warp 10      index: slots, scales and validity of the tiles to come
//                     warp 11      queries: the next segment's rows of q, while this one runs
//                     warps 12-15  loaders, two for K and two for V: rows of a tile, slot by slot,
//                                  into a ring each of 128-byte-swizzled shared-memory stages (e4m3:
//                                  converted on the way)
//                   S = Q K^T (kind::f16, both operands in shared memory) and O += P V (P from
//                   TMEM, written over S; V as a matrix with rows of keys, "MN-major").
//                   Two streams keep the tensor core and the exponentials busy at once: with more
//                   than 128 rows each warpgroup owns 128 of them and both use every tile, else
//                   both own the same rows and take every other tile, with an accumulator each,
//                   joined at the end.  Each stream has two score buffers, so the scores of its
//                   next tile are computed while it works on one: with tiles of 128 keys and one
//                   buffer the chain scores -> weights -> accumulate -> scores set the pace.
//   combine_kernel  joins the partial results of items that a cut went through.
//
// Softmax: weights are 2^(s c - ref), c = scale log2(e), ref a running reference that follows the
// row's maximum but moves only when the maximum has outgrown it by more than 2^8 (fp16: 2^5): the
// accumulator is then rescaled (a TMEM round trip), else left alone.  Any reference gives the same
// quotient; fp16's lies 2^9 below the maximum, so that a row's largest weight lies in [2^9, 2^14] and
// a weight below 2^-23 of it, which fp16 holds with fewer bits, is off by at most 2^-34 of it.  Sums
// and the accumulator are fp32; the weights are rounded once to the operand type.
//
// e4m3 caches: codes are exact in fp16, so they are converted between two rings in shared memory
// and the matrix instructions run on fp16.  q goes to fp16 with a power of two per row.  K
// scales multiply the scores; V scales multiply the weights.  The products are what is rounded to
// fp16, so the reference follows the row's largest product: the maximum, over the keys that the row
// sees, of s c + e, 2^e the first power of two above the key's V scale.  Where the V scales of a tile
// lie within 2^kNear of each other and of the last tile's (nearly always; two ballots), one e serves for
// all its keys, at most kNear too large, so that the row's largest product lies in [4, 2^14]: products
// keep fp16's full precision down to 2^-16 of it and are off by at most 2^-27 of it below.  Other
// tiles take an e a key, in a function of its own (far_unit).  e is held within [-90, 120], so that
// sums of the weights themselves stay within fp32.
//
// A near tile costs what one e for the whole context did (64 x 16 247 us from 245, 1 x 16 long 87 from 84; an e a
// key for every tile: 277 and 93).  The rare forms are calls: code beside the loop slowed it whether it
// ran or not.  With V scales that spread over 2^8 in every tile: 338 and 151 us; over 2^3: as without.
//
// Masked positions: scores of unseen keys are replaced by -inf, rows of unreadable positions are
// zeros in shared memory.  A V element of a drafted token that is not finite would reach rows that
// do not see it through 0 x inf; tiles with drafted tokens are scanned, such elements zeroed and
// added back to the rows that do see them.
//
// Measured (32 query heads over 8 KV heads of 128 unless said; ragged lengths; caches larger than L2, three sets of
// inputs in turn).  Cycles are from a build that reads the clock, which is up to a third slower in all:
//   64 requests x 1 token, up to 8192 cached, bf16, pages of 16     245 us, 4.9 TB/s: the cache's bytes
//       (copy bandwidth would take 186), less what segment switches cost (a tenth)
//   16 requests x trees of up to 64, 64 query heads, up to 16384    368 us, 0.62 PFLOP/s: the latency of a unit, whose
//       phases (scores from TMEM, maximum, exponentials, weights to TMEM) follow one another with two softmax warps a
//       scheduler: 1390 cycles of work and 630 of waiting for scores for 64 keys; no pipe is above 40%
//   64 requests x 16 tokens, up to 4096 cached, e4m3, pages of 1    247 us: softmax warps work 3900 cycles on a unit
//       and wait 600 for its scores, loaders convert 1800 a tile and wait 3200 for a free stage (two tiles a ring): the
//       chain of conversion, scores, weights and accumulation through short rings; a switch of segments takes 9400
//   1 request x 16 tokens, 131071 cached, 4 KV heads, e4m3          86 us: work 2400 a unit and 600 of waiting,
//       conversion 1950 a tile and 500 of waiting: both sides nearly always at work, each by its own latency
//   1 request x 1 token, 333 cached                                 24 us a call from Python, the host's time (16 us
//       in attn_kernel when all caches are cold: the chain of waits from the plan to the join)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "dsv_common.cuh"
#include "dsv_kernels.h"

namespace dsv {
namespace attn {

constexpr int kRows = 128;                 // rows of a Q tile (MMA M)
constexpr int kTile = 64;                  // keys of a tile
constexpr int kQBlock = kRows * 128;       // bytes of a [128 rows][128 bytes] swizzled block of Q
constexpr int kBlock = kTile * 128;        // the same of a K or V tile
constexpr int kMaxCtas = 148;              // SMs of a B200; partial results are laid out for these
constexpr int kInfo = 16;                  // tiles that are described in shared memory at once
constexpr int kSoftmaxThreads = 256;
// tiles per CTA below which fewer CTAs take part; the device's time for 1 request of 333 cached
// positions (8 items of 6 tiles): 1 tile 16.9 us, 2 16.4, 4 18.4, 8 23.5
constexpr int kMinTiles = 2;
// log2 by which a maximum may outgrow the reference, and fp16: by which the reference is set below the maximum
constexpr float kSlack = 8.0f, kHalfSlack = 5.0f, kHalfRoom = 9.0f;
constexpr int kNear = 6;                   // e4m3: powers of two between V scales that one e serves
constexpr int kFar = 0x10000;              // a biased exponent near to none
constexpr int kSpan = 60;                  // see far_unit
constexpr float kReach = 120.0f, kFarthest = 400.0f;   // log2 of a step of scaling; beyond kFarthest nothing is left in any case
constexpr float kL2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// warps 0-7 softmax, 8 and 9 MMA issuers (scores, accumulation), 10 index, 11 queries, 12-15 loaders
constexpr int kScoreWarp = 8, kAccumWarp = 9, kIndexWarp = 10, kQueryWarp = 11, kFirstLoader = 12, kLoaders = 4, kThreads = 512;

// a tile of keys, as the index warp describes it to the others
struct alignas(16) TileInfoPlain {
    int slot[kTile];          // of each position; 0 where there is none or it cannot be read
    uint32_t valid[2];        // the positions with a slot
    int head;                 // KV head
    int pad;
};
struct TileInfoScaled : TileInfoPlain {
    alignas(16) float ks[kTile];   // scales of K and V, 0 where there is no slot
    alignas(16) float vs[kTile];
};
template <bool kFp8> struct InfoOf { using type = TileInfoPlain; };
template <> struct InfoOf<true> { using type = TileInfoScaled; };

// ---- partial results ------------------------------------------------------------------------
// CTA c has two slots: 2c for a segment that continues an item, 2c + 1 for one that begins an item
// and does not finish it.
struct Split {          // written by CTA c for the item that reaches into it from CTA c - 1
    int valid;
    int b, h, block;
    int first, last;    // CTAs that hold parts of it
    int pad[2];
};

// division by a number fixed for the launch: q = (m + ((n - m) >> s1)) >> s2 with m = mul * n >> 32,
// exact for every 32-bit n (Granlund and Montgomery's round-up method)
struct Divisor {
    uint32_t mul;
    int s1, s2;
    __device__ __forceinline__ uint32_t divide(uint32_t n) const {
        const uint32_t m = __umulhi(mul, n);
        return (m + ((n - m) >> s1)) >> s2;
    }
};

struct KernelArgs {
    TreeAttnArgs t;
    Divisor page, group;    // by page_size, by t.group
    int pages;              // of the cache
    int wait_us, hold;      // limit of a wait; tile of a CTA that is never described (tests of that limit), -1
    int qt;                 // Q tiles of a row block
    Split* splits;          // [kMaxCtas]
    float2* part_ml;        // [2 * kMaxCtas][128 qt] (reference, sum)
    float4* part_o;         // [2 * kMaxCtas][DP / 4][128 qt], not normalised: columns in fours, rows
                            // adjacent, so that the threads of a warp (a row each) write in one run
};

// ---- requests, items, segments ---------------------------------------------------------------

struct Request {
    int lo, n;              // rows of q
    int len, p0;            // cached positions that the page table reaches, the first drafted one
    int rows, blocks;       // n x group, row blocks
};

__device__ __forceinline__ Request request_of(const TreeAttnArgs& a, int qt, int b) {
    Request r;
    long long lo, hi;
    if (a.indptr) {
        lo = __ldg(a.indptr + b);
        hi = __ldg(a.indptr + b + 1);
        lo = lo < 0 ? 0 : (lo > a.rows ? a.rows : lo);
        hi = hi < lo ? lo : (hi > a.rows ? a.rows : hi);
    } else {
        lo = (long long)b * a.width;
        hi = lo + a.width;
    }
    const int len = max(0, __ldg(a.lens + b));
    r.lo = (int)lo;
    r.n = (int)(hi - lo);
    r.len = min(len, a.max_pages * a.page_size);            // positions past the table are unseen,
    r.p0 = len - r.n;                                       // which moves no drafted token
    r.rows = r.n * a.group;
    r.blocks = (r.rows + kRows * qt - 1) / (kRows * qt);
    return r;
}

// tiles of keys that a row block needs: up to the last position its last row sees, one at least
__device__ __forceinline__ int tiles_of(const TreeAttnArgs& a, int qt, const Request& r, int block) {
    int end = r.len;
    if (!a.mask) {
        const int past = min(r.rows, (block + 1) * kRows * qt);
        end = min(end, r.p0 + (past - 1) / a.group + 1);
    }
    return end <= kTile ? 1 : (end + kTile - 1) / kTile;
}

__device__ __forceinline__ long long tiles_of_head(const TreeAttnArgs& a, int qt, const Request& r) {
    if (r.blocks <= 1 || a.mask) return r.blocks == 0 ? 0 : (long long)r.blocks * tiles_of(a, qt, r, r.blocks - 1);
    long long n = 0;
    for (int i = 0; i < r.blocks; ++i) n += tiles_of(a, qt, r, i);
    return n;
}

__device__ __forceinline__ long long first_tile(long long c, long long total, int ctas) {
    return total < (1 << 24) ? (long long)((uint32_t)c * (uint32_t)total / (uint32_t)ctas) : c * total / ctas;
}
// the CTA whose piece holds tile x
__device__ __forceinline__ int cta_of(long long x, long long total, int ctas) {
    return total < (1 << 24) ? (int)(((uint32_t)(x + 1) * (uint32_t)ctas - 1u) / (uint32_t)total)
                             : (int)(((x + 1) * ctas - 1) / total);
}

// The segments (runs of tiles of one item) of a CTA, in order, walked by the index and the query warp.
struct Walk {
    Request r;
    int b, h, block;
    int tiles;              // of the item
    int k0, k1;             // this segment's tiles
    long long left;         // tiles of this CTA after this segment

    // tile in_b of request b0's tiles (per_head of them for each KV head)
    __device__ __forceinline__ void begin(const KernelArgs& a, int b0, const Request& r0, long long per_head, long long in_b,
                                          long long count) {
        b = b0;
        r = r0;
        if (in_b < 0x7fffffff && per_head < 0x7fffffff)
            h = (int)((uint32_t)in_b / (uint32_t)per_head);
        else
            h = (int)(in_b / per_head);
        long long at = in_b - h * per_head;
        block = 0;
        tiles = tiles_of(a.t, a.qt, r, 0);
        while (at >= tiles) {
            at -= tiles;
            ++block;
            tiles = tiles_of(a.t, a.qt, r, block);
        }
        k0 = (int)at;
        left = count;
        take();
    }
    __device__ __forceinline__ void take() {
        k1 = (long long)(tiles - k0) < left ? tiles : k0 + (int)left;
        left -= k1 - k0;
    }
    // the next segment; false at the end of the CTA's piece.  By a whole warp, whose lanes all see
    // (and write) the same
    __device__ __noinline__ bool advance(const KernelArgs& a) {
        __syncwarp();
        if (left <= 0) return false;
        int b_ = b, h_ = h, block_ = block + 1;
        Request r_ = r;
        if (block_ >= r_.blocks) {
            block_ = 0;
            if (++h_ >= a.t.c.heads) {
                h_ = 0;
                do {
                    ++b_;
                    r_ = request_of(a.t, a.qt, b_);
                } while (r_.rows == 0);
            }
        }
        const int tiles_ = tiles_of(a.t, a.qt, r_, block_);
        const int take_ = tiles_ < left ? tiles_ : (int)left;
        const long long left_ = left - take_;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            b = b_;
            h = h_;
            block = block_;
            r = r_;
            tiles = tiles_;
            k0 = 0;
            k1 = take_;
            left = left_;
        }
        __syncwarp();
        return true;
    }
    __device__ __forceinline__ int count() const { return k1 - k0; }
    __device__ __forceinline__ int first_row(int qt) const { return block * kRows * qt; }
    __device__ __forceinline__ int rows(int qt) const { return min(r.rows - first_row(qt), kRows * qt); }
    __device__ __forceinline__ bool shared_rows(int qt) const { return rows(qt) <= kRows; }
};

constexpr int kMaxStages = 6;              // of the K ring, and of the V ring
constexpr int kRaw = 2;                    // e4m3: tiles of codes that a loader warp holds, one of them in flight

struct alignas(16) Shared {
    uint64_t full[2][kMaxStages];    // stage holds a K (first), a V tile
    uint64_t empty[2][kMaxStages];   // the matrix instructions that read it are done
    uint64_t info_full[kInfo];       // tile described
    uint64_t info_empty[kInfo];      // its last matrix instructions are done
    uint64_t q_full[2];              // a segment and its Q in shared memory
    uint64_t q_free[2];              // the segment is done with
    uint64_t s_full[2][2];           // scores of a stream's buffer in TMEM
    uint64_t p_full[2][2];           // weights of a stream's buffer in TMEM
    uint64_t s_free[2][2];           // the weights in a stream's buffer have been accumulated
    uint64_t described;              // the segment's walk is there, its Q is not yet
    uint64_t o_full;                 // the segment's accumulators are complete
    uint64_t joined;                 // both warpgroups have written what the other reads
    uint64_t drain[2];
    uint32_t tmem;
    int abort, wait_us;              // a wait has given up, and after how long: see wait_limit
    int odd[2];                      // a drafted V element was not finite (by segment parity)
    int e_low[8], e_eff[8];          // e4m3, a softmax warp each: see far_unit
    int v_done[2];                   // e4m3: V tiles (even, odd) in their stages, as one past the last
    long long scan[32];
    Walk start;                      // where this CTA starts on the line of tiles
    Walk seg[2];                     // the segments whose Q is here; read in place, registers are full
    Walk walk[2];                    // where the index and the query warp are
};

template <int DP, bool kFp8> struct Layout {
    static constexpr int kQTile = (DP / 64) * kQBlock;     // bytes of a Q tile
    static constexpr int kStage = (DP / 64) * kBlock;      // bytes of a K or V stage
    static constexpr int kRawTile = kFp8 ? kTile * DP : 0; // bytes of a tile of codes
    // stages of the K ring, and of the V ring.  Even: two loader warps share a ring, and a stage is
    // always filled by the same one and read by the same issuer, so that a wait on a stage's parity
    // never meets a phase two behind.
    static __host__ __device__ constexpr int stages() { return kFp8 ? (DP == 128 ? 2 : 4) : (DP == 128 ? 4 : 6); }
    static constexpr size_t info_bytes = sizeof(typename InfoOf<kFp8>::type) * kInfo;
    static constexpr size_t smem() {
        return (size_t)2 * kQTile + (size_t)2 * stages() * kStage + kLoaders * kRaw * kRawTile + sizeof(Shared) + info_bytes + (kFp8 ? 1024 : 0) + 1024;
    }
};
static_assert(Layout<128, false>::smem() <= 232448 && Layout<128, true>::smem() <= 232448 && Layout<64, false>::smem() <= 232448 &&
                  Layout<64, true>::smem() <= 232448,
              "shared memory of one CTA");

// ---- PTX helpers ------------------------------------------------------------------------------

// Order between the threads' writes to shared memory and the matrix instructions' reads (another
// proxy): the issuing thread runs the proxy fence, after it has seen the writers' barrier.  A fence
// in the producers would do as well, but there it waits for their loads in flight: measured, it
// left one tile in flight (64x1 bf16 455 us).

// shared-memory matrix descriptors: the low word holds the address and the distance between
// 128-byte column blocks (of an MN-major operand), both in 16-byte units, and takes offsets by
// addition; the high word is the same for all: 8 rows 1024 bytes apart, sm100 version, 128-byte swizzle
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lead_bytes) {
    return ((saddr >> 4) & 0x3FFFu) | ((lead_bytes >> 4) << 16);
}
__device__ __forceinline__ uint64_t desc(uint32_t low) { return ((uint64_t)kDescHigh << 32) | low; }

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Executed by the whole warp, issued by one elected lane: outside a divergent branch the operands
// stay in uniform registers, where the instruction wants them (issued from `if (lane == 0)` each
// took 90 cycles).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, one;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|one, 0xffffffff;\n\t"
        "@one tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, one;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|one, 0xffffffff;\n\t"
        "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred one;\n\telect.sync _|one, 0xffffffff;\n\t"
        "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

#define DSV_R16(x, o)                                                                                             \
    x(r[o + 0]), x(r[o + 1]), x(r[o + 2]), x(r[o + 3]), x(r[o + 4]), x(r[o + 5]), x(r[o + 6]), x(r[o + 7]),        \
        x(r[o + 8]), x(r[o + 9]), x(r[o + 10]), x(r[o + 11]), x(r[o + 12]), x(r[o + 13]), x(r[o + 14]), x(r[o + 15])

// 32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
#define DSV_OUT(y) "=r"(y)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : DSV_R16(DSV_OUT, 0), DSV_R16(DSV_OUT, 16)
        : "r"(taddr));
#undef DSV_OUT
}
// the loads issued so far are complete; `r` is in the operands so that no use of it moves ahead
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
#define DSV_IO(y) "+r"(y)
    asm volatile("tcgen05.wait::ld.sync.aligned;" : DSV_R16(DSV_IO, 0), DSV_R16(DSV_IO, 16)::"memory");
#undef DSV_IO
}
// 8 columns, and the wait for them
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
#define DSV_IN(y) "r"(y)
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::DSV_R16(DSV_IN, 0),
        DSV_R16(DSV_IN, 16), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15};" ::DSV_R16(DSV_IN, 0),
        "r"(taddr)
        : "memory");
#undef DSV_IN
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};\n\ttcgen05.wait::st.sync.aligned;" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%4], {%0, %1, %2, %3};\n\ttcgen05.wait::st.sync.aligned;" ::"r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(taddr)
                 : "memory");
}
#undef DSV_R16

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, __nv_bfloat16) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
}

__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool ok) {   // nothing is read where !ok
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
// 16 bytes global -> shared
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
// arrives at `bar` once this thread's copies so far have landed
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ns after which a wait gives up; Shared holds the limit beside the word that says that one has
__device__ __forceinline__ uint64_t wait_limit(volatile int* abort) { return (uint64_t)abort[1] * 1000u; }

// bounded wait that also gives up when another warp of the CTA has given up
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort) {
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if (i % 32 != 0) continue;
        if (*abort) return false;
        if (globaltimer_ns() - t0 > wait_limit(abort)) {
            *abort = 1;
            return false;
        }
    }
}
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort) {
    return mbar_try_wait(bar, parity) || wait_slow(bar, parity, abort);
}

// the same by shared-memory address, for the issuing warps: all lanes wait, one vote
__device__ __forceinline__ bool try_wait_at(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __noinline__ bool wait_slow_at(uint32_t bar, uint32_t parity, volatile int* abort) {
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t i = 1;; ++i) {
        if (try_wait_at(bar, parity)) return true;
        if (i % 32 != 0) continue;
        if (*abort) return false;
        if (globaltimer_ns() - t0 > wait_limit(abort)) {
            *abort = 1;
            return false;
        }
    }
}
// until *at is past `value`
__device__ __noinline__ bool wait_past(volatile int* at, int value, volatile int* abort) {
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t i = 1; *at <= value; ++i) {
        if (i % 32 != 0) continue;
        if (*abort) return false;
        if (globaltimer_ns() - t0 > wait_limit(abort)) {
            *abort = 1;
            return false;
        }
    }
    __threadfence_block();
    return true;
}
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, volatile int* abort) {
    if (__all_sync(0xffffffffu, try_wait_at(bar, parity))) return true;
    return __all_sync(0xffffffffu, wait_slow_at(bar, parity, abort));
}

// 16-byte chunk c of row `row` in a tile of 128-byte-swizzled blocks of `block` bytes
template <int block>
__device__ __forceinline__ uint32_t chunk_at(int row, int c) {
    return (uint32_t)((c >> 3) * block + row * 128 + (((c ^ row) & 7) << 4));
}

// Rows of q of a segment into a Q tile, by `warps` warps of which this is `warp`.  e4m3: as fp16 with a
// power of two per row, whose inverse goes to mul.
template <typename TQ, bool kFp8, int DP>
__device__ __noinline__ void bring_queries(const KernelArgs& a, const Walk& w, uint8_t* dst, float* mul, int warp, int warps) {
    constexpr int kTileBytes = (DP / 64) * kQBlock;
    constexpr int kLanes = DP / 8, kAtOnce = 32 / kLanes;       // lanes of a row (16-byte chunks), rows at once
    constexpr int kRun = 8 * kAtOnce;                           // adjacent rows of a warp
    const TreeAttnArgs& t = a.t;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, dr = lane / kLanes;
    const bool live = sub * 8 < t.c.dim;
    const int nrows = w.rows(a.qt), row0 = w.first_row(a.qt);
    const int filled = (nrows + 31) & ~31;                      // whole warps of rows: zeros past the last
    const int token0 = row0 / t.group, rem0 = row0 - token0 * t.group;
    const TQ* q = static_cast<const TQ*>(t.q) + (long long)(w.r.lo + token0) * t.q_token_stride +
                  (long long)(w.h * t.group) * t.q_head_stride + sub * 8;
    auto place = [&](int r) { return dst + (r >> 7) * kTileBytes + chunk_at<kQBlock>(r & 127, sub); };
    for (int r0 = warp * kRun + dr; r0 - dr < filled; r0 += warps * kRun) {
#pragma unroll 4
        for (int k = 0; k < 8; ++k) {
            const int r = r0 + k * kAtOnce, i = (int)a.group.divide(rem0 + r);
            const bool have = r < nrows && live;
            cp16_or_zero(smem_u32(place(r)), have ? q + i * t.q_token_stride + (rem0 + r - i * t.group) * t.q_head_stride : q, have);
        }
    }
    cp_wait_all();
    if constexpr (kFp8) {
        // to fp16 in place, each lane what it has copied
#pragma unroll 1
        for (int r0 = warp * kRun + dr; r0 - dr < filled; r0 += warps * kRun) {
            uint4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4*>(place(r0 + i * kAtOnce));
            // the largest size in each row, as bits without the sign (ordered as the values are); all
            // rows before the first store, so that the shuffles overlap
            uint32_t top[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t sizes = __vmaxu2(__vmaxu2(x[i].x & 0x7FFF7FFFu, x[i].y & 0x7FFF7FFFu),
                                                __vmaxu2(x[i].z & 0x7FFF7FFFu, x[i].w & 0x7FFF7FFFu));
                top[i] = max(sizes >> 16, sizes & 0xFFFFu);
            }
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = r0 + i * kAtOnce;
                float f[8], m, none;
                unpack2(x[i].x, f[0], f[1], TQ());
                unpack2(x[i].y, f[2], f[3], TQ());
                unpack2(x[i].z, f[4], f[5], TQ());
                unpack2(x[i].w, f[6], f[7], TQ());
                unpack2(top[i], m, none, TQ());
                // a power of two that brings the row's largest value to [2^13, 2^14): products stay
                // exact, values down to 2^-27 of the largest keep fp16's precision (a bf16 value is
                // whole down to 2^-30), those down to 2^-37 a place in fp16.  A
                // row with a NaN or an infinity is left as it is: its scores are NaN or infinite
                int e = (int)(__float_as_uint(m) >> 23) - 127;
                e = m > 0.f && e < 128 ? max(e, -100) : 13;
                const float up = __uint_as_float((uint32_t)(13 - e + 127) << 23);
                if (sub == 0) mul[r] = __uint_as_float((uint32_t)(e - 13 + 127) << 23);
                *reinterpret_cast<uint4*>(place(r)) =
                    make_uint4(pack2(f[0] * up, f[1] * up, __half()), pack2(f[2] * up, f[3] * up, __half()),
                               pack2(f[4] * up, f[5] * up, __half()), pack2(f[6] * up, f[7] * up, __half()));
            }
        }
    }
}

// columns [c, end) of this thread's TMEM lane times f
__device__ __noinline__ void scale_columns(uint32_t taddr, int c, int end, float f) {
#pragma unroll 1
    for (; c < end; c += 8) {
        uint32_t x[8];
        tmem_ld8(taddr + c, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
        tmem_st8(taddr + c, x);
    }
}

// e4m3: of two accumulators 128 columns apart the one with the lower reference (by kReach to kFarthest) is
// scaled towards the other, in columns [c, end)
__device__ __noinline__ float4 bring_nearer(uint32_t taddr, int c, int end, float2 x, float2 y) {
    for (int k = 0; k < 3; ++k) {
        const float apart = x.x - y.x, by = 7.5231638e-37f;     // 2^-120
        const bool low_x = apart < -kReach && apart > -kFarthest, low_y = apart > kReach && apart < kFarthest;
        if (!__any_sync(0xffffffffu, low_x || low_y)) break;
        scale_columns(taddr, c, end, low_x ? by : 1.f);
        scale_columns(taddr + 128, c, end, low_y ? by : 1.f);
        if (low_x) x = make_float2(x.x + kReach, x.y * by);
        if (low_y) y = make_float2(y.x + kReach, y.y * by);
    }
    return make_float4(x.x, x.y, y.x, y.y);
}

// e4m3: NaN into the columns [c, end) of a row's accumulator where a V element of a drafted token that the row sees is one
// (the tile's own have been zeroed); by whole warps, `mine` where the lane has a row
__device__ __noinline__ void add_nan(const KernelArgs& a, const Walk& w, uint32_t taddr, int c, int end, int token, uint64_t bits, bool mine) {
    const TreeAttnArgs& t = a.t;
    const int n0 = max(max(0, w.k0 * kTile - w.r.p0), -w.r.p0), n1 = min(w.r.len, w.k1 * kTile) - w.r.p0;
#pragma unroll 1
    for (; c < end; c += 8) {
        uint32_t x[8];
        tmem_ld8(taddr + c, x);
        for (int j = n0; j < n1; ++j) {
            if (!mine || !(t.mask ? j < 64 && ((bits >> j) & 1) : j <= token)) continue;
            const int pos = w.r.p0 + j;
            const int page = __ldg(t.table + (long long)w.b * t.table_stride + pos / t.page_size);
            if (page < 0 || page >= a.pages) continue;
            const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.c.v) +
                                                            (long long)(page * t.page_size + pos % t.page_size) * t.c.slot_stride +
                                                            (long long)w.h * t.c.head_stride + c);
#pragma unroll
            for (int d = 0; d < 8; ++d)
                if ((((d < 4 ? q.x : q.y) >> (8 * (d & 3))) & 0x7F) == 0x7F) x[d] = 0x7fffffffu;
        }
        __syncwarp();
        tmem_st8(taddr + c, x);
    }
}

// where V scales have to lie to be near those of a tile (biased; e within [-90, 120])
__device__ __forceinline__ int first_window(const float* vs, const uint32_t* valid) {
    const int lane = threadIdx.x & 31;
    int most = -1;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if ((valid[e] >> lane) & 1u) most = max(most, (int)(__float_as_uint(fabsf(vs[e * 32 + lane])) >> 23));
    most = __reduce_max_sync(0xffffffffu, most);
    return most < 0 || most > 246 ? kFar : max(36, most + 1 - kNear);
}

struct FarResult {
    float ref, sum;
    int e_low;                // -1 after a wait that gave up
};

// e4m3: a unit whose V scales lie far apart or are not finite, from its scores to its weights in TMEM, with an e for each key.
//
// A reference may rise by the whole range of e here, more than one factor in fp32 bridges, so
// accumulator and sum follow in steps of 2^-kReach (three at most; scores that differ by kFarthest
// leave nothing).  The tiles between scale in one step.  What that flushes to zero (factors below
// 2^-126) has to be nothing beside the new sum.  A sum is at most (keys) x 2^(14 - e_eff), e_eff the least
// that e has added to the maximum of a row's scores so far, and the new one at least 2^(9 - kNear - e): with
// 2^31 keys and e <= e_eff + kSpan, 2^(31 + 14 - 3 + kSpan - 126) = 2^-24 of it, and 2^-38 with 2^17
// keys.  So where the V scales have risen by more than kSpan above e_eff, the tiles to come are far
// as well.
__device__ __noinline__ FarResult far_unit(uint32_t ts, uint32_t to, int dim, float cm, uint2 vis, const TileInfoScaled& inf, float ref,
                                           float sum, int e_low, Shared* sh, uint64_t* used, uint32_t parity) {
    __syncwarp();
    const float *ks = inf.ks, *vs = inf.vs;
    volatile int *e_eff = &sh->e_eff[threadIdx.x >> 5], *abort = &sh->abort;
    auto power = [](float scale) {                              // e of a scale; of one that is not finite the least
        const uint32_t x = __float_as_uint(fabsf(scale));
        return x >= 0x7f800000u ? -90 : max(-90, min(120, (int)(x >> 23) - 126));
    };
    float target = -INFINITY, top = -INFINITY;
    int most = -90;
#pragma unroll 1
    for (int j = 0; j < kTile; j += 8) {
        uint32_t x[8];
        tmem_ld8(ts + j, x);
        const uint32_t seen = (j & 32 ? vis.y : vis.x) >> (j & 31);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(ks + j + i), v4 = *reinterpret_cast<const float4*>(vs + j + i);
            const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, vv[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = power(vv[k]);
                const float s = __uint_as_float(x[i + k]) * kk[k];
                most = max(most, e);
                if ((seen >> (i + k)) & 1u) {
                    top = fmaxf(top, s * cm);
                    target = fmaxf(target, fmaf(s, cm, (float)e));
                }
            }
        }
    }
    int least = min(*e_eff, e_low == kFar ? kFar : e_low - 126);
    least = min(least, __reduce_min_sync(0xffffffffu, target > -INFINITY && top < INFINITY ? (int)floorf(target - top) : kFar));
    __syncwarp();
    *e_eff = least;                                             // every lane the same
    most += 127 - kNear;                                        // biased; room for one power above these
    e_low = max(most, 36) - 126 > least + kSpan - kNear ? kFar : max(most, 36);
    target -= kHalfRoom;
    for (int k = 0; k < 4 && __any_sync(0xffffffffu, target > ref + kHalfSlack); ++k) {
        float to_ref = fmaxf(ref, target);
        if (k < 3 && to_ref < ref + kFarthest) to_ref = fminf(to_ref, ref + kReach);
        if (used) {                                             // the accumulator holds something
            if (!__all_sync(0xffffffffu, wait_or_abort(used, parity, abort))) return {ref, sum, -1};
            tc_fence_after();
            const float f = ref == -INFINITY ? 1.0f : ex2(ref - to_ref);
            sum *= f;
            scale_columns(to, 0, dim, f);
        }
        ref = to_ref;
    }
    const float nref = ref == -INFINITY ? 0.f : -ref;
    float part = 0.f;
#pragma unroll 1
    for (int j = 0; j < kTile; j += 8) {
        uint32_t x[8], p[4];
        tmem_ld8(ts + j, x);
        const uint32_t seen = (j & 32 ? vis.y : vis.x) >> (j & 31);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(ks + j + i), v4 = *reinterpret_cast<const float4*>(vs + j + i);
            const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, vv[4] = {v4.x, v4.y, v4.z, v4.w};
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool sees = (seen >> (i + k)) & 1u;
                w[k] = sees ? ex2(fmaf(__uint_as_float(x[i + k]) * kk[k], cm, nref)) : 0.f;
                part += w[k];
                w[k] = sees ? w[k] * vv[k] : 0.f;              // a scale that is not finite: the rows that see it alone
            }
            p[i / 2] = pack2(w[0], w[1], __half());
            p[i / 2 + 1] = pack2(w[2], w[3], __half());
        }
        tmem_st4(ts + j / 2, p);                                // over scores that have been read
    }
    return {ref, sum + part, e_low};
}

// A wait has given up: NaN for all rows of this CTA's segments, so that none passes for a result.  By one warp.
__device__ __noinline__ void give_up(const KernelArgs& a, Shared* sh) {
    Walk& w = sh->walk[0];
    const TreeAttnArgs& t = a.t;
    const int lane = threadIdx.x & 31, per = kRows * a.qt;
    const float nan = __int_as_float(0x7fffffff);
    if (lane == 0) {
        w = sh->start;
        if (t.err) atomicOr(t.err, 4u);
    }
    __syncwarp();
    do {
        const bool whole = w.k0 == 0 && w.k1 == w.tiles;
        for (int r = lane; r < w.rows(a.qt); r += 32) {
            const int token = (w.first_row(a.qt) + r) / t.group, hq = w.h * t.group + (w.first_row(a.qt) + r) - token * t.group;
            if (!whole) {                                       // the join makes NaN of it
                a.part_ml[(long long)(2 * blockIdx.x + (w.k0 == 0 ? 1 : 0)) * per + r] = make_float2(nan, nan);
                continue;
            }
            uint16_t* out = static_cast<uint16_t*>(t.out) + (w.r.lo + token) * t.out_token_stride + hq * t.out_head_stride;
            for (int d = 0; d < t.c.dim; ++d) out[d] = 0x7fff;  // NaN of either type
            if (t.lse) t.lse[(long long)(w.r.lo + token) * t.q_heads + hq] = nan;
        }
    } while (w.advance(a));
}

// A unit is one stream's share of a tile: unit u of a segment belongs to stream u & 1 and uses its
// score buffer (u >> 1) & 1; its tile is u, or u >> 1 where both streams use every tile.

// ---- the kernel ---------------------------------------------------------------------------------

template <typename TQ, bool kFp8, int DP>
__global__ void __launch_bounds__(kThreads, 1) attn_kernel(const __grid_constant__ KernelArgs a) {
    using L = Layout<DP, kFp8>;
    using Info = typename InfoOf<kFp8>::type;
    using TO = typename std::conditional<kFp8, __half, TQ>::type;   // operands of the matrix instructions
    extern __shared__ uint8_t smem_raw[];
    constexpr int stages = L::stages();
    const int qt = a.qt, q_bufs = qt == 1 ? 2 : 1;         // segments whose Q is held at once
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sq = base;                                    // two Q tiles: of two segments, or of one with both streams' rows
    uint8_t* ring = base + 2 * L::kQTile;                  // [K, V][stages][kStage]
    uint8_t* raw = ring + 2 * stages * L::kStage;              // e4m3: [kLoaders][kRaw][kRawTile]
    Shared* sh = reinterpret_cast<Shared*>(raw + (kFp8 ? kLoaders * kRaw * L::kRawTile : 0));
    Info* info = reinterpret_cast<Info*>(sh + 1);
    float* row_mul = reinterpret_cast<float*>(info + kInfo);        // e4m3: [128 qt] power of two of a row of q
    volatile int* abort = &sh->abort;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const TreeAttnArgs& t = a.t;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (tid == 0) a.splits[blockIdx.x].valid = 0;     // before the scan's barrier, after which it may be set

    // ---- this CTA's piece of the line of tiles: a block scan over the requests' tiles, a second
    // round over the requests only where they are more than the threads
    long long total = 0, per_head = 0, c = 0, upto = 0;   // of all; of this thread's request; up to it
    Request rq;
    auto scan = [&](int b0) {
        const int b = b0 + tid;
        c = per_head = 0;
        if (b < t.batch) {
            rq = request_of(t, qt, b);
            per_head = tiles_of_head(t, qt, rq);
            c = per_head * t.c.heads;
        }
        upto = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += up;
        }
        if (lane == 31) sh->scan[warp] = upto;
        __syncthreads();
        long long all = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) {
            const long long x = sh->scan[i];
            if (i < warp) upto += x;
            all += x;
        }
        return all;
    };
    for (int b0 = 0; b0 < t.batch; b0 += kThreads) {
        if (b0 > 0) __syncthreads();
        total += scan(b0);
        if (t.err && blockIdx.x == 0 && b0 + tid < t.batch && __ldg(t.lens + b0 + tid) > t.max_pages * t.page_size)
            atomicOr(t.err, 2u);
    }
    // the same in every lane; said so, that what follows counts as uniform control flow
    total = __shfl_sync(0xffffffffu, total, 0);
    const long long want = total / kMinTiles;
    const int ctas = (int)(want < 1 ? 1 : (want < (long long)gridDim.x ? want : (long long)gridDim.x));
    if (total == 0 || (int)blockIdx.x >= ctas) return;
    const long long mine = first_tile(blockIdx.x, total, ctas);
    const long long count = first_tile(blockIdx.x + 1, total, ctas) - mine;
    {
        long long before = 0;
        for (int b0 = 0; b0 < t.batch; b0 += kThreads) {
            if (t.batch > kThreads) {
                __syncthreads();
                const long long all = scan(b0);
                upto += before;
                before += all;
            }
            if (c > 0 && mine >= upto - c && mine < upto) {
                Walk w0;
                w0.begin(a, b0 + tid, rq, per_head, mine - (upto - c), count);
                sh->start = w0;
                if (w0.k0 > 0) {
                    const long long i0 = mine - w0.k0;
                    Split sp = {1, w0.b, w0.h, w0.block, cta_of(i0, total, ctas), cta_of(i0 + w0.tiles - 1, total, ctas), {0, 0}};
                    a.splits[blockIdx.x] = sp;
                }
            }
        }
    }

    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&sh->full[i][s], kFp8 ? 1 : 32);
                mbar_init(&sh->empty[i][s], 1);
            }
        }
        for (int i = 0; i < kInfo; ++i) {
            mbar_init(&sh->info_full[i], kFp8 ? 33 : 1);
            mbar_init(&sh->info_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh->q_full[i], kSoftmaxThreads / 32);
            mbar_init(&sh->q_free[i], 8);
            for (int j = 0; j < 2; ++j) {
                mbar_init(&sh->s_full[i][j], 1);
                mbar_init(&sh->p_full[i][j], 4);
                mbar_init(&sh->s_free[i][j], 1);
            }
            mbar_init(&sh->drain[i], 1);
        }
        mbar_init(&sh->described, 1);
        mbar_init(&sh->o_full, 1);
        mbar_init(&sh->joined, 8);
        sh->abort = 0;
        sh->wait_us = a.wait_us;
        sh->odd[0] = sh->odd[1] = 0;
        sh->v_done[0] = sh->v_done[1] = 0;
        fence_mbar_init();
    }
    if (warp == kScoreWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh->tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;                           // all 512 columns were allocated
    // Up to 64 rows only the softmax warps of schedulers 0 and 1 have any: the loaders there change
    // places with the index and the query warp (the change alone, on one set of inputs repeated, which L2
    // serves in part: 64 x 16 e4m3, 64 rows: 243.2 us from 246.0; 64 x 1 bf16, 4 rows: 215.3 from 216.0).
    // With more rows they would meet on schedulers 2 and 3 alone.
    const int role = (long long)t.group * t.width <= 64 && warp >= kIndexWarp && warp < kFirstLoader + 2 ? warp ^ 6 : warp;
    if (role >= kFirstLoader) {
        // ---------------- loaders: rows of K and V by 16-byte copies of the lanes -----------------
        // Two warps for K tiles, two for V, every other tile each.  fp16, bf16: straight into the
        // swizzled stage.  e4m3: as codes into a raw tile of its own, the next one's on the way
        // while each lane brings what it has copied into the stage as fp16.
        // Copies of a lane, not TMA: one warp of them reaches 5.6 TB/s, two 6.7, whatever the page
        // size; gathers of four rows and bulk copies of one stay at 2.2 and 1.3 (scattered rows of
        // 256 bytes, nothing else running).
        const int lw = role - kFirstLoader;
        constexpr int kElem = kFp8 ? 1 : 2;                     // bytes of a cached element
        const uint32_t stride = (uint32_t)t.c.slot_stride * (uint32_t)kElem;   // bytes from slot to slot
        constexpr int kLanes = DP * kElem / 16, kAtOnce = 32 / kLanes;         // lanes of a row, rows at once
        constexpr int kSteps = kTile / kAtOnce;
        // e4m3: a row of codes becomes up to two blocks of fp16; four lanes of one row then stand beside
        // four of the next, so that their stores of eight hit eight different groups of banks
        const int sub = kFp8 && DP == 128 ? (lane & 3) | ((lane >> 1) & 4) : lane % kLanes;
        const int dr = kFp8 && DP == 128 ? ((lane >> 2) & 1) | ((lane >> 3) & 2) : lane / kLanes;
        // rows of step k: e4m3 kAtOnce adjacent ones; else dr's own run of kSteps
        const int row0 = kFp8 ? dr : dr * kSteps;
        const bool live = sub * (16 / kElem) < t.c.dim;
        const int which = lw >> 1;                              // 0: K, 1: V
        const uint32_t bars = smem_u32(sh), empty = bars + offsetof(Shared, empty) + which * (kMaxStages * 8);
        uint64_t* full = sh->full[which];
        uint8_t* stage0 = ring + which * (stages * L::kStage);
        const uint8_t* rows = static_cast<const uint8_t*>(which ? t.c.v : t.c.k) + sub * 16;
        int tl = (lw & 1) - 2;                                  // this warp's tile
        bool ok = true;
        const uint8_t* src = nullptr;
        const int* slots = nullptr;
        auto next = [&]() {                                     // false past the last, or after a wait that gave up
            tl += 2;
            if (tl >= (int)count) return false;
            ok = wait_at(bars + offsetof(Shared, info_full) + 8 * (tl % kInfo), (uint32_t)(tl / kInfo) & 1u, abort);
            slots = info[tl % kInfo].slot + row0;
            src = rows + kElem * (info[tl % kInfo].head * t.c.head_stride);
            return ok;
        };
        uint32_t s = lw & 1, ph = 1;                            // stage, and the parity that says it is free
        auto step_stage = [&]() {
            s += 2;
            if (s >= (uint32_t)stages) {
                s -= stages;
                ph ^= 1u;
            }
        };
        if constexpr (!kFp8) {
            while (next()) {
                ok = wait_at(empty + 8 * s, ph, abort);
                if (!ok) break;
                // chunk of row r: rows are 128 bytes apart, the chunk's place is xored with r & 7
                const uint32_t dst = smem_u32(stage0 + s * L::kStage) + (sub >> 3) * kBlock + row0 * 128 + ((sub & 7) << 4);
                if (live) {
                    // slots four at a time, and the next four before the copies of these are issued
                    // (loads do not move past the copies by themselves)
                    int4 four = *reinterpret_cast<const int4*>(slots);
#pragma unroll 2
                    for (int k = 0; k < kSteps; k += 4) {
                        const int4 now = four;
                        four = *reinterpret_cast<const int4*>(slots + (k + 4 < kSteps ? k + 4 : 0));
                        const uint32_t at = dst ^ ((k & 4) << 4), to = k * 128;
                        cp16(at + to, src + (uint64_t)(uint32_t)now.x * stride);
                        cp16((at ^ 16) + to + 128, src + (uint64_t)(uint32_t)now.y * stride);
                        cp16((at ^ 32) + to + 256, src + (uint64_t)(uint32_t)now.z * stride);
                        cp16((at ^ 48) + to + 384, src + (uint64_t)(uint32_t)now.w * stride);
                    }
                }
                cp_arrive(full + s);
                step_stage();
            }
        } else {
            uint8_t* own = raw + lw * (kRaw * L::kRawTile) + dr * DP + sub * 16;
            auto fetch = [&](uint32_t r) {                      // this warp's next tile on its way to raw tile r
                if (!next()) return false;
                if (live) {
                    const uint32_t dst = smem_u32(own + r * L::kRawTile);
#pragma unroll 1
                    for (int k = 0; k < kSteps; k += 8) {
                        int slot[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) slot[q] = slots[(k + q) * kAtOnce];
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            cp16(dst + (k + q) * kAtOnce * DP, src + (uint64_t)(uint32_t)slot[q] * stride);
                    }
                }
                return true;
            };
            uint32_t r = 0;
            int done = lw & 1;                                  // the tile being converted
            bool have = fetch(0);
            cp_commit();
#pragma unroll 1
            while (have) {
                have = fetch(r ^ 1);
                cp_commit();
                if (!ok) break;
                cp_wait<1>();                                   // this tile's codes have landed
                ok = wait_at(empty + 8 * s, ph, abort);
                if (!ok) break;
                const uint8_t* from = own + r * L::kRawTile;
                uint8_t* dst = stage0 + s * L::kStage;
                if (live) {
                    uint4 next4[4];                             // loads ahead of the stores of those before
#pragma unroll
                    for (int k = 0; k < 4; ++k) next4[k] = *reinterpret_cast<const uint4*>(from + k * kAtOnce * DP);
#pragma unroll 1
                    for (int k0 = 0; k0 < kSteps; k0 += 4) {
                        uint4 x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] = next4[k];
                        if (k0 + 4 < kSteps) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) next4[k] = *reinterpret_cast<const uint4*>(from + (k0 + 4 + k) * kAtOnce * DP);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int row = row0 + (k0 + k) * kAtOnce;
                            const uint32_t c4[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
                            uint32_t o[8];
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((uint16_t)(c4[q >> 1] >> (16 * (q & 1))), __NV_E4M3);
                                o[q] = (uint32_t)h.x | ((uint32_t)h.y << 16);
                            }
                            *reinterpret_cast<uint4*>(dst + chunk_at<kBlock>(row, 2 * sub)) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(dst + chunk_at<kBlock>(row, 2 * sub + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) {
                    if (which) {
                        __threadfence_block();
                        *(volatile int*)&sh->v_done[lw & 1] = done + 1;
                    }
                    mbar_arrive(full + s);
                }
                done += 2;
                step_stage();
                r ^= 1;
            }
        }
        cp_wait_all();
    } else if (role == kIndexWarp) {
        // ---------------- index: slots, scales and validity of the tiles to come ----------------
        Walk& w = sh->walk[0];
        if (lane == 0) w = sh->start;
        __syncwarp();
        int ti = 0;
        bool ok = true;
        do {
            const int nt = w.count();
            const int* table = t.table + (long long)w.b * t.table_stride;
            // a tile's page table entries are fetched one round of two tiles ahead
            auto entry_of = [&](int tl, int e) {
                const int pos = (w.k0 + tl) * kTile + e * 32 + lane;
                return tl < nt && pos < w.r.len ? __ldg(table + a.page.divide(pos)) : 0;
            };
            int entry[2][2] = {{entry_of(0, 0), entry_of(0, 1)}, {entry_of(1, 0), entry_of(1, 1)}};
#pragma unroll 1
            for (int t0 = 0; ok && t0 < nt; t0 += 2) {
                int now[2][2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) now[k][e] = entry[k][e];
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) entry[k][e] = entry_of(t0 + 2 + k, e);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (t0 + k >= nt) break;
                    const int at = ti % kInfo;
                    ok = __all_sync(0xffffffffu, ti != a.hold &&
                                    wait_or_abort(&sh->info_empty[at], ((uint32_t)(ti / kInfo) & 1u) ^ 1u, abort));
                    if (!ok) break;
                    Info* f = info + at;
                    uint32_t valid[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int pos = (w.k0 + t0 + k) * kTile + e * 32 + lane, page = now[k][e];
                        int slot = -1;
                        if (pos < w.r.len) {
                            if (page >= 0 && page < a.pages)
                                slot = page * t.page_size + (pos - (int)a.page.divide(pos) * t.page_size);
                            else if (t.err)
                                atomicOr(t.err, 2u);
                        }
                        f->slot[e * 32 + lane] = max(slot, 0);
                        valid[e] = __ballot_sync(0xffffffffu, slot >= 0);
                        if constexpr (kFp8) {
                            const long long from = max(slot, 0) * t.c.scale_stride + w.h;
                            cp4(smem_u32(f->ks + e * 32 + lane), t.c.k_scale + from, slot >= 0);
                            cp4(smem_u32(f->vs + e * 32 + lane), t.c.v_scale + from, slot >= 0);
                        }
                    }
                    if constexpr (kFp8) cp_arrive(&sh->info_full[at]);
                    if (lane == 0) {
                        f->valid[0] = valid[0];
                        f->valid[1] = valid[1];
                        f->head = w.h;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->info_full[at]);
                    ++ti;
                }
            }
        } while (ok && w.advance(a));
        if constexpr (kFp8) cp_wait_all();
    } else if (role == kQueryWarp) {
        // ---------------- queries: the next segment and its rows of q, a segment ahead ------------
        // (the softmax warps bring the first segment's, and all where there is no room for two)
        Walk& w = sh->walk[1];
        if (lane == 0) w = sh->start;
        __syncwarp();
        uint32_t seg = 1;
        while (w.advance(a)) {
            const uint32_t buf = seg % q_bufs;
            if (!wait_at(smem_u32(&sh->q_free[buf]), ((seg / q_bufs) & 1u) ^ 1u, abort)) break;
            if (lane == 0) sh->seg[buf] = w;
            if (q_bufs > 1) bring_queries<TQ, kFp8, DP>(a, w, sq + buf * L::kQTile, row_mul + buf * kRows, 0, 1);
            __syncwarp();
            if (lane == 0) {
                if (q_bufs > 1)
                    mbar_arrive_n(smem_u32(&sh->q_full[buf]), kSoftmaxThreads / 32);
                else
                    mbar_arrive(&sh->described);
            }
            ++seg;
        }
    } else if (warp == kScoreWarp || warp == kAccumWarp) {
        // ---------------- MMA issuers: one warp for S = Q K^T, one for O += P V ----------------
        // Two, because a unit costs the issuing warp more in waits, commits and issue than the
        // tensor core needs for it (one warp: 1960 cycles a unit of 640 tensor cycles).
        constexpr uint32_t kFormat = std::is_same<TO, __nv_bfloat16>::value ? 1u : 0u;
        constexpr uint32_t kCommon = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((uint32_t)(kRows >> 4) << 24);
        constexpr uint32_t kIdescS = kCommon | ((uint32_t)(kTile >> 3) << 17);
        const bool scores = warp == kScoreWarp;
        const uint32_t bars = smem_u32(sh), full = bars + offsetof(Shared, full) + (scores ? 0 : kMaxStages * 8),
                       empty = bars + offsetof(Shared, empty) + (scores ? 0 : kMaxStages * 8),
                       s_full = bars + offsetof(Shared, s_full), p_full = bars + offsetof(Shared, p_full),
                       s_free = bars + offsetof(Shared, s_free);
        uint32_t seg = 0, tile0 = 0, ph = 0;                 // ph: parity of each (stream, buffer)
        uint32_t st = 0, sp = 0;                             // stage of the warp's ring, and its parity
        bool ok = true;
        auto step_stage = [&]() {
            if (++st == (uint32_t)stages) {
                st = 0;
                sp ^= 1u;
            }
        };
        do {
            // broadcasts: what the loop turns on is uniform, and so its operands stay in uniform registers
            const uint32_t buf = seg % q_bufs;
            ok = wait_at(bars + offsetof(Shared, q_full) + 8 * buf, (seg / q_bufs) & 1u, abort);
            if (!ok) break;
            const bool both = __shfl_sync(0xffffffffu, (int)!sh->seg[buf].shared_rows(qt), 0) != 0;   // both streams use every tile
            const int nt = __shfl_sync(0xffffffffu, sh->seg[buf].count(), 0);
            const uint32_t step = both ? 1u : 0u;
            const int units = nt << step;
            if (scores) {
                const int ksteps = t.c.dim / 16;
                const uint32_t q0 = desc_low(smem_u32(sq + buf * L::kQTile), 16), k0 = desc_low(smem_u32(ring), 16);
                auto ready = [&](int u) {                    // K tile and score buffer of unit u
                    const uint32_t s = u & 1, sb = (s << 1) | ((u >> 1) & 1);
                    if (!(s & step)) {
                        ok = wait_at(full + 8 * st, sp, abort);
                        fence_proxy_async_smem();
                    }
                    ok = ok && wait_at(s_free + 8 * sb, ((ph >> sb) & 1u) ^ 1u, abort);
                    ph ^= 1u << sb;
                    tc_fence_after();
                };
                ready(0);
                for (int u = 0; ok && u < units; ++u) {
                    const uint32_t s = u & 1, sb = (s << 1) | ((u >> 1) & 1), mine = st;
                    const uint32_t qa = q0 + (s & step) * (L::kQTile >> 4), kb = k0 + st * (L::kStage >> 4), d = tmem + sb * kTile;
                    const bool last = (s & step) == step;    // the last use of the tile
                    auto issue = [&](int k) {
                        const uint32_t col = (k & 3) * 2;
                        if (k < ksteps)
                            mma_ss(d, desc(qa + (k >> 2) * (kQBlock >> 4) + col), desc(kb + (k >> 2) * (kBlock >> 4) + col), kIdescS,
                                   k != 0);
                    };
#pragma unroll
                    for (int k = 0; k < DP / 32; ++k) issue(k);
                    if (last) step_stage();
                    // the next unit's waits while these execute; not with a ring of two, where the
                    // next tile's warp may be waiting for this stage
                    if (stages > 2 && u + 1 < units) ready(u + 1);
                    if (!ok) break;
#pragma unroll
                    for (int k = DP / 32; k < DP / 16; ++k) issue(k);
                    mma_commit(s_full + 8 * sb);
                    if (last) mma_commit(empty + 8 * mine);
                    if (stages <= 2 && u + 1 < units) ready(u + 1);
                }
            } else {
                const uint32_t v0 = desc_low(smem_u32(ring + stages * L::kStage), kBlock);
                const uint32_t idesc_o = kCommon | (1u << 16) | ((uint32_t)(t.c.dim >> 3) << 17);  // B: MN-major
                for (int u = 0; ok && u < units; ++u) {
                    const uint32_t s = u & 1, sb = (s << 1) | ((u >> 1) & 1);
                    if (!(s & step)) ok = wait_at(full + 8 * st, sp, abort);
                    ok = ok && wait_at(p_full + 8 * sb, (ph >> sb) & 1u, abort);
                    if (!ok) break;
                    ph ^= 1u << sb;
                    // V, and the zeros that each warpgroup has put into all of it; so once a tile
                    if (!(s & step)) fence_proxy_async_smem();
                    tc_fence_after();
                    const uint32_t vb = v0 + st * (L::kStage >> 4), d = tmem + 256 + s * 128, p = tmem + sb * kTile;
#pragma unroll
                    for (int k = 0; k < kTile / 16; ++k)
                        mma_ts(d, p + k * 8, desc(vb + k * (2048 >> 4)), idesc_o, k ? 1u : (uint32_t)(u > 1));
                    mma_commit(s_free + 8 * sb);
                    if ((s & step) == step) {
                        mma_commit(empty + 8 * st);
                        mma_commit(bars + offsetof(Shared, info_empty) + 8 * ((tile0 + (u >> step)) % kInfo));
                        step_stage();
                    }
                }
                if (ok) mma_commit(bars + offsetof(Shared, o_full));
            }
            tile0 += nt;
            ++seg;
        } while (ok && tile0 < (uint32_t)count);
        // every instruction issued here is done before TMEM is released
        uint64_t* drain = &sh->drain[scores ? 0 : 1];
        mma_commit(smem_u32(drain));
        if (!mbar_wait_bounded(drain, 0)) *abort = 1;
        __syncwarp();
    } else if (warp < 8) {
        // ---------------- softmax and epilogue: one row per thread ----------------
        const int s = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t to = tmem + lanes + 256 + s * 128;
        constexpr int kLanes = DP / 8;                          // 16-byte chunks of a row
        constexpr int kStep = kSoftmaxThreads / kLanes;         // rows that the 256 threads move at once
        uint32_t seg = 0, tile0 = 0, jp = 0;                    // jp: phases of `joined`
        uint32_t ph = 0;                                        // parity of each buffer
        bool ok = true;
        auto join = [&]() {                                     // both warpgroups have come here
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->joined);
            ok = __all_sync(0xffffffffu, ok && wait_or_abort(&sh->joined, jp & 1u, abort));
            ++jp;
        };
        do {
            const uint32_t buf = seg % q_bufs;
            if (seg == 0 || q_bufs == 1) {
                // Queries that could not be brought ahead: by eight warps, as copies behind those of the
                // loaders are slow to issue (one warp took 27 thousand cycles for 256 rows)
                if (seg == 0) {
                    if (tid == 0) sh->seg[0] = sh->start;
                } else {
                    ok = wait_at(smem_u32(&sh->described), (seg - 1) & 1u, abort);
                    if (!ok) break;
                }
                bring_queries<TQ, kFp8, DP>(a, seg == 0 ? sh->start : sh->seg[0], sq, row_mul, warp, kSoftmaxThreads / 32);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->q_full[0]);
                if constexpr (kFp8) {
                    if (seg == 0) {                             // V scales like those of the first tile are near
                        ok = wait_at(smem_u32(&sh->info_full[0]), 0, abort);
                        if (!ok) break;
                        const int from = first_window(info[0].vs, info[0].valid);
                        if (lane == 0) sh->e_low[warp] = from;
                        __syncwarp();
                    }
                }
            }
            ok = wait_at(smem_u32(&sh->q_full[buf]), (seg / q_bufs) & 1u, abort);
            if (!ok) break;
            const Walk& w = sh->seg[buf];
            uint8_t* sqb = sq + buf * L::kQTile;
            const bool both = !w.shared_rows(qt);
            const int nt = w.count(), nrows = w.rows(qt), row0 = w.first_row(qt);
            const int my = both ? s * kRows + row : row;        // row of the block
            const int token0 = row0 / t.group, rem0 = row0 - token0 * t.group;
            const bool any_row = (both ? s * kRows : 0) + quarter * 32 < nrows;  // this warp has rows
            const float cm = t.scale * kL2E * (kFp8 && any_row ? row_mul[buf * kRows + my] : 1.f);
            int token = 0, gq = 0;                              // this row's drafted token and head
            uint64_t bits = 0;
            if (my < nrows) {
                token = (int)a.group.divide(rem0 + my);
                gq = rem0 + my - token * t.group;
                token += token0;
                if (t.mask) bits = (uint64_t)__ldg(reinterpret_cast<const long long*>(t.mask) + w.r.lo + token);
            }
            float ref = -INFINITY, sum = 0.f;
            if (kFp8 && lane == 0) sh->e_eff[warp] = kFar;
            const int step = both ? 1 : 2;
            int b = 0;
            for (int tl = both ? 0 : s; ok && tl < nt; tl += step, b ^= 1) {
                const uint32_t ti = tile0 + tl, ts = tmem + lanes + s * 128 + b * kTile;
                const Info* inf = info + ti % kInfo;
                ok = wait_at(smem_u32(&sh->info_full[ti % kInfo]), (ti / kInfo) & 1u, abort) &&
                     wait_at(smem_u32(&sh->s_full[s][b]), (ph >> b) & 1u, abort);
                if (!ok) break;
                ph ^= 1u << b;
                tc_fence_after();
                const int kb = (w.k0 + tl) * kTile;             // first position of the tile
                const bool drafted = kb + kTile > w.r.p0;
                const uint2 valid = *reinterpret_cast<const uint2*>(inf->valid);
                const bool masked = drafted || (valid.x & valid.y) != ~0u;
                if (masked) {
                    // V rows of positions that do not exist are zeroed (another slot's row was loaded);
                    // elements of drafted tokens that are not finite too, and added to the rows that
                    // see them at the end
                    // (S of tile ti is there, so V of tile ti - 4 has been used: with four stages the parity
                    // of V's barrier says which phase it is; a shorter ring has a counter beside it)
                    const uint32_t st = ti % stages;
                    if constexpr (stages >= 4)
                        ok = wait_at(smem_u32(&sh->full[1][st]), (ti / stages) & 1u, abort);
                    else
                        ok = __all_sync(0xffffffffu, wait_past(&sh->v_done[ti & 1], (int)ti, abort));
                    if (!ok) break;
                    const int key = row & (kTile - 1);          // two threads a key
                    const bool gone = !(((key & 32 ? valid.y : valid.x) >> (key & 31)) & 1u);
                    if (gone || kb + key >= w.r.p0) {
                        uint8_t* v = ring + (stages + st) * L::kStage;
                        constexpr uint32_t kExp = std::is_same<TO, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
                        bool found = false;
#pragma unroll 1
                        for (int c = row / kTile; c < t.c.dim / 8; c += 2) {
                            uint4* at = reinterpret_cast<uint4*>(v + chunk_at<kBlock>(key, c));
                            const uint4 x = *at;
                            uint32_t xw[4] = {x.x, x.y, x.z, x.w};
                            bool here = gone;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (gone || (xw[i] & kExp) == kExp) {
                                    xw[i] &= 0xFFFF0000u;
                                    here = true;
                                }
                                if (gone || (xw[i] & (kExp << 16)) == (kExp << 16)) {
                                    xw[i] &= 0xFFFFu;
                                    here = true;
                                }
                            }
                            if (here) *at = make_uint4(xw[0], xw[1], xw[2], xw[3]);
                            found |= here;
                        }
                        if (found && !gone) *(volatile int*)&sh->odd[seg & 1] = 1;
                    }
                }
                if (any_row) {
                    // this row's 64 scores stay in registers: one read of TMEM
                    uint32_t v[2][32];
                    tmem_ld32(ts, v[0]);
                    tmem_ld32(ts + 32, v[1]);
                    uint32_t vis[2] = {~0u, ~0u};
                    bool far = false;
                    [[maybe_unused]] int e_low = 0;
                    if constexpr (kFp8) {
                        e_low = *(volatile int*)&sh->e_low[warp];
                        const uint32_t x0 = __float_as_uint(fabsf(inf->vs[lane])) >> 23, x1 = __float_as_uint(fabsf(inf->vs[32 + lane])) >> 23;
                        const uint32_t out0 = __ballot_sync(0xffffffffu, x0 - (uint32_t)e_low > (uint32_t)kNear) & valid.x,
                                       out1 = __ballot_sync(0xffffffffu, x1 - (uint32_t)e_low > (uint32_t)kNear) & valid.y;
                        far = (out0 | out1) != 0;
                    }
                    if (masked) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int pos = kb + 32 * i;
                            const int n = (t.mask ? w.r.p0 : w.r.p0 + token + 1) - pos;
                            uint32_t m = n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u);
                            if (t.mask) {
                                const int d = pos - w.r.p0;     // drafted token of the word's first bit
                                if (d >= 0)
                                    m |= d < 64 ? (uint32_t)(bits >> d) : 0u;
                                else if (d > -32)
                                    m |= (uint32_t)(bits << -d);
                            }
                            vis[i] = m & (i ? valid.y : valid.x);
                        }
                    }
                    if constexpr (kFp8) {
                        if (far) {
                            tmem_wait_ld(v[0]);
                            tmem_wait_ld(v[1]);
                            const FarResult r = far_unit(ts, to, t.c.dim, cm, make_uint2(vis[0], vis[1]), *inf, ref, sum, e_low, sh,
                                                         tl >= step ? &sh->s_free[s][b ^ 1] : nullptr, ((ph >> (b ^ 1)) & 1u) ^ 1u);
                            ref = r.ref;
                            sum = r.sum;
                            ok = r.e_low >= 0;
                            if (lane == 0) sh->e_low[warp] = r.e_low;
                            __syncwarp();
                            if (!ok) break;
                        }
                    }
                    if (!kFp8 || !far) {
                        float mx[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            tmem_wait_ld(v[c]);
                            if constexpr (kFp8) {
#pragma unroll
                                for (int j = 0; j < 32; j += 4) {
                                    const float4 k4 = *reinterpret_cast<const float4*>(&inf->ks[c * 32 + j]);
                                    const float2 lo = __fmul2_rn(make_float2(__uint_as_float(v[c][j]), __uint_as_float(v[c][j + 1])),
                                                                 make_float2(k4.x, k4.y));
                                    const float2 hi = __fmul2_rn(make_float2(__uint_as_float(v[c][j + 2]), __uint_as_float(v[c][j + 3])),
                                                                 make_float2(k4.z, k4.w));
                                    v[c][j] = __float_as_uint(lo.x);
                                    v[c][j + 1] = __float_as_uint(lo.y);
                                    v[c][j + 2] = __float_as_uint(hi.x);
                                    v[c][j + 3] = __float_as_uint(hi.y);
                                }
                            }
                            if (masked) {
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (!((vis[c] >> j) & 1u)) v[c][j] = 0xFF800000u;
                            }
                            float a0 = -INFINITY, a1 = -INFINITY;
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                a0 = fmaxf(a0, fmaxf(__uint_as_float(v[c][j]), __uint_as_float(v[c][j + 1])));
                                a1 = fmaxf(a1, fmaxf(__uint_as_float(v[c][j + 2]), __uint_as_float(v[c][j + 3])));
                            }
                            mx[c] = fmaxf(a0, a1);
                        }
                        float target = fmaxf(mx[0], mx[1]) * cm;
                        if constexpr (kFp8) {
                            target += (float)(e_low + kNear - 126) - kHalfRoom;
                        } else if constexpr (std::is_same<TO, __half>::value) {
                            target -= kHalfRoom;
                        }
                        if (__any_sync(0xffffffffu, target > ref + (std::is_same<TO, __half>::value ? kHalfSlack : kSlack))) {
                            const float to_ref = fmaxf(ref, target);
                            if (tl >= step) {                       // the accumulator holds something
                                ok = __all_sync(0xffffffffu, wait_or_abort(&sh->s_free[s][b ^ 1], ((ph >> (b ^ 1)) & 1u) ^ 1u, abort));
                                if (!ok) break;
                                tc_fence_after();
                                const float f = ref == -INFINITY ? 1.0f : ex2(ref - to_ref);
                                sum *= f;
#pragma unroll 1
                                for (int c = 0; c < t.c.dim; c += 32) {
                                    uint32_t o[32];
                                    tmem_ld32(to + c, o);
                                    tmem_wait_ld(o);
#pragma unroll
                                    for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                                    tmem_st32(to + c, o);
                                }
                            }
                            ref = to_ref;
                        }
                        const float nref = ref == -INFINITY ? 0.f : -ref;
                        const float2 cm2 = make_float2(cm, cm), nref2 = make_float2(nref, nref);
                        float2 part0 = make_float2(0.f, 0.f), part1 = part0;
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint32_t p[16];
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                float2 lo = __ffma2_rn(make_float2(__uint_as_float(v[c][j]), __uint_as_float(v[c][j + 1])), cm2, nref2);
                                float2 hi = __ffma2_rn(make_float2(__uint_as_float(v[c][j + 2]), __uint_as_float(v[c][j + 3])), cm2, nref2);
                                lo = make_float2(ex2(lo.x), ex2(lo.y));
                                hi = make_float2(ex2(hi.x), ex2(hi.y));
                                part0 = __fadd2_rn(part0, lo);
                                part1 = __fadd2_rn(part1, hi);
                                if constexpr (kFp8) {
                                    const float4 v4 = *reinterpret_cast<const float4*>(&inf->vs[c * 32 + j]);
                                    lo = __fmul2_rn(lo, make_float2(v4.x, v4.y));
                                    hi = __fmul2_rn(hi, make_float2(v4.z, v4.w));
                                }
                                p[j / 2] = pack2(lo.x, lo.y, TO());
                                p[j / 2 + 1] = pack2(hi.x, hi.y, TO());
                            }
                            tmem_st16(ts + c * 16, p);              // over scores that have been read
                        }
                        sum += (part0.x + part0.y) + (part1.x + part1.y);
                        tmem_wait_st();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->p_full[s][b]);
            }
            // ---- the segment's result
            if (tid == 0) sh->odd[(seg + 1) & 1] = 0;
            ok = __all_sync(0xffffffffu, ok && wait_or_abort(&sh->o_full, seg & 1u, abort));
            if (!ok) break;
            tc_fence_after();
            float2* swap = reinterpret_cast<float2*>(sqb);      // [2][128]: Q has been used
            if (!both) swap[s * kRows + row] = make_float2(ref, sum);
            join();
            if (!ok) break;
            float f0 = 1.f, f1 = 0.f;                           // factors of the two accumulators
            if (!both) {
                float2 x = swap[row];
                ref = x.x;
                sum = x.y;
                if (nt > 1) {
                    float2 y = swap[kRows + row];
                    if constexpr (kFp8) {
                        // references further apart than one factor bridges
                        if (any_row && __any_sync(0xffffffffu, fabsf(x.x - y.x) > kReach)) {
                            const float4 xy = bring_nearer(tmem + lanes + 256, s * (DP / 2), min((s + 1) * (DP / 2), t.c.dim), x, y);
                            x = make_float2(xy.x, xy.y);
                            y = make_float2(xy.z, xy.w);
                        }
                    }
                    ref = fmaxf(x.x, y.x);
                    f0 = ref == -INFINITY ? 1.f : ex2(x.x - ref);
                    f1 = ref == -INFINITY ? 1.f : ex2(y.x - ref);
                    sum = x.y * f0 + y.y * f1;
                }
            }
            const bool odd = *(volatile int*)&sh->odd[seg & 1] != 0;
            join();                                             // the exchange area is about to be reused
            if (!ok) break;
            const bool whole = w.k0 == 0 && w.k1 == w.tiles;
            if (any_row) {
                const long long slot = 2 * blockIdx.x + (w.k0 == 0 ? 1 : 0);
                const int per = kRows * qt;
                float4* po = a.part_o + slot * (DP / 4) * per + my;
                uint8_t* so = sqb + (my >> 7) * L::kQTile;
                const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                const int c0 = both ? 0 : s * (DP / 2), c1 = both ? DP : c0 + DP / 2;
                if (kFp8 && odd) add_nan(a, w, tmem + lanes + 256 + (both ? s * 128 : 0), c0, min(c1, t.c.dim), token, bits, my < nrows);
#pragma unroll 1
                for (int c = c0; c < c1 && c < t.c.dim; c += 32) {
                    uint32_t v[32];
                    tmem_ld32(tmem + lanes + 256 + (both ? s * 128 : 0) + c, v);
                    if (!both && nt > 1) {
                        uint32_t y[32];
                        tmem_ld32(tmem + lanes + 256 + 128 + c, y);
                        tmem_wait_ld(v);
                        tmem_wait_ld(y);
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            v[j] = __float_as_uint(__uint_as_float(v[j]) * f0 + __uint_as_float(y[j]) * f1);
                    } else {
                        tmem_wait_ld(v);
                    }
                    if (!kFp8 && odd && my < nrows) {
                        const int pages = (int)(t.c.slots / t.page_size);
                        const int n0 = max(max(0, w.k0 * kTile - w.r.p0), -w.r.p0), n1 = min(w.r.len, w.k1 * kTile) - w.r.p0;
                        for (int j = n0; j < n1; ++j) {
                            if (!(t.mask ? j < 64 && ((bits >> j) & 1) : j <= token)) continue;
                            const int pos = w.r.p0 + j;
                            const int page = __ldg(t.table + (long long)w.b * t.table_stride + pos / t.page_size);
                            if (page < 0 || page >= pages) continue;
                            const long long at = (long long)(page * t.page_size + pos % t.page_size) * t.c.slot_stride +
                                                 (long long)w.h * t.c.head_stride + c;
#pragma unroll
                            for (int d = 0; d < 32; ++d) {
                                if (c + d >= t.c.dim) break;
                                float x = (float)static_cast<const TQ*>(t.c.v)[at + d];
                                if (fabsf(x) < __int_as_float(0x7f800000)) x = 0.f;
                                v[d] = __float_as_uint(__uint_as_float(v[d]) + x);
                            }
                        }
                    }
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            uint32_t p[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                p[i] = pack2(__uint_as_float(v[j + 2 * i]) * inv, __uint_as_float(v[j + 2 * i + 1]) * inv, TQ());
                            *reinterpret_cast<uint4*>(so + chunk_at<kQBlock>(row, (c + j) / 8)) = make_uint4(p[0], p[1], p[2], p[3]);
                        }
                    } else if (my < nrows) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            po[(c + j) / 4 * per] = make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]),
                                                                __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
                    }
                }
                if (my < nrows && (both || s == 0)) {
                    if (!whole)
                        a.part_ml[slot * per + my] = make_float2(ref, sum);
                    else if (t.lse)
                        t.lse[(long long)(w.r.lo + token) * t.q_heads + w.h * t.group + gq] =
                            sum == 0.f ? -INFINITY : (ref + log2f(sum)) * kLn2;
                }
            }
            tc_fence_before();
            join();                                             // TMEM has been read, rows are staged
            if (!ok) break;
            if (whole) {
                // rows leave through shared memory, 16 bytes a thread and whole rows a warp
                const int sub = tid % kLanes;
                if (sub * 8 < t.c.dim) {
                    TQ* out = static_cast<TQ*>(t.out) + (long long)(w.r.lo + token0) * t.out_token_stride +
                              (long long)(w.h * t.group) * t.out_head_stride + sub * 8;
#pragma unroll 4
                    for (int r = tid / kLanes; r < nrows; r += kStep) {
                        const int i = (int)a.group.divide(rem0 + r);
                        *reinterpret_cast<uint4*>(out + i * t.out_token_stride + (rem0 + r - i * t.group) * t.out_head_stride) =
                            *reinterpret_cast<const uint4*>(sqb + (r >> 7) * L::kQTile + chunk_at<kQBlock>(r & 127, sub));
                    }
                }
            }
            tile0 += nt;
            ++seg;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->q_free[buf]);
        } while (tile0 < (uint32_t)count);
    }

    __syncthreads();
    if (warp == 0 && *abort) give_up(a, sh);
    if (warp == kScoreWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh->tmem) : "memory");
    }
}

// ---- joining the parts of an item ------------------------------------------------------------
// CTAs first..last hold parts of an item; the blocks (first + 1..last, y) share its rows and
// columns, four columns a thread, rows adjacent as the parts have them.
constexpr int kCombineThreads = 128;

template <typename TQ, int DP>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const __grid_constant__ KernelArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Split sp = a.splits[blockIdx.x];
    if (!sp.valid) return;
    const TreeAttnArgs& t = a.t;
    const Request r = request_of(t, a.qt, sp.b);
    const int row0 = sp.block * kRows * a.qt, nrows = min(r.rows - row0, kRows * a.qt);
    const int parts = sp.last - sp.first + 1, per = kRows * a.qt;
    const int workers = (parts - 1) * gridDim.y * kCombineThreads;
    for (int u = (((int)blockIdx.x - sp.first - 1) * gridDim.y + blockIdx.y) * kCombineThreads + threadIdx.x;
         u < nrows * (t.c.dim / 4); u += workers) {
        const int c4 = u / nrows, row = u - c4 * nrows;
        const float2* ml = a.part_ml + row;
        const float4* po = a.part_o + c4 * per + row;
        auto slot_of = [&](int p) { return (long long)(2 * (sp.first + p) + (p == 0)); };
        float top = -INFINITY;
#pragma unroll 4
        for (int p = 0; p < parts; ++p) top = fmaxf(top, __ldcg(ml + slot_of(p) * per).x);
        float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int p = 0; p < parts; ++p) {
            const float2 m = __ldcg(ml + slot_of(p) * per);
            const float4 x = __ldcg(po + slot_of(p) * (DP / 4) * per);
            // in two factors, as references may lie further apart than one bridges (see kReach)
            const float d = top == -INFINITY ? 0.f : m.x - top, near = fmaxf(d, -kReach), f = ex2(near), g = ex2(d - near);
            sum = fmaf(m.y * g, f, sum);
            acc[0] = fmaf(x.x * g, f, acc[0]);
            acc[1] = fmaf(x.y * g, f, acc[1]);
            acc[2] = fmaf(x.z * g, f, acc[2]);
            acc[3] = fmaf(x.w * g, f, acc[3]);
        }
        const int token = (row0 + row) / t.group;
        const long long qrow = r.lo + token;
        const int hq = sp.h * t.group + (row0 + row) - token * t.group;
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        TQ* out = static_cast<TQ*>(t.out) + qrow * t.out_token_stride + hq * t.out_head_stride + 4 * c4;
        *reinterpret_cast<uint2*>(out) =
            make_uint2(pack2(acc[0] * inv, acc[1] * inv, TQ()), pack2(acc[2] * inv, acc[3] * inv, TQ()));
        if (c4 == 0 && t.lse) t.lse[qrow * t.q_heads + hq] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
}

// ---- host side ---------------------------------------------------------------------------------

Divisor divisor(uint32_t d) {
    int l = 0;
    while ((1ull << l) < d) ++l;
    const uint64_t mul = ((((1ull << l) - d) << 32) / d) + 1;
    return {(uint32_t)mul, l < 1 ? l : 1, l > 1 ? l - 1 : 0};
}

int q_tiles(int group, int width) { return (long long)group * width > kRows ? 2 : 1; }
int padded_dim(int dim) { return dim <= 64 ? 64 : 128; }

bool joins(const TreeAttnArgs& t) { return (long long)t.max_pages * t.page_size > kTile; }   // items of one tile are never cut

constexpr size_t kSplitBytes = sizeof(Split) * kMaxCtas;
constexpr size_t kMlBytes(int qt) { return sizeof(float2) * 2 * kMaxCtas * kRows * qt; }

template <typename TQ, bool kFp8, int DP>
int launch(const KernelArgs& a, int sms, cudaStream_t st) {
    using L = Layout<DP, kFp8>;
    auto kern = attn_kernel<TQ, kFp8, DP>;
    const size_t smem = L::smem();
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return kLaunchFailed;
    const int grid = sms < kMaxCtas ? sms : kMaxCtas;
    kern<<<grid, kThreads, smem, st>>>(a);
    if (cudaGetLastError() != cudaSuccess) return kLaunchFailed;
    if (!joins(a.t)) return kOk;
    cudaLaunchConfig_t cfg = {};
    // two units of four columns a thread where an item is cut in two
    const long long rows = (long long)a.t.group * a.t.width;
    const long long units = (rows < kRows * a.qt ? rows : kRows * a.qt) * (a.t.c.dim / 4);
    cfg.gridDim = dim3(grid, (unsigned)((units + 2 * kCombineThreads - 1) / (2 * kCombineThreads)));
    cfg.blockDim = dim3(kCombineThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, combine_kernel<TQ, DP>, a) == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace attn

static std::atomic<int> g_wait_us{2000000}, g_hold{-1};
void tree_attn_waits(int wait_us, int hold) {
    g_wait_us = wait_us;
    g_hold = hold;
}

size_t tree_attn_workspace_bytes(int q_heads, int kv_heads, int dim, int width) {
    const int qt = attn::q_tiles(q_heads / kv_heads, width);
    return attn::kSplitBytes + attn::kMlBytes(qt) +
           sizeof(float) * 2 * attn::kMaxCtas * attn::kRows * qt * attn::padded_dim(dim);
}

int tree_attn_kernels(const TreeAttnArgs& t) { return attn::joins(t) ? 2 : 1; }

int launch_tree_attn(const TreeAttnArgs& t, int dtype, cudaStream_t st) {
    using namespace attn;
    KernelArgs a = {};
    a.t = t;
    a.qt = q_tiles(t.group, t.width);
    a.page = divisor((uint32_t)t.page_size);
    a.group = divisor((uint32_t)t.group);
    a.pages = (int)(t.c.slots / t.page_size);
    a.wait_us = g_wait_us;
    a.hold = g_hold;
    char* ws = static_cast<char*>(t.ws);
    a.splits = reinterpret_cast<Split*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + kSplitBytes);
    a.part_o = reinterpret_cast<float4*>(ws + kSplitBytes + kMlBytes(a.qt));
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return kLaunchFailed;
    const bool fp8 = t.c.dtype == kE4m3, wide = padded_dim(t.c.dim) == 128;
    if (dtype == kBf16) {
        if (fp8) return wide ? launch<__nv_bfloat16, true, 128>(a, sms, st) : launch<__nv_bfloat16, true, 64>(a, sms, st);
        return wide ? launch<__nv_bfloat16, false, 128>(a, sms, st) : launch<__nv_bfloat16, false, 64>(a, sms, st);
    }
    if (fp8) return wide ? launch<__half, true, 128>(a, sms, st) : launch<__half, true, 64>(a, sms, st);
    return wide ? launch<__half, false, 128>(a, sms, st) : launch<__half, false, 64>(a, sms, st);
}

}  // namespace dsv
