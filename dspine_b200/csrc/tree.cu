// tree.cu -- greedy acceptance over draft trees (sm_100a).
//
// The tree form of greedy_kernel (small.cu; verification/caps.py:32-59 _accept_capped): request b
// has up to 64 drafted nodes, node 0 the root (the last committed token) and every parent before
// its children.  Bit j of mask[i] says that node j is node i or an ancestor of it; the parent is
// the highest bit below i.  Node i agrees when its token is the target's top-1 token at its
// parent, and is accepted when it and all its ancestors agree.  The deepest accepted node (the
// lowest index among equals) ends the accepted path; the bonus token is the top-1 token there.
//
//   accept_kernel   one warp per request, two nodes per lane: the agreement of all nodes is one
//                   64-bit ballot, after which "all ancestors agree" is one AND per node, so no
//                   walk over the tree is needed.  The cost is the latency of two dependent loads: 256
//                   trees of up to 64 nodes take as long as 4 of 16 (26 us as called from Python,
//                   nearly all of it the host's).
#include <cuda_runtime.h>
#include <stdint.h>

#include "dsv_common.cuh"
#include "dsv_kernels.h"

namespace dsv {
namespace tree {

constexpr int kWarps = 4;

__global__ void __launch_bounds__(kWarps * 32) accept_kernel(TreeAcceptArgs a) {
    const int b = blockIdx.x * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (b >= a.batch) return;
    long long lo, hi;
    if (a.indptr) {
        lo = a.indptr[b];
        hi = a.indptr[b + 1];
        lo = lo < 0 ? 0 : (lo > a.rows ? a.rows : lo);
        hi = hi < lo ? lo : (hi > a.rows ? a.rows : hi);
    } else {
        lo = (long long)b * a.nodes;
        hi = lo + a.nodes;
    }
    int n = (int)(hi - lo < 64 ? hi - lo : 64);
    if (n > a.width) n = a.width;  // a path has at most `width` nodes
    uint64_t up[2];                // ancestors and itself
    int64_t tok[2], top[2];
    bool agree[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = lane + 32 * k;
        up[k] = 0;
        tok[k] = top[k] = 0;
        agree[k] = false;
        if (i < n) {
            tok[k] = a.tokens[lo + i];
            top[k] = a.top1[lo + i];
            up[k] = ((uint64_t)a.mask[lo + i] & ((1ull << i) - 1ull)) | (1ull << i);
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = lane + 32 * k;
        const uint64_t above = up[k] & ~(1ull << i);
        const int parent = above ? 63 - __clzll((long long)above) : 0;
        const int64_t t0 = __shfl_sync(0xffffffffu, top[0], parent & 31);
        const int64_t t1 = __shfl_sync(0xffffffffu, top[1], parent & 31);
        agree[k] = i < n && (i == 0 || (above != 0 && tok[k] == (parent < 32 ? t0 : t1)));
    }
    const uint64_t good = (uint64_t)__ballot_sync(0xffffffffu, agree[0]) |
                          ((uint64_t)__ballot_sync(0xffffffffu, agree[1]) << 32);
    int best = -1;  // depth * 64 + (63 - node): deepest first, then the lowest index
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = lane + 32 * k;
        if (i < n && (up[k] & 1ull) && (up[k] & ~good) == 0)
            best = max(best, __popcll(up[k]) * 64 + (63 - i));
    }
    best = __reduce_max_sync(0xffffffffu, best);
    const int node = best < 0 ? -1 : 63 - (best & 63);
    const int src = node < 0 ? 0 : node & 31;
    const uint64_t p0 = __shfl_sync(0xffffffffu, up[0], src), p1 = __shfl_sync(0xffffffffu, up[1], src);
    const int64_t b0 = __shfl_sync(0xffffffffu, top[0], src), b1 = __shfl_sync(0xffffffffu, top[1], src);
    const uint64_t on = node < 0 ? 0ull : (node < 32 ? p0 : p1);
    const int64_t bonus = node < 0 ? -1 : (node < 32 ? b0 : b1);
    const int commit = __popcll(on);
    const long long row = (long long)b * a.width;
    // node i of the path is entry r = (nodes of the path before it); its token is output r - 1
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = lane + 32 * k;
        if (i < n && ((on >> i) & 1ull)) {
            const int r = __popcll(on & ((1ull << i) - 1ull));
            a.path[row + r] = i;
            if (a.kept) a.kept[row + r] = a.slots[lo + i];
            if (r > 0) a.output[row + r - 1] = tok[k];
        }
    }
    for (int r = lane; r < a.width; r += 32) {
        if (r >= commit) {
            a.path[row + r] = -1;
            if (a.kept) a.kept[row + r] = -1;
            a.output[row + r] = 0;
        }
    }
    if (lane == 0) {
        if (commit > 0) a.output[row + commit - 1] = bonus;
        a.accept[b] = commit > 0 ? commit - 1 : 0;
        a.commit[b] = commit;
        a.bonus[b] = bonus;
        a.new_seq[b] = (a.prefix ? a.prefix[b] : 0) + commit;
    }
}

}  // namespace tree

int launch_tree_accept(const TreeAcceptArgs& a, cudaStream_t st) {
    tree::accept_kernel<<<(a.batch + tree::kWarps - 1) / tree::kWarps, tree::kWarps * 32, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? kOk : kLaunchFailed;
}

}  // namespace dsv
