// Drafted trees, the two ends of a step: masks, rotary positions and slots from parents (p1a_tree_rows), and the accepted path moved behind node 0 in every
// layer (p1a_tree_commit). Both move next to nothing; what they cost is a launch and as many round trips to memory as depend on each other: 1.8 us for eight nodes, 4.0 for 64
// sequences of 33 ... 256; 3.4 us for one sequence's path in 16 layers, 4.6 for 32 sequences' (9.7 MB, 2.1 TB/s).
#include "p1a_tiles.hpp"

#include <algorithm>

namespace p1a {
namespace {

constexpr int RTHR = 256;

// A workgroup per sequence: parents into LDS, then every row climbs from its node. Parents come before their children, so a climb passes the words of its
// mask from the last to the first and each is finished when it is left.
__global__ void __launch_bounds__(RTHR) rows_k(const int32_t * parent, const rows_view R, uint32_t * mask, int words, int32_t * pos, int32_t * slot) {
    __shared__ int16_t up[P1A_TREE_NODES];
    const seq_view v = seq_of<true>(R, blockIdx.x);
    const int n = min(v.count, P1A_TREE_NODES);
    for (int i = threadIdx.x; i < n; i += RTHR) {
        const int p = parent[v.first + i];
        up[i] = (int16_t) (p >= 0 && p < i ? p : -1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += RTHR) {
        const size_t row = (size_t) v.first + i;
        int j = i, depth = -1;
        for (int w = words - 1; w >= 0; --w) {
            uint32_t bits = 0;
            while (j >= 0 && j >> 5 == w) {
                bits |= 1u << (j & 31);
                j = up[j];
                ++depth;
            }
            mask[row * words + w] = bits;
        }
        if (pos) pos[row] = v.pos0 + depth;
        if (slot) slot[row] = v.pos0 + i;
    }
}

// A workgroup per (layer, K or V, sequence); a thread has W bytes of a row to itself and moves them for one accepted node after the other, eight asked for at a time.
// A slot only ever receives what stood behind it, and the rows of later nodes stand behind every slot that is written before they are read: no copy, and nothing
// waits but a thread for its own loads. Lane k of each wave looks up where node k of the path is and where it goes.
template <int W> struct word_of;
template <> struct word_of<16> { typedef u4 type; };
template <> struct word_of<8> { typedef u2w type; };
template <> struct word_of<4> { typedef uint32_t type; };
template <> struct word_of<2> { typedef uint16_t type; };

struct commit_params {
    const int32_t * n_accept, * path;
    kv_view pg;
    rows_view R;
    int ld_path, words;
    char * at[2 * P1A_TREE_LAYERS];                         // K of the layers, then V
};
constexpr int CTHR = 256, AHEAD = 8;

template <int W> __global__ void __launch_bounds__(CTHR) commit_k(const commit_params P) {
    typedef typename word_of<W>::type word;
    typedef __attribute__((address_space(1))) word * gword;
    const int s = blockIdx.x % P.R.n_seq, which = blockIdx.x / P.R.n_seq, lane = threadIdx.x & 63;
    const int n = min(max(sload_i32(P.n_accept + s), 0), P.ld_path);
    if (n < 1) return;
    const seq_view v = seq_of<true>(P.R, s);
    const int32_t * const ptab = P.pg.pt ? P.pg.pt + (P.pg.rtab ? sload_i32(P.pg.rtab + s) : 0) : nullptr;
    char * const base = P.at[which];
    const int32_t * const path = P.path + (size_t) s * P.ld_path;
    for (int k0 = 0; k0 < n; k0 += 64) {
        const int k = k0 + lane, node = k < n ? path[k] : -1, from = v.pos0 + node, to = v.pos0 + 1 + k;
        const bool go = node > k + 1 && node < v.count && to >= 0 && from < P.R.n_ctx;
        const size_t src = go ? kv_off_tab(P.pg, ptab, from) : 0, dst = go ? kv_off_tab(P.pg, ptab, to) : 0;
        const unsigned long long all = __ballot(go);
        for (int w = threadIdx.x; w < P.words; w += CTHR) {
            unsigned long long left = all;
            while (left) {
                word x[AHEAD];
                size_t off[AHEAD];
                int m = 0;
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    if (!left) break;
                    const int l = __builtin_ctzll(left);
                    left &= left - 1;
                    const size_t f = (size_t) (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) src, l) | (size_t) (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (src >> 32), l) << 32;
                    off[a] = (size_t) (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) dst, l) | (size_t) (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (dst >> 32), l) << 32;
                    x[a] = *(gword) (base + f + (size_t) w * W);
                    m = a + 1;
                }
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) if (a < m) *(gword) (base + off[a] + (size_t) w * W) = x[a];
            }
        }
    }
}

}   // namespace

int launch_tree_rows(const int32_t * parent, const rows_view & R, uint32_t * mask, int words, int32_t * pos, int32_t * slot, hipStream_t s) {
    rows_k<<<R.n_seq, RTHR, 0, s>>>(parent, R, mask, words, pos, slot);
    return launched();
}

int launch_tree_commit(const p1a_kv * layers, int n_layers, const rows_view & R, const int32_t * n_accept, const int32_t * path, int ld_path, hipStream_t s) {
    commit_params P;
    P.n_accept = n_accept; P.path = path; P.pg = view_of(layers[0]); P.R = R; P.ld_path = ld_path;
    size_t al = P.pg.rowb | (layers[0].pt ? layers[0].pstride : 0);
    for (int i = 0; i < n_layers; ++i) {
        P.at[i] = (char *) layers[i].k;
        P.at[n_layers + i] = (char *) layers[i].v;
        al |= (size_t) layers[i].k | (size_t) layers[i].v;
    }
    const int W = al & 15 ? al & 7 ? al & 3 ? 2 : 4 : 8 : 16;
    P.words = (int) (P.pg.rowb / W);
    const unsigned grid = (unsigned) R.n_seq * 2 * n_layers;
    if (W == 16) commit_k<16><<<grid, CTHR, 0, s>>>(P);
    else if (W == 8) commit_k<8><<<grid, CTHR, 0, s>>>(P);
    else if (W == 4) commit_k<4><<<grid, CTHR, 0, s>>>(P);
    else commit_k<2><<<grid, CTHR, 0, s>>>(P);
    return launched();
}

}   // namespace p1a
