// Attention of the rows of drafted trees - per sequence a few to a thousand nodes, each of which sees what is in front of the tree and its own path - over
// paged caches: p1a_attn_tree.
//
// Work: a column is one q head of a node's row. Where sequences have up to 32 columns under a kv head (few_k) the four waves of a workgroup share the keys, each with
// tiles of 32 of its own; where they have more (team_k) the waves share tiles in LDS and take 32 columns each, up to 128 a group. Steps - 128 keys, or a tile - are
// counted through over all groups of all sequences, and a workgroup takes a run of them as long as every other's, whatever the lengths; a group that lies in one run
// is finished there, the others' partials are merged by tree_merge_k.
// Arithmetic: S^T = K Q^T and O^T = V^T P^T on f16 matrix instructions, one pass with a running reference of every column. With bf16 results q, P, K and V enter as one f16
// each, a quantized value times its scale; where results are f32 (EXACT) q and P are two halves and quantized K and V two planes (team_k) or whole numbers whose
// scales multiply fp32 results (K) or P (V; few_k), as in p1a_chunk.hip and p1a_step.hip.
// Only the last tiles hold nodes of the tree: there a column's 32 bits of its mask are shifted out of two words.
// What bounds it, on one MI355X (team_k in a row of calls, tree_merge_k's 9 ... 11 us behind it not counted; traced launch by launch 100, 192 and 73 us): one wave a SIMD with heads of 256,
// whose accumulators and q fill the registers. 63 nodes over 32768 keys (24 / 4 heads of 256, q8_0, bf16 results): 88 us, a tile of 32 keys in 1.7 us = 356 instructions and 32
// products of 32 clocks, some 9 clocks an instruction, 29 % of the waves' time waiting; 16 sequences of 4 ... 16 nodes over 300 ... 32768 keys with f32 results: 163 us, 2.2 us a tile, 1.4 of
// them the 96 products of a wave whose columns are all there, 45 % waiting. With heads of 128 two workgroups share a compute unit: 24 sequences of 3 ... 64 nodes over
// 500 ... 8000 keys (32 / 8 heads, f16) 70 us with the same inputs again, 83 and 3.4 TB/s with others, 45 % waiting. Where all of it is few_k: 16 sequences of 1 ... 5 nodes over 300 ... 32768 keys (24 / 4 of 256) 108 us
// (f16, 4.6 TB/s), 101 (q8_0, f32 results), 66 (q8_0, bf16). Built and not kept: two waves a SIMD that share
// columns, each with half of O (20 % slower: both make all of S), loads from LDS asked for further ahead with two planes (8 %), results through LDS to whole lines (11 %), a
// merge by four threads for one (24 sequences: 25 us for 9), eight waves for a sequence alone (nothing).
#include "p1a_tiles.hpp"

#include <algorithm>
#include <atomic>

namespace p1a {
namespace {

constexpr int NW = 4, NTHR = NW * 64;                         // waves
constexpr int COLS = 32 * NW;                                 // columns of a group of team_k

struct group_of { int cols, blocks, groups, bpg; };           // a sequence's columns under a kv head, blocks of BC of them, groups of at most `waves` blocks, a group's blocks
__host__ __device__ __forceinline__ group_of groups_of(int rows, int GQA, int BC, int waves) {
    group_of s;
    s.cols = rows * GQA;
    s.blocks = (s.cols + BC - 1) / BC;
    s.groups = (s.blocks + waves - 1) / waves;
    s.bpg = s.groups ? (s.blocks + s.groups - 1) / s.groups : 1;
    return s;
}

struct tree_params : chunk_params {
    const uint32_t * mask;                                    // [T][words]
    int words, max_groups;
};

// ---- runs of steps of equal length over the groups of all sequences (lane i of a wave counts for sequence s0 + i) ----
// BN: keys of a tile; TPS: tiles of a step; BC: columns of a block; WAVES: blocks of a group. A group counts SETUP steps more than it has: what it takes to find it, to ask for its first
// tiles and q and to write its results (24 sequences of 3 ... 64 nodes over 500 ... 8000 keys: workgroups with many short groups were still at work for 34 us when half of all had ended)
template <int BN, int TPS, int BC, int WAVES, int SETUP_> struct tree_runs {
    static constexpr int SETUP = SETUP_;
    // (shape: rows, up to P1A_TREE_NODES, and groups in one register - lanes keep all of this while they work)
    struct of_lane {
        int first, pos0, table, shape, per_group;
        __device__ __forceinline__ int steps() const { return per_group * (shape >> 11); }
    };
    static_assert(P1A_TREE_NODES < 1 << 11);
    of_lane first64;
    int first, end, per;
    static __device__ __forceinline__ span span_of_rows(const rows_view & R, const seq_view & v) { return span_of<BN>(R, v.pos0, v.pos0 + v.count - 1); }
    static __device__ __forceinline__ of_lane look(const rows_view & R, const kv_view & pg, int GQA, int s) {
        of_lane r{0, 0, 0, 0, 0};
        if (s >= R.n_seq) return r;
        const seq_view v = seq_of(R, s);
        r.table = pg.pt && pg.rtab ? pg.rtab[s] : 0;
        r.first = v.first;
        r.pos0 = v.pos0;
        if (v.count > 0) {
            r.per_group = SETUP + max((span_of_rows(R, v).nt + TPS - 1) / TPS, 1);
            r.shape = v.count | groups_of(v.count, GQA, BC, WAVES).groups << 11;
        }
        return r;
    }
    // run number `run` of `runs`, no group in more than `most_runs` of them. False: there is nothing for it
    __device__ __forceinline__ bool begin(const rows_view & R, const kv_view & pg, int GQA, int run, int runs, int most_runs) {
        const int lane = threadIdx.x & 63;
        first64 = look(R, pg, GQA, lane);
        int n = 0, most = 0;
        for (int s0 = 0; s0 < R.n_seq; s0 += 64) {
            const of_lane x = s0 ? look(R, pg, GQA, s0 + lane) : first64;
            n += __builtin_amdgcn_readlane(lanes_up_to(x.steps()), 63);
            most = max(most, x.per_group);
        }
        most = rfl((int) wave_max((float) most));             // (a group has 2^25 steps at most: the f32 next to it, 1 off in 2^24, only moves the cut)
        per = max((n + runs - 1) / runs, (most + most_runs - 2) / (most_runs - 1) + (most >> 23));
        first = run * per;
        end = min(first + per, n);
        return first < end;
    }
    // What of a group's steps, as found, is in this run: from .. to - 1 (counted without SETUP; nothing: to <= 0), which of its pieces that is and how many there are
    struct share { int from, to, piece, pieces; };
    template <class F> __device__ __forceinline__ share share_of(const F & f, int at, int run) const {
        const int lo = f.first + SETUP, run0 = lo / per;
        return share{max(at - lo, 0), min(end, f.first + f.steps) - lo, run - run0, (f.first + f.steps - 1) / per - run0 + 1};
    }
    // whose step `at` is: sequence, group, the group's first step, its steps (SETUP among them). False: nobody's (row0 or pos0 were written since begin())
    struct found { int seq, group, first, steps, table; seq_view v; };
    __device__ __forceinline__ bool find(const rows_view & R, const kv_view & pg, int GQA, int at, int lane, found & f) const {
        int base = 0;
        for (int s0 = 0; s0 < R.n_seq; s0 += 64) {
            const of_lane x = s0 ? look(R, pg, GQA, s0 + lane) : first64;
            const int u = base + lanes_up_to(x.steps());
            const unsigned long long behind = __ballot(u > at);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                f.seq = s0 + l;
                f.steps = __builtin_amdgcn_readlane(x.per_group, l);
                const int shape = __builtin_amdgcn_readlane(x.shape, l), start = __builtin_amdgcn_readlane(u, l) - f.steps * (shape >> 11);
                f.group = (at - start) / f.steps;
                f.first = start + f.group * f.steps;
                f.v.first = __builtin_amdgcn_readlane(x.first, l);
                f.v.count = shape & 2047;
                f.v.pos0 = __builtin_amdgcn_readlane(x.pos0, l);
                f.table = __builtin_amdgcn_readlane(x.table, l);
                return true;
            }
            base = __builtin_amdgcn_readlane(u, 63);
        }
        return false;
    }
};

// ---- 16 keys as the rows of a 16 x 32 operand, a quantized value times its scale ----
// Lane (key c = lane % 16, group g) holds D / 4 dims on end, so that the scales it needs are its own: step b of the product takes 8 of them.
template <uint32_t KT, int D> struct keysd {
    static constexpr int NB = D / 32, TAB = 0;
    static constexpr bool Q8 = KT == P1A_KV_Q8_0;
    static constexpr int NL = D / 64, NSC = D == 256 ? 2 : 1;   // 16-byte loads of codes (q8_0); scales of a lane
    typedef uint32_t u1_a2 __attribute__((aligned(2)));
    typedef u2w u2_a2 __attribute__((aligned(2)));
    struct raw { u4 w[Q8 ? NL : NSC]; uint32_t d; };           // (q4_0 of D = 64: half a block, 8 bytes)
    static __device__ __forceinline__ int dim(int b, int g, int half) {
        if constexpr (Q8) return g * (D / 4) + 8 * b + 4 * half;
        else if constexpr (D == 64) return 32 * (g >> 1) + 4 * (2 * (g & 1) + b) + 16 * half;
        else return 32 * (g * NSC + (b >> 2)) + 4 * (b & 3) + 16 * half;
    }
    static __device__ __forceinline__ void load(raw & r, gbytes row, int g) {
        if constexpr (Q8) {
            if constexpr (D == 256) r.d = gload<uint32_t>(row + 4 * g);
            else r.d = gload<uint16_t>(row + 2 * (D == 128 ? g : g >> 1));
#pragma unroll
            for (int j = 0; j < NL; ++j) r.w[j] = gload<u4_a4>(row + 2 * NB + g * (D / 4) + 16 * j);
        } else if constexpr (D == 64) {
            r.d = gload<uint16_t>(row + 18 * (g >> 1));
            const u2w t = gload<u2_a2>(row + 18 * (g >> 1) + 2 + 8 * (g & 1));
            r.w[0] = u4{t[0], t[1], 0, 0};
        } else {
            uint32_t d[NSC];
#pragma unroll
            for (int x = 0; x < NSC; ++x) {
                d[x] = gload<uint16_t>(row + 18 * (g * NSC + x));
                r.w[x] = gload<u4_a2>(row + 18 * (g * NSC + x) + 2);
            }
            r.d = NSC == 2 ? d[0] | d[NSC - 1] << 16 : d[0];
        }
    }
    static __device__ __forceinline__ h8 operand(const raw & r, int b) {
        const uint32_t s = NSC == 2 && b >= 4 ? r.d >> 16 : r.d & 0xffff;
        const h2 d = __builtin_bit_cast(h2, s | s << 16);
        uint32_t a[4];
        if constexpr (Q8) {
            times4<1>(r.w[b >> 1][2 * (b & 1)] ^ 0x80808080u, 1152.f, d, a, nullptr);
            times4<1>(r.w[b >> 1][2 * (b & 1) + 1] ^ 0x80808080u, 1152.f, d, a + 2, nullptr);
        } else {
            const uint32_t w = r.w[b >> 2][b & 3];
            times4<1>(w & 0x0f0f0f0fu, 1032.f, d, a, nullptr);
            times4<1>((w >> 4) & 0x0f0f0f0fu, 1032.f, d, a + 2, nullptr);
        }
        return __builtin_bit_cast(h8, u4{a[0], a[1], a[2], a[3]});
    }
};

template <uint32_t KT, int D, int NT, bool EXACT> struct few_cfg {
    static constexpr bool F16 = KT == P1A_KV_F16, CODES = EXACT && !F16;      // codes as whole numbers, scales outside of the products
    static constexpr int VT_B = 2 * plane_bytes(D);           // 32 keys of V
    static constexpr int V_B = (F16 ? 2 : 1) * VT_B;
    static constexpr int TAB = CODES ? keys16<KT, D>::TAB : 0;
    static constexpr int WAVE_B = V_B + 4 * TAB * 4;          // and the scales of 2 x 16 keys of K and V
    // (the low halves of q, where registers do not hold them: the same for every wave, each writes all of them)
    static constexpr bool QL = EXACT && (CODES || D == 128) && NT * D >= 256;
    static constexpr int QL_B = QL ? NT * D * 32 : 0, ML_B = NW * 2 * 16 * NT * 4;
    static constexpr bool ML_OVER = 4 * TAB * 4 >= ML_B;      // references and sums go where the first wave's scales were
    static_assert(D == 256 || 2 * NW * (WAVE_B + QL_B / NW + ML_B / NW) <= 160 * 1024, "two workgroups' LDS");
    static constexpr int ML_AT = ML_OVER ? V_B : NW * WAVE_B + QL_B, LDS = NW * WAVE_B + QL_B + (ML_OVER ? 0 : ML_B);
    static constexpr int WGS = D == 256 ? 1 : 2;              // workgroups of a compute unit
    static constexpr int PC = 16 * (D + 4) * 4 <= V_B ? 16 : 8;   // columns folded at a time, where V was
    static_assert(PC * (D + 4) * 4 <= V_B);
};

// bits `at` .. `at + 31` of a row's mask (at: from -31 on; what is not there is 0)
__device__ __forceinline__ uint32_t mask_bits(const uint32_t * row, int words, int at) {
    const int w = at >> 5;                                    // (-1 at the least)
    const uint32_t lo = w >= 0 && w < words ? row[w] : 0, hi = w + 1 < words ? row[w + 1] : 0;
    return __builtin_amdgcn_alignbit(hi, lo, at & 31);
}

// The kernel's arguments, read again from here on: kept in registers from the kernel's start to its end they and what follows from them are too many, and
// would be spilled to lanes of vector registers
typedef const __attribute__((address_space(4))) tree_params * args;
__device__ __forceinline__ const tree_params & read_again() {
    args p = (args) __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const tree_params *) p;
}

// What the row of a sequence's node `tok` sees of the 32 keys from k0 on: key j where (j <= hi && (j > lo || j < sk)) or bit j
struct sight { int hi, lo, sk; uint32_t bits; };
__device__ __forceinline__ sight sight_of(const tree_params & P, const seq_view & sv, int tok, int k0) {
    const int slot = sv.pos0 + tok, at = k0 - sv.pos0;
    const bool live = slot >= 0 && slot < P.R.n_ctx;
    const uint32_t * const row = P.mask + (size_t) (sv.first + tok) * P.words;
    sight v{live ? sv.pos0 - 1 - k0 : INT32_MIN / 2, -1 - k0, 0, 0};
    if (P.R.window != INT32_MAX) {                            // (its place: as many nodes behind the first as its path has)
        int nodes = 0;
        for (int w = 0; 32 * w < sv.count; ++w) nodes += __popc(sv.count - 32 * w >= 32 ? row[w] : row[w] & ((1u << (sv.count - 32 * w)) - 1));
        v.lo = sv.pos0 + max(nodes - 1, 0) - P.R.window - k0;
        v.sk = P.R.n_sink - k0;
    }
    if (live && at > -32) {
        const int left = min(sv.count, P.R.n_ctx - sv.pos0) - at;   // nodes that are there, in slots that are
        v.bits = mask_bits(row, P.words, at);
        v.bits = left >= 32 ? v.bits : left > 0 ? v.bits & ((1u << left) - 1) : 0;
    }
    return v;
}

// 1 / (1 + e^-g) by the hardware's exponential and reciprocal: (6 + 1.25 max(-g, 0)) 2^-24 of itself off - 2^-23 each for the two, 2^-24 for the sum; and what rounds g log2 e and log2 e itself
// moves the exponential by, 1.22 |g| 2^-24, of which a gate above 1/2 takes little. gate_of, 6 2^-24 off for any g, costs 13 us of 174 here (16 trees of 4 ... 16 nodes, q8_0, heads of
// 256), and taking the product's rounding back 3; down to gates of -80 that stays below 7e-6, within the 1e-5 that f32 results have.
__device__ __forceinline__ float tree_gate(float g) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -LOG2E)); }
// Four results of a row from its sums relative to M: a partial (piece >= 0) or what the call is to give
__device__ __forceinline__ void finish(const tree_params & P, size_t row, int d, int D, int piece, f4 acc, float M, float l) {
    if (piece >= 0) {
        if (d == 0) *reinterpret_cast<float2 *>(P.part_ml + (row * P.nks + piece) * 2) = float2{part_ref(M, l), l};
        if (part_ref(M, l) != MINUS_INF) *reinterpret_cast<f4 *>(P.part_o + (row * P.nks + piece) * D + d) = acc;
        return;
    }
    if (P.lse && d == 0) P.lse[row] = (M + log2f(l)) * LN2;
    f4 v = acc * (l == 0.f ? 0.f : 1.0f / l);                 // (nothing seen: 0)
    if (P.gate) {
        const f4 gt = *reinterpret_cast<const f4 *>(P.gate + row * D + d);
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] *= tree_gate(gt[y]);
    }
    put4(P.out, P.out_bf16, row * D + d, v);
}

template <uint32_t KT, int D, int NT, bool EXACT>
__global__ void __launch_bounds__(NTHR, (few_cfg<KT, D, NT, EXACT>::WGS)) few_k(const tree_params) {
    const tree_params & P0 = read_again();
    const int Hkv = P0.Hkv, runs = P0.runs;
    using C = few_cfg<KT, D, NT, EXACT>;
    constexpr bool F16 = C::F16, CODES = C::CODES;
    using K = typename std::conditional<F16 || CODES, keys16<KT, D>, keysd<KT, D>>::type;
    using G = group<KT, D, CODES ? 0 : 1>;
    constexpr int NB = D / 32, NDT = D / 16, NQ = EXACT ? 2 : 1, PL_B = plane_bytes(D);
    using runs_t = tree_runs<32, NW, 16 * NT, 1, 4>;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the kv heads of a run of steps, whose rows have cache lines in common, on one XCD
    const int xcd = blockIdx.x & 7, jx = blockIdx.x >> 3, hk = jx % Hkv, run = jx / Hkv * 8 + xcd;
    if (run >= runs) return;
    runs_t steps;
    steps.first = 0;
    steps.end = 1;
    steps.per = 1 << 30;
    if (P0.nks > 1 && !steps.begin(P0.R, P0.pg, P0.GQA, run, runs, P0.nks)) return;
    char * const mine = lds + wave * C::WAVE_B;
    float * const tk = reinterpret_cast<float *>(mine + C::V_B), * const tv = tk + 2 * C::TAB;
    const size_t head_off = (size_t) hk * head_bytes(KT, D);

  for (int at_step = steps.first; at_step < steps.end;) {
    const tree_params & P = read_again();
    auto tok_of = [&](int r) {
        const int t = (int) __umulhi((uint32_t) r, P.gqa_magic);
        return r - t * P.GQA >= P.GQA ? t + 1 : t;
    };
    // (the lane's number anew for each group: what follows from it would be worked out ahead of the loop and kept)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, c = lane & 15, g = lane >> 4;
    typename runs_t::found f;
    if (P.nks > 1) {
        if (!steps.find(P.R, P.pg, P.GQA, at_step, lane, f)) return;
    } else {                                                  // a sequence each
        f.seq = run; f.group = 0; f.first = 0; f.steps = 1;
        f.v = seq_of<true>(P.R, f.seq);
        f.table = P.pg.pt && P.pg.rtab ? sload_i32(P.pg.rtab + f.seq) : 0;
        if (f.v.count < 1) return;
    }
    const seq_view & sv = f.v;
    typename runs_t::share due{0, 1 << 26, 0, 1};
    if (P.nks > 1) due = steps.share_of(f, at_step, run);
    at_step = f.first + f.steps;
    if (due.to <= 0) continue;
    const int pieces = due.pieces, piece = due.piece;
    const int R = min(sv.count * P.GQA, 16 * NT);
    auto row_index = [&](int r) { const int t = tok_of(r); return (size_t) (sv.first + t) * P.Hq + (size_t) hk * P.GQA + (r - t * P.GQA); };
    const span sp = runs_t::span_of_rows(P.R, sv);
    const int ta = due.from * NW, tb = min(due.to * NW, sp.nt);
    // positions that all rows see
    const bool odd = sv.pos0 < 0 || sv.pos0 + sv.count > P.R.n_ctx;
    const int all_hi = odd ? -1 : sv.pos0 - 1, all_lo = P.R.window == INT32_MAX ? 0 : sp.pmax - P.R.window + 1;

    const key_rows keys{sp, P.pg, P.pg.pt ? P.pg.pt + f.table : nullptr, head_off, c};
    using where = key_rows::where;
    int vbase[2];                                             // V^T operand: dims 16 dt + lane % 16, keys 4 g .. of a group; for even and odd dt
    {
        const int kk = c >> 2, jq = c & 3;
#pragma unroll
        for (int e = 0; e < 2; ++e) vbase[e] = chunk_at(4 * g + kk, 2 * e + (jq >> 1)) + (jq & 1) * 8;
    }
    auto v_read = [&](const char * grp, int dt) {
        return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4 __attribute__((address_space(3))) *) (grp + vbase[dt & 1] + (dt >> 1) * 1024)));
    };
    struct none {};
    typename K::raw kr[2], kn[2];                             // K of the tile in hand, and of the next one
    typename std::conditional<F16, none, typename group<F16 ? P1A_KV_Q8_0 : KT, D, CODES ? 0 : 1>::raw>::type vr[2];
    typename keys16<KT, D>::scales vs[2];
    auto ask_k = [&](const where & w) {
#pragma unroll
        for (int x = 0; x < 2; ++x) K::load(kn[x], (gbytes) P.kc + w.off[x], g);
    };
    auto ask_v = [&](const where & w, int st) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if constexpr (F16) {                              // (this lane's part of the direct load belongs to another key)
                const size_t off = __shfl((unsigned long long) w.off[x], G::key(lane));
                G::load((gbytes) P.vc + off, mine + st * C::VT_B + x * PL_B, lane);
            } else {
                G::load(vr[x], (gbytes) P.vc + w.off[x], lane);
                if constexpr (CODES) keys16<KT, D>::load_scales(vs[x], (gbytes) P.vc + w.off[x], g);
            }
        }
    };

    // ---- q, the first tile, Q^T: columns 16 n + c. (Page-table entries are asked for a tile ahead of the rows, which come a tile ahead of their products) ----
    f4 qx[NT][NB][2];
    auto dim_of = [&](int b, int e) { if constexpr (F16 || CODES) return 32 * b + K::dims(g, e); else return K::dim(b, g, e); };
    auto fetch_q = [&](auto as_bf16) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const size_t row = row_index(min(16 * n + c, R - 1)) * D;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) qx[n][b][e] = q4_at(P.q, as_bf16, row + dim_of(b, e));
        }
    };
    if (P.q_bf16) fetch_q(std::true_type{});
    else fetch_q(std::false_type{});
    uint32_t warm[NT];                                        // (the rows' masks come to the cache with q; the tiles that ask for them are the last ones)
#pragma unroll
    for (int n = 0; n < NT; ++n) warm[n] = P.mask[(size_t) (sv.first + tok_of(min(16 * n + c, R - 1))) * P.words];
    int i = ta + wave;
    auto tile_of = [&](int i) { return sp.tile(min(i, tb - 1)); };   // (past the last: that one once more, unused)
    key_rows::pages pg;
    if (i < tb) {
        const key_rows::pages now = keys.pages_of(tile_of(i));
        pg = keys.pages_of(tile_of(i + NW));
        const where at = keys.at(tile_of(i), now);
        ask_v(at, 0);
        ask_k(at);
    }
    constexpr int NQR = C::QL ? 1 : NQ;                       // halves in registers
    h8 qf[NT][NQR][NB];
    char * const ql = lds + NW * C::WAVE_B + lane * 16;
    auto q_at = [&](int n, int k, int b) { return k < NQR ? qf[n][k < NQR ? k : 0][b] : *reinterpret_cast<const h8 *>(ql + (n * NB + b) * 1024); };
    float factor[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float most = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(qx[n][b][e >> 2][e & 3]));
        const int ex = row_exponent(max_swap32(max_swap16(most)));
        factor[n] = ldexpf(P.factor, ex);
        const float by = ldexpf(P.sign, -ex);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            h8 r[NQ];
            halves<NQ>([&](int e) { return qx[n][b][e >> 2][e & 3]; }, [&](int) { return by; }, r);
#pragma unroll
            for (int k = 0; k < NQR; ++k) qf[n][k][b] = r[k];
            if constexpr (C::QL) *reinterpret_cast<h8 *>(ql + (n * NB + b) * 1024) = r[NQ - 1];
        }
        asm volatile("" :: "v"(warm[n]));
        __builtin_amdgcn_sched_barrier(0);
    }

    f4 o[NT][NDT];
    float ref[NT], l[NT];
    int E = -40;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        ref[n] = MINUS_INF;
        l[n] = 0.f;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[n][dt] = f4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) kr[x] = kn[x];
    for (int st = 0; i < tb; i += NW, st ^= 1) {
        const int k0 = sp.tile(i) * 32;
        const bool more = i + NW < tb;                     // (no load is left behind: V's go to LDS, where results are folded)
        // what was asked for a tile ago is there; now the next tile
        if constexpr (F16) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const where at = keys.at(tile_of(i + NW), pg);
        pg = keys.pages_of(tile_of(i + 2 * NW));
        if (more) {
            if constexpr (F16) ask_v(at, st ^ 1);
            ask_k(at);
        }
        // ---- V's values (or codes, and all scales) into LDS ----
        if constexpr (CODES) {
            float dm = 0.f;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < keys16<KT, D>::NSC; ++y) dm = fmaxf(dm, fabsf(keys16<KT, D>::scale(vs[x], y)));
            dm = wave_max(dm);
            const int e = __builtin_amdgcn_readfirstlane(dm > 0.f && dm < __builtin_inff() ? __builtin_amdgcn_frexp_expf(dm) : E);
            if (e > E) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                        for (int y = 0; y < 4; ++y) o[n][dt][y] = ldexpf(o[n][dt][y], E - e);
                E = e;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                keys16<KT, D>::put(tk + x * C::TAB, kr[x].d, c, g);
                keys16<KT, D>::put(tv + x * C::TAB, vs[x], c, g, -E);
                G::store(vr[x], mine + x * PL_B, lane);
            }
            if (more) ask_v(at, 0);
            __builtin_amdgcn_wave_barrier();
        } else if constexpr (!F16) {
#pragma unroll
            for (int x = 0; x < 2; ++x) G::store(vr[x], mine + x * PL_B, lane);
            if (more) ask_v(at, 0);
            __builtin_amdgcn_wave_barrier();
        }
        // ---- S^T ----
        f4 s[2][NT];
        if constexpr (F16 || CODES) K::template scores<NT, NQ>(kr, q_at, tk, g, s);
        else {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NT; ++n) s[x][n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const h8 a0 = K::operand(kr[0], b), a1 = K::operand(kr[1], b);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    s[0][n] = mfma16(a0, qf[n][0][b], s[0][n]);
                    s[1][n] = mfma16(a1, qf[n][0][b], s[1][n]);
                }
            }
        }
        // ---- what a column does not see: in front of the tree by its window, in the tree by its mask ----
        if (!(k0 + 31 <= all_hi && k0 >= all_lo)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const sight v = sight_of(P, sv, tok_of(min(16 * n + c, R - 1)), k0);
                const int hi = v.hi - 4 * g, lo = v.lo - 4 * g, sk = v.sk - 4 * g;
                const uint32_t bits = v.bits >> (4 * g);
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 16 * x + e;             // (and 4 g)
                        s[x][n][e] = ((j <= hi) & ((j > lo) | (j < sk))) | (int) (bits >> j & 1) ? s[x][n][e] : MINUS_INF;
                    }
            }
        }
        // ---- softmax ----
        float p[NT][8];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float mx = MINUS_INF;
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][n][e & 3]);
            mx = max_swap32(max_swap16(mx)) * factor[n];
            const bool fresh = ref[n] == MINUS_INF, move = mx > (fresh ? MINUS_INF : ref[n] + (HEAD + STEP));
            if (__any(move)) {
                const float to = move ? mx - HEAD : ref[n], alpha = fresh ? 1.f : __builtin_amdgcn_exp2f(ref[n] - to);
                ref[n] = to;
                l[n] *= alpha;
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) o[n][dt] *= alpha;
            }
            const float nr = ref[n] == MINUS_INF ? 0.f : -ref[n];
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[n][e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][n][e & 3], factor[n], nr));
                sum += p[n][e];
            }
            l[n] += sum;
        }
        // ---- O^T += V^T P ----
        const char * const vt = mine + (F16 ? st * C::VT_B : 0);
        // (a block's scales and rows of V^T are asked for a block ahead)
        struct block_of { f4 d[2]; h4 a[2][2]; };
        auto read = [&](int b) {
            block_of r;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (CODES) r.d[x] = *reinterpret_cast<const f4 *>(tv + x * C::TAB + b * 16 + 4 * g);
#pragma unroll
                for (int y = 0; y < 2; ++y) r.a[y][x] = v_read(vt + x * PL_B, 2 * b + y);
            }
            return r;
        };
        h8 pb[NT][NQ];
        block_of next = read(0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const block_of now = next;
            if (b + 1 < NB) next = read(b + 1);
            if (CODES || b == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n) halves<NQ>([&](int e) { return p[n][e]; }, [&](int e) { return CODES ? now.d[e >> 2][e & 3] : 1.f; }, pb[n]);
            }
#pragma unroll
            for (int k = 0; k < NQ; ++k)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const h4 a0 = now.a[y][0], a1 = now.a[y][1];
                        o[n][2 * b + y] = mfma16(h8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]}, pb[n][k], o[n][2 * b + y]);
                    }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) kr[x] = kn[x];
    }

    // ---- results: lane (column c, group g) holds dims 16 dt + 4 g .. ----
    {
    asm volatile("" : "+v"(tid));
    const int c = tid & 15, g = (tid >> 4) & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
    }
    // ---- fold the waves, in their order, PC columns at a time ----
    auto ml = [&](int w, int which, int col) -> float & { return reinterpret_cast<float *>(lds + C::ML_AT)[(w * 2 + which) * 16 * NT + col]; };
    if constexpr (C::ML_OVER) __syncthreads();                // (until the first wave has done with its scales)
    if (g == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n) { ml(wave, 0, 16 * n + c) = ref[n]; ml(wave, 1, 16 * n + c) = l[n]; }
    }
    float * const parked = reinterpret_cast<float *>(mine);
    constexpr int OS = D + 4, D4 = D / 4;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int half = 0; half < 16; half += C::PC) {
            const int h0 = 16 * n + half;
            if (h0 >= R) break;
            if (h0) __syncthreads();
            if (c >= half && c < half + C::PC) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    f4 v = o[n][dt];
                    if constexpr (CODES) {
#pragma unroll
                        for (int y = 0; y < 4; ++y) v[y] = ldexpf(v[y], E);
                    }
                    *reinterpret_cast<f4 *>(parked + (c - half) * OS + 16 * dt + 4 * g) = v;
                }
            }
            __syncthreads();
            for (int t = tid; t < (min(h0 + C::PC, R) - h0) * D4; t += NTHR) {
                const int cc = t / D4, d = 4 * (t - cc * D4), col = h0 + cc;
                float m[NW], lw[NW], M = MINUS_INF, lt = 0.f;
                f4 x[NW], acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    m[w] = ml(w, 0, col);
                    lw[w] = ml(w, 1, col);
                    x[w] = *reinterpret_cast<const f4 *>(reinterpret_cast<const float *>(lds + w * C::WAVE_B) + cc * OS + d);
                    M = fmaxf(M, m[w]);
                }
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float fw = m[w] == MINUS_INF ? 0.f : __builtin_amdgcn_exp2f(m[w] - M);
                    lt += m[w] == MINUS_INF ? lw[w] : lw[w] * fw;     // (no maximum: 0, or NaN where scores were)
                    acc += x[w] * fw;
                }
                finish(P, row_index(col), d, D, pieces > 1 ? piece : -1, acc, M, lt);
            }
        }
    }
    if (P.nks > 1 && piece == 0 && hk == 0 && tid == 0) P.part_n[f.seq * P.max_groups + f.group] = pieces;
    __syncthreads();                                          // (what was folded is read; the next group's V goes there)
  }
}

// ---- more columns: waves that share tiles ----
// K or V of a tile is brought by two waves each, 16 keys a wave, and lies in LDS as f16 (two planes where results are exact): converted once for all columns. Products take it
// as their first operand, so that a column is a lane's own: its maximum and sum need one exchange with the other half of the wave. A step holds P of a tile beside the
// products S^T of the next one, and O^T beside that one's maximum; parts of what is put into LDS stand between products.
template <uint32_t KT, int D, bool EXACT> struct team_cfg {
    static constexpr bool F16 = KT == P1A_KV_F16;
    static constexpr int NPL = group_planes(KT, EXACT), BN = 32, NG = BN / 16, G_B = NPL * plane_bytes(D), T_B = NG * G_B;   // T_B: K or V of a tile
    // Tiles are asked for four steps ahead. f16 goes to LDS by itself: places for four; the others wait in registers, two deep, and LDS holds two
    static constexpr int PLACES = F16 ? 4 : 2;
    static constexpr int PAST = 2 * PLACES * T_B;             // (behind the tiles: what the lanes know of the sequences)
    static constexpr int LDS = PAST + 64 * sizeof(typename tree_runs<BN, 1, 32, NW, 6>::of_lane);
    static constexpr int WGS = D <= 128 ? 2 : 1;
};

// a quantized group's way into LDS in parts, to stand between products
template <uint32_t KT, int D, int NPL> struct parts;
template <int D, int NPL> struct parts<P1A_KV_Q8_0, D, NPL> {
    using G = group<P1A_KV_Q8_0, D, NPL>;
    static constexpr int N = 2 * G::NJ;
    template <int i> static __device__ __forceinline__ void store(const typename G::raw & r, char * to, int lane) {
        constexpr int j = i / 2, x = i % 2;
        const int q = lane >> 4, k = lane & 15;
        const uint32_t s = q & 2 ? r.d[j] >> 16 : r.d[j] & 0xffff;
        const h2 d = __builtin_bit_cast(h2, s | (s << 16));
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) times4<NPL>(r.w[j][2 * x + e] ^ 0x80808080u, 1152.f, d, h + 2 * e, l + 2 * e);
        char * const at = to + chunk_at(k, 8 * j + 2 * q + x);
        *reinterpret_cast<u4 *>(at) = u4{h[0], h[1], h[2], h[3]};
        if constexpr (NPL == 2) *reinterpret_cast<u4 *>(at + plane_bytes(D)) = u4{l[0], l[1], l[2], l[3]};
    }
};
template <int D, int NPL> struct parts<P1A_KV_Q4_0, D, NPL> {
    using G = group<P1A_KV_Q4_0, D, NPL>;
    static constexpr int N = 4 * G::NJ;
    template <int i> static __device__ __forceinline__ void store(const typename G::raw & r, char * to, int lane) {
        constexpr int j = i / 4, x = i % 4;
        const int k = lane & 15, b = 4 * j + (lane >> 4);
        if (G::NB % 4 && b >= G::NB) return;
        const h2 d = __builtin_bit_cast(h2, r.d[j] | (r.d[j] << 16));
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t w = r.w[j][2 * (x & 1) + e];
            times4<NPL>((x & 2 ? w >> 4 : w) & 0x0f0f0f0fu, 1032.f, d, h + 2 * e, l + 2 * e);
        }
        char * const at = to + chunk_at(k, 4 * b + x);
        *reinterpret_cast<u4 *>(at) = u4{h[0], h[1], h[2], h[3]};
        if constexpr (NPL == 2) *reinterpret_cast<u4 *>(at + plane_bytes(D)) = u4{l[0], l[1], l[2], l[3]};
    }
};
template <int D, int NPL> struct parts<P1A_KV_F16, D, NPL> {
    static constexpr int N = 0;
};

// Position that the row of key j is fetched from, one that some row sees: j itself, or the nearest of its 16 keys that is, or (none of them) of the tile - so that the 16 rows
// lie in one page wherever pages have 16 positions and more
template <int BN> __device__ __forceinline__ int seen_in_group(const span & s, int k0, int kb, int j) {
    if (j > s.pmax) return s.pmax;
    if (j >= s.lo || j < s.ns) return j;
    return s.lo < kb + 16 ? s.lo : s.ns > kb ? s.ns - 1 : k0 + BN > s.lo ? s.lo : s.ns - 1;
}

template <uint32_t KT, int D, bool EXACT>
__global__ void __launch_bounds__(NTHR, (team_cfg<KT, D, EXACT>::WGS)) team_k(const tree_params) {
    const tree_params & P0 = read_again();
    const int Hkv = P0.Hkv, runs = P0.runs;
    using C = team_cfg<KT, D, EXACT>;
    using G = group<KT, D, C::NPL>;
    using PT = parts<KT, D, C::NPL>;
    constexpr bool F16 = C::F16;
    constexpr int BN = C::BN, G_B = C::G_B, T_B = C::T_B, PL_B = plane_bytes(D), NPL = C::NPL;
    constexpr int NKS = D / 16, NDT = D / 32, NQ = EXACT ? 2 : 1, PF_K = NPL == 2 ? 1 : EXACT ? 2 : 4, PF_V = NPL == 2 ? 1 : EXACT ? 2 : 3;
    using runs_t = tree_runs<BN, 1, 32, NW, 6>;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int xcd = blockIdx.x & 7, jx = blockIdx.x >> 3, hk = jx % Hkv, run = jx / Hkv * 8 + xcd;
    if (run >= runs) return;
    runs_t steps;
    steps.first = 0;
    steps.end = 1;
    steps.per = 1 << 30;
    auto * const seqs = (typename runs_t::of_lane *) (lds + C::PAST);
    if (P0.nks > 1) {
        if (!steps.begin(P0.R, P0.pg, P0.GQA, run, runs, P0.nks)) return;
        if (wave == 0) seqs[threadIdx.x] = steps.first64;    // (kept in registers it would take five of those that a group's work needs)
        __syncthreads();
    }
    const size_t head_off = (size_t) hk * head_bytes(KT, D);
    // wave w brings group w % 2 of every tile's K (waves 0 and 1) or V
    const int grp = wave & 1;
    const bool my_v = wave >= 2;
    char * const k_place = lds, * const v_place = lds + C::PLACES * T_B;

  for (int at_step = steps.first; at_step < steps.end;) {
    const tree_params & P = read_again();
    auto tok_of = [&](int r) {
        const int t = (int) __umulhi((uint32_t) r, P.gqa_magic);
        return r - t * P.GQA >= P.GQA ? t + 1 : t;
    };
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, c = lane & 31, g = lane >> 5;
    typename runs_t::found f;
    if (P.nks > 1) {
        steps.first64 = seqs[lane];
        if (!steps.find(P.R, P.pg, P.GQA, at_step, lane, f)) return;
    } else {                                                  // a group each
        f.seq = run / P.max_groups; f.group = run - f.seq * P.max_groups; f.first = 0; f.steps = 1;
        f.v = seq_of<true>(P.R, f.seq);
        f.table = P.pg.pt && P.pg.rtab ? sload_i32(P.pg.rtab + f.seq) : 0;
        if (f.v.count < 1) return;
    }
    const seq_view & sv = f.v;
    const group_of sh = groups_of(sv.count, P.GQA, 32, NW);
    if (P.nks == 1 && f.group >= sh.groups) return;
    typename runs_t::share due{0, 1 << 26, 0, 1};
    if (P.nks > 1) due = steps.share_of(f, at_step, run);
    at_step = f.first + f.steps;
    if (due.to <= 0) continue;
    const int pieces = due.pieces, piece = due.piece;
    const int col0 = (f.group * sh.bpg + wave) * 32, ncols = wave < sh.bpg ? min(sh.cols - col0, 32) : 0;   // this wave's columns (none: it brings keys only)
    const int my_col = ncols > 0 ? col0 + min(c, ncols - 1) : 0, my_tok = tok_of(my_col);
    const size_t my_row = (size_t) (sv.first + my_tok) * P.Hq + (size_t) hk * P.GQA + (my_col - my_tok * P.GQA);
    const span sp = runs_t::span_of_rows(P.R, sv);
    const int ta = due.from, tb = min(due.to, sp.nt);
    // positions that all rows see
    const bool odd = sv.pos0 < 0 || sv.pos0 + sv.count > P.R.n_ctx;
    const int all_hi = odd ? -1 : sv.pos0 - 1, all_lo = P.R.window == INT32_MAX ? 0 : sp.pmax - P.R.window + 1;

    // ---- where rows of the cache are ----
    const gbytes from = (gbytes) (my_v ? P.vc : P.kc);
    const int32_t * const ptab = P.pg.pt ? P.pg.pt + f.table : nullptr;
    const bool paged16 = P.pg.psh >= 4;
    auto tile_of = [&](int i) { return sp.tile(min(i, tb - 1)); };   // (past the last: that one once more, unused)
    auto tile_of_item = [&](int e) { return tile_of(ta + max(e - (my_v ? 1 : 0), 0)); };   // (items: below)
    auto pos_of = [&](int tile) { return seen_in_group<BN>(sp, tile * BN, tile * BN + 16 * grp, tile * BN + 16 * grp + G::key(lane)); };
    // Pages of 16 positions and more: one page for the wave's 16 keys of a tile, and lane l holds that of item 64 n + l - a load every 64 items, so that none has to be waited for
    // while tiles are on their way. Smaller ones: a load for every item, and a wait for it.
    auto pages_from = [&](int e0) {
        const int tile = tile_of_item(e0 + lane), kb = tile * BN + 16 * grp;
        return ptab && paged16 ? ptab[seen_in_group<BN>(sp, tile * BN, kb, kb) >> P.pg.psh] : 0;
    };

    // ---- Q^T operands: lane (column c, half g) holds dims 16 ks + 8 g .. + 7 ----
    h8 qf[NQ][NKS];
    float factor = P.factor;
    f4 qx[NKS][2];
    auto fetch_q = [&] {
        auto fetch = [&](auto as_bf16) {
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) qx[ks][e] = q4_at(P.q, as_bf16, my_row * D + 16 * ks + 8 * g + 4 * e);
        };
        if (P.q_bf16) fetch(std::true_type{});
        else fetch(std::false_type{});
    };
    auto take_q = [&] {
        float most = 0.f;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(qx[ks][e >> 2][e & 3]));
        const int ex = row_exponent(max_swap32(most));
        factor = ldexpf(factor, ex);
        const float by = ldexpf(P.sign, -ex);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            h8 r[NQ];
            halves<NQ>([&](int e) { return qx[ks][e >> 2][e & 3]; }, [&](int) { return by; }, r);
#pragma unroll
            for (int k = 0; k < NQ; ++k) {
                qf[k][ks] = r[k];
                // (in accumulation registers, where the products read it as it is: what vector instructions work on has the others)
                if constexpr (D == 256) asm volatile("" : "+a"(qf[k][ks]));
            }
        }
    };

    f16x o[NDT];
    float ref = MINUS_INF, l = 0.f, mx = MINUS_INF;           // mx: the column's largest score of the tile in hand

    auto clear = [&] {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    };
    const k_frag kf(lane, G_B);
    const v_frag vf(lane);
    // (a place in LDS as a number the compiler does not see through - offsets from it fit the instructions, those from the start do not)
    auto hidden = [&](int at) {
        asm volatile("" : "+s"(at));
        return (const char *) lds + at;
    };
    auto s_product = [&](f16x & s, int ks, const h8 (&a)[NPL]) {
        if (ks == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
        }
        s = mfma32(a[0], qf[0][ks], s);
        if constexpr (EXACT) s = mfma32(a[0], qf[NQ - 1][ks], s);
        if constexpr (NPL == 2) s = mfma32(a[NPL - 1], qf[0][ks], s);
    };
    // (what only the ends need is worked out there once more: kept, it would hold registers all the way)
    auto again = [&](int x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    auto mask = [&](f16x & s, int k0) {
        const int me = again(lane), g = me >> 5;
        const sight v = sight_of(P, sv, tok_of(col0 + min(me & 31, ncols - 1)), k0);
        const int hi = v.hi - 4 * g, lo = v.lo - 4 * g, sk = v.sk - 4 * g;
        const uint32_t bits = v.bits >> (4 * g);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int j = mfma_row(i, 0);                     // (and 4 g)
            s[i] = ((j <= hi) & ((j > lo) | (j < sk))) | (int) (bits >> j & 1) ? s[i] : MINUS_INF;
        }
    };
    float top = -MINUS_INF;
    asm volatile("" : "+s"(top));
    auto most_of = [&](const f16x & s) {
        float m = MINUS_INF;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = larger(m, s[i], top);
        return m;
    };
    auto whole = [&](int k0) { return k0 + BN - 1 <= all_hi && k0 >= all_lo; };

    // ---- what a wave brings: of item e K of tile e or V of tile e - 1. Item e is asked for at step e - 4 and in LDS at the end of step e - 2 ----
    typename G::raw raw[2];
    auto to_of = [&](int e) { return (my_v ? v_place + (e + C::PLACES - 1) % C::PLACES * T_B : k_place + e % C::PLACES * T_B) + grp * G_B; };
    int pages = 0;
    size_t row = 0;
    auto next_row = [&](int e) {
        if (!(e & 63)) {
            pages = pages_from(e);
            asm volatile("" : "+v"(pages));                    // (waited for here: behind the branch every item would wait)
        }
        const int tile = tile_of_item(e), kb = tile * BN + 16 * grp;
        if (paged16 || !ptab) {                               // where the first of the 16 rows is, the same for all lanes, and how far behind it a lane's own
            int a = kb, off = G::key(again(lane)) * (int) P.pg.rowb;
            if (!(kb + 15 <= sp.pmax && (kb >= sp.lo || kb + 15 < sp.ns))) {
                const int j = pos_of(tile);
                a = __builtin_amdgcn_readfirstlane(j);
                off = (j - a) * (int) P.pg.rowb;
            }
            const size_t at = ptab ? (size_t) __builtin_amdgcn_readlane(pages, e & 63) * P.pg.pstride + (size_t) (a & ((1 << P.pg.psh) - 1)) * P.pg.rowb : (size_t) a * P.pg.rowb;
            row = head_off + at + (ptrdiff_t) off;
        } else {
            const int j = pos_of(tile);
            int page = ptab[j >> P.pg.psh];
            asm volatile("" : "+v"(page));
            row = head_off + (size_t) page * P.pg.pstride + (size_t) (j & ((1 << P.pg.psh) - 1)) * P.pg.rowb;
        }
    };
    auto load = [&](auto y, int e, typename G::raw & r) __attribute__((always_inline)) { G::template piece<y>(r, from + row, to_of(e), lane); };
    auto part = [&](auto y, int e, const typename G::raw & r) __attribute__((always_inline)) { if constexpr (!F16) PT::template store<y>(r, to_of(e), lane); };
    // ---- a step: P of this tile beside the products S^T of the next one, then O^T beside the next one's maximum; item i + 4 is asked for, item i + 2 put down ----
    auto step = [&](int i, int next, f16x & s, f16x & sn, typename G::raw & r) __attribute__((always_inline)) {
        const char * const kp = hidden((i + 1) % C::PLACES * T_B), * const vp = hidden((C::PLACES + i % C::PLACES) * T_B);
        const bool fresh = ref == MINUS_INF, move = mx > (fresh ? MINUS_INF : ref + (HEAD + STEP));
        if (__builtin_expect(__any(move), 0)) {
            const float to = move ? mx - HEAD : ref, alpha = fresh ? 1.f : __builtin_amdgcn_exp2f(ref - to);   // (fresh: nothing accumulated)
            ref = to;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int k = 0; k < 16; ++k) o[dt][k] *= alpha;
        }
        const float nr = ref == MINUS_INF ? 0.f : -ref;       // (a column that has seen nothing: exp2(-inf))
        constexpr int NF = 2 * NDT;
        h8 pb[NQ][2];
        float ls[2] = {0.f, 0.f};
        auto k_read = [&](int ks, int pl) { return kf.read(kp + pl * PL_B, ks); };
        auto v_read = [&](int f, int pl) { return vf.read(vp + (f / NDT) * G_B + pl * PL_B, f % NDT); };
        // (operands from LDS are asked for a few products ahead, and no further: registers)
        h8 fr[PF_K][NPL];
#pragma unroll
        for (int k = 0; k < PF_K; ++k)
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) fr[k][pl] = k_read(k, pl);
        each<NKS>([&](auto k) __attribute__((always_inline)) {
            h8 a[NPL];
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) {
                a[pl] = fr[k % PF_K][pl];
                if (k + PF_K < NKS) fr[k % PF_K][pl] = k_read(k + PF_K, pl);
            }
            s_product(sn, k, a);
#pragma unroll
            for (int v = k * 16 / NKS / 2 * 2; v < (k + 1) * 16 / NKS / 2 * 2; v += 2) {   // pairs of values of P
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[v], factor, nr)), p1 = __builtin_amdgcn_exp2f(fmaf(s[v + 1], factor, nr));
                ls[0] += p0;
                ls[1] += p1;
                asm volatile("" : "+v"(ls[0]), "+v"(ls[1]));  // (here: put off, all of P would stay in registers)
                h2 h = __builtin_convertvector(f2w{p0, p1}, h2);
                asm("" : "+v"(h));
                pb[0][v >> 3][v & 7] = h[0];
                pb[0][v >> 3][(v & 7) + 1] = h[1];
                if constexpr (EXACT) {
                    pb[NQ - 1][v >> 3][v & 7] = (half_t) (p0 - (float) h[0]);
                    pb[NQ - 1][v >> 3][(v & 7) + 1] = (half_t) (p1 - (float) h[1]);
                }
            }
            // (a part of what is put down every few products: one behind the other they would hold the wave)
            each<PT::N>([&](auto y) __attribute__((always_inline)) { if constexpr (y * 2 < PT::N && (y * 2 + 1) * NKS / (PT::N + 1) == k) part(y, i + 2, r); });
            __builtin_amdgcn_sched_barrier(0);
        });
        l += ls[0] + ls[1];
        h8 fv[PF_V][NPL];
#pragma unroll
        for (int f = 0; f < PF_V; ++f)
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) fv[f][pl] = v_read(f, pl);
        mx = MINUS_INF;
        each<NF>([&](auto f) __attribute__((always_inline)) {
            constexpr int ps = f / NDT, dt = f % NDT;
            h8 a[NPL];
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) {
                a[pl] = fv[f % PF_V][pl];
                if (f + PF_V < NF) fv[f % PF_V][pl] = v_read(f + PF_V, pl);
            }
            o[dt] = mfma32(a[0], pb[0][ps], o[dt]);
            if constexpr (EXACT) o[dt] = mfma32(a[0], pb[NQ - 1][ps], o[dt]);
            if constexpr (NPL == 2) o[dt] = mfma32(a[NPL - 1], pb[0][ps], o[dt]);
#pragma unroll
            for (int v = f * 16 / NF; v < (f + 1) * 16 / NF; ++v) mx = larger(mx, sn[v], top);
            asm volatile("" : "+v"(mx));
            each<PT::N>([&](auto y) __attribute__((always_inline)) { if constexpr (y * 2 >= PT::N && (y * 2 - PT::N) * NF / PT::N == f) part(y, i + 2, r); });
            __builtin_amdgcn_sched_barrier(0);
        });
        if (__builtin_expect(!whole(next * BN), 0)) {
            mask(sn, next * BN);
            mx = most_of(sn);
        }
        mx = max_swap32(mx) * factor;
    };

    // what was asked for `left` items ago and earlier is there, and put down; every wave
    auto arrived = [&](auto left) __attribute__((always_inline)) {
        if constexpr (F16) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(left * G::PIECES) : "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto ask = [&](int e, typename G::raw & r) __attribute__((always_inline)) {
        next_row(e);
        each<G::PIECES>([&](auto y) __attribute__((always_inline)) { load(y, e, r); });
    };
    auto put = [&](int e, const typename G::raw & r) __attribute__((always_inline)) { each<PT::N>([&](auto y) __attribute__((always_inline)) { part(y, e, r); }); };
    fetch_q();
    if (ta < tb) {
        ask(0, raw[0]);
        ask(1, raw[1]);
        if constexpr (F16) {
            ask(2, raw[0]);
            ask(3, raw[1]);
        }
        take_q();
        if constexpr (!F16) {
            put(0, raw[0]);
            ask(2, raw[0]);
        }
        arrived(std::integral_constant<int, 3>{});
        clear();
        f16x sa, sb;
        if (ncols > 0) {
            const char * const kp = hidden(0);
#pragma unroll
            for (int k = 0; k < NKS; ++k) {
                h8 a[NPL];
#pragma unroll
                for (int pl = 0; pl < NPL; ++pl) a[pl] = kf.read(kp + pl * PL_B, k);
                s_product(sa, k, a);
            }
            if (!whole(tile_of(ta) * BN)) mask(sa, tile_of(ta) * BN);
            mx = max_swap32(most_of(sa)) * factor;
        }
        if constexpr (!F16) {
            put(1, raw[1]);
            ask(3, raw[1]);
        }
        arrived(std::integral_constant<int, 2>{});
        // tile i (counted from ta): K(i + 1) and V(i) are there
        auto turn = [&](int i, f16x & s, f16x & sn, typename G::raw & r) __attribute__((always_inline)) {
            if constexpr (F16) ask(i + 4, r);
            if (ncols > 0) step(i, tile_of(ta + i + 1), s, sn, r);
            else put(i + 2, r);
            if constexpr (!F16) ask(i + 4, r);
            arrived(std::integral_constant<int, 2>{});
        };
        // (in pairs, the last one by itself: with a way out between the two the compiler waits at the top for what was asked for last)
        int i = 0;
        for (; ta + i + 1 < tb; i += 2) {
            turn(i, sa, sb, raw[0]);
            turn(i + 1, sb, sa, raw[1]);
        }
        if (ta + i < tb) turn(i, sa, sb, raw[0]);
        if constexpr (F16) asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");   // (nothing is on its way to LDS when the next group begins)
    } else clear();

    // ---- results: lane (column c, half g) holds dims 32 dt + 8 (i / 4) + 4 g + i % 4 ----
    {
    const tree_params & P = read_again();
    l += __shfl_xor(l, 32);
    const int me = again(lane), c = me & 31, g = me >> 5;
    if (c < ncols) {
        const int col = col0 + c, tok = tok_of(col);
        const size_t my_row = (size_t) (sv.first + tok) * P.Hq + (size_t) hk * P.GQA + (col - tok * P.GQA);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                finish(P, my_row, 32 * dt + 8 * q + 4 * g, D, pieces > 1 ? piece : -1, f4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]}, ref, l);
    }
    if (P.nks > 1 && piece == 0 && hk == 0 && threadIdx.x == 0) P.part_n[f.seq * P.max_groups + f.group] = pieces;
    }
  }
}

// Partials of a row -> its result: 256 / (D / 4) rows of one sequence a workgroup, four dims a thread
struct tree_merge_params {
    rows_view R;
    const float * part_o, * part_ml, * gate;
    void * out;
    float * lse;
    int Hq, GQA, D, nks, out_bf16, BC, waves, max_groups;
    const int * part_n;    // [n_seq][max_groups] partials of a group's rows (1: they are finished)
};
__global__ void __launch_bounds__(NTHR) tree_merge_k(const tree_merge_params P) {
    const int tpr = P.D >> 2, per = NTHR / tpr, sub = threadIdx.x / tpr, d = 4 * (threadIdx.x - sub * tpr);
    item_at at;
    if (!find_item(P.R, blockIdx.x, P.Hq, per, threadIdx.x & 63, at)) return;
    const int r = at.index * per + sub;                       // of the sequence
    if (r >= (long long) at.v.count * P.Hq) return;
    const int t = r / P.Hq, h = r - t * P.Hq;
    const group_of sh = groups_of(at.v.count, P.GQA, P.BC, P.waves);
    const int n = min(P.part_n[at.seq * P.max_groups + (t * P.GQA + h % P.GQA) / (sh.bpg * P.BC)], P.nks);
    if (n < 2) return;                                        // (finished already)
    const long long row = (long long) at.v.first * P.Hq + r;
    // four partials at a time, asked for together
    const float2 * ml = reinterpret_cast<const float2 *>(P.part_ml) + row * P.nks;
    const float * po = P.part_o + row * P.nks * P.D + d;
    float M = MINUS_INF, l = 0.f;
    f4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += 4) {
        float2 p[4];
        f4 v[4];
        float m = M;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int kk = min(k0 + k, n - 1);
            p[k] = ml[kk];
            v[k] = *reinterpret_cast<const f4 *>(po + (size_t) kk * P.D);
            if (k0 + k >= n) p[k].x = MINUS_INF;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) m = fmaxf(m, p[k].x);
        const float w0 = M == MINUS_INF ? 0.f : __builtin_amdgcn_exp2f(M - m);
        l *= w0;
        acc *= w0;
        M = m;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (p[k].x == MINUS_INF) continue;                // (it has seen nothing, and written no values)
            const float w = __builtin_amdgcn_exp2f(p[k].x - M);
            l += p[k].y * w;
            acc += v[k] * w;
        }
    }
    if (P.lse && d == 0) P.lse[row] = (M + log2f(l)) * LN2;
    f4 v = acc * (l == 0.f ? 0.f : 1.0f / l);
    const size_t e = (size_t) row * P.D + d;
    if (P.gate) {
        const f4 gt = *reinterpret_cast<const f4 *>(P.gate + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= tree_gate(gt[i]);
    }
    put4(P.out, P.out_bf16, e, v);
}

// (NT = 0: team_k)
template <uint32_t KT, int D, int NT, bool EXACT> int launch_cfg(const tree_params & P, unsigned grid, hipStream_t s) {
    constexpr int lds = [] { if constexpr (NT) return few_cfg<KT, D, NT, EXACT>::LDS; else return team_cfg<KT, D, EXACT>::LDS; }();
    auto * const k = [] { if constexpr (NT) return few_k<KT, D, NT, EXACT>; else return team_k<KT, D, EXACT>; }();
    // (the attribute belongs to the function on ONE device: remembered per device, set again on another)
    static std::atomic<uint32_t> attr_set{0};
    int dev = 0;
    (void) hipGetDevice(&dev);
    const uint32_t bit = 1u << (dev & 31);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        if (hipFuncSetAttribute((const void *) k, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
            (void) hipGetLastError();
            set_error("p1a_attn_tree: cannot reserve %d bytes of LDS", lds);
            return P1A_E_LAUNCH;
        }
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    k<<<grid, NTHR, lds, s>>>(P);
    return launched();
}
// f(cache type, D, NT, EXACT), each as a constant
template <typename F> int for_build(uint32_t type, int D, int NT, bool exact, F && f) {
    auto e = [&](auto kt, auto d, auto nt) { return exact ? f(kt, d, nt, std::true_type{}) : f(kt, d, nt, std::false_type{}); };
    auto n = [&](auto kt, auto d) { return NT == 0 ? e(kt, d, std::integral_constant<int, 0>{}) : NT == 1 ? e(kt, d, std::integral_constant<int, 1>{}) : e(kt, d, std::integral_constant<int, 2>{}); };
    auto dd = [&](auto kt) { return D == 256 ? n(kt, std::integral_constant<int, 256>{}) : D == 128 ? n(kt, std::integral_constant<int, 128>{}) : n(kt, std::integral_constant<int, 64>{}); };
    return type == P1A_KV_F16 ? dd(std::integral_constant<uint32_t, P1A_KV_F16>{}) : type == P1A_KV_Q8_0 ? dd(std::integral_constant<uint32_t, P1A_KV_Q8_0>{}) : dd(std::integral_constant<uint32_t, P1A_KV_Q4_0>{});
}

// the most items of `unit` that the sequences' rows times `mul` can make (as find_item counts them)
long long item_bound(const rows_view & R, int mul, int unit) {
    const long long each = ((long long) R.max_rows * mul + unit - 1) / unit * R.n_seq;
    return R.row0 ? std::min(each, (long long) R.T * mul / unit + R.n_seq) : each;
}

}   // namespace

// How a call is dealt out, from its host numbers and the device: as many runs of steps as there are places for workgroups, unless a workgroup for each group takes no longer
// than a run, its set-up (3), a second group's (2) and the merge (3). Partials take 128 MB at most.
tree_plan plan_tree(const p1a_kv & c, const rows_view & R, int Hq, int max_n, bool exact, int cus) {
    tree_plan pl{};
    const int GQA = Hq / c.Hkv;
    const long long cols = (long long) R.max_rows * GQA;
    pl.NT = cols <= 16 ? 1 : cols <= 32 ? 2 : 0;
    pl.max_groups = pl.NT ? 1 : groups_of(R.max_rows, GQA, 32, NW).groups;
    pl.nks = 1;
    const long long groups = (long long) R.n_seq * pl.max_groups;
    pl.runs = (int) groups;
    const int wgs = for_build(c.type, c.D, pl.NT, exact, [](auto kt, auto d, auto nt, auto ex) {
        if constexpr (nt.value != 0) return few_cfg<kt.value, d.value, nt.value, ex.value>::WGS;
        else return team_cfg<kt.value, d.value, ex.value>::WGS;
    });
    const int step = pl.NT ? 32 * NW : for_build(c.type, c.D, 0, exact, [](auto kt, auto d, auto, auto ex) { return team_cfg<kt.value, d.value, ex.value>::BN; });
    const long long slots = (long long) std::max(cus, 1) * wgs, units = groups * c.Hkv;
    const long long keys = R.window == INT32_MAX ? max_n : std::min<long long>(max_n, (long long) R.window + R.max_rows + R.n_sink);
    const long long nt = std::max<long long>((keys + step - 1) / step, 1) + (pl.NT ? 4 : 6);   // (set-up among them: SETUP of the kernels' runs)
    const size_t rows = (size_t) R.T * Hq, row_bytes = (size_t) c.D * 4 + 8;
    const long long runs = std::min(std::max(slots / c.Hkv, 1LL), groups * nt), per = (groups * nt + runs - 1) / runs;
    const long long most = std::min({64LL, runs, nt + 1, (128LL << 20) / (long long) (rows * row_bytes)});
    if (most > 1 && (units + slots - 1) / slots * nt > std::max(per, (nt + most - 2) / (most - 1)) + 8) {
        pl.runs = (int) runs;
        pl.nks = (int) most;
        pl.bytes_n = ((size_t) groups * 4 + 255) & ~(size_t) 255;
        pl.bytes_ml = (rows * pl.nks * 8 + 255) & ~(size_t) 255;
        pl.bytes_o = rows * pl.nks * c.D * 4;
    }
    return pl;
}

int launch_tree(const p1a_kv & c, const chunk_args & a, const uint32_t * mask, int words, hipStream_t s) {
    tree_params P;
    P.q = a.q; P.out = a.out; P.gate = a.gate; P.lse = a.lse; P.mask = mask; P.words = words;
    P.kc = (const char *) c.k; P.vc = (const char *) c.v; P.pg = view_of(c); P.R = a.R;
    P.Hq = a.Hq; P.Hkv = c.Hkv; P.GQA = a.Hq / c.Hkv;
    P.gqa_magic = (uint32_t) (P.GQA == 1 ? (1ull << 32) - 1 : (1ull << 32) / (unsigned) P.GQA);
    P.factor = a.scale == 0.f ? 1.f : (a.scale < 0 ? -a.scale : a.scale) * LOG2E;
    P.sign = a.scale == 0.f ? 0.f : a.scale < 0 ? -1.f : 1.f;
    P.q_bf16 = a.q_bf16; P.out_bf16 = a.out_bf16;
    const bool exact = !a.out_bf16 || a.lse;
    const tree_plan pl = plan_tree(c, a.R, a.Hq, a.max_n, exact, cu_count());
    const long long steps = (((long long) c.n_ctx + 31) / 32 + 1) * pl.max_groups * a.R.n_seq, grid = (pl.runs + 7LL) / 8 * 8 * c.Hkv;
    if (steps > 1 << 30 || grid > MOST_GROUPS) { set_error("p1a_attn_tree: too many positions and nodes for one call (%lld steps, %lld workgroups)", steps, grid); return P1A_E_SHAPE; }
    P.nks = pl.nks; P.runs = pl.runs; P.max_groups = pl.max_groups;
    P.part_o = P.part_ml = nullptr; P.part_n = nullptr;
    if (P.nks > 1) {
        if (a.scratch && !((uintptr_t) a.scratch & 255) && a.scratch_bytes >= pl.bytes_n + pl.bytes_ml + pl.bytes_o) {
            P.part_n = (int *) a.scratch;
            P.part_ml = (float *) ((char *) a.scratch + pl.bytes_n);
            P.part_o = (float *) ((char *) a.scratch + pl.bytes_n + pl.bytes_ml);
        } else {
            float * first;
            if (!split_scratch(s, kept_bytes(pl.bytes_o), kept_bytes(pl.bytes_n + pl.bytes_ml), P.part_o, first)) return P1A_E_SCRATCH;
            P.part_n = (int *) first;
            P.part_ml = (float *) ((char *) first + pl.bytes_n);
        }
    }
    const int rc = for_build(c.type, c.D, pl.NT, exact, [&](auto kt, auto d, auto nt, auto ex) { return launch_cfg<kt.value, d.value, nt.value, ex.value>(P, (unsigned) grid, s); });
    if (rc != P1A_OK || P.nks == 1) return rc;
    const tree_merge_params M{a.R, P.part_o, P.part_ml, a.gate, a.out, a.lse, a.Hq, P.GQA, c.D, P.nks, a.out_bf16, pl.NT ? 16 * pl.NT : 32, pl.NT ? 1 : NW, pl.max_groups, P.part_n};
    tree_merge_k<<<(unsigned) item_bound(a.R, a.Hq, NTHR / (c.D / 4)), NTHR, 0, s>>>(M);
    return launched();
}

}   // namespace p1a
