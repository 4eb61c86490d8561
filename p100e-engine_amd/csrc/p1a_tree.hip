// Attention of the rows of drafted trees - per sequence a few to a thousand nodes, each of which sees what is in front of the tree and its own path - over
// paged caches: p1a_attn_tree.
//
// Work: a column is one q head of a node's row. A sequence's columns under a kv head are cut into blocks of 16 NT, its blocks into groups of at most four; the
// four waves of a workgroup take a block each and walk the same tiles of 32 keys (four blocks), or share the keys among the waves of a block (one block or two).
// Waves share nothing but what the L1 cache holds for them: each reads its own keys, converts them and keeps its own sums. Steps - a tile for every stream of
// keys - are counted through over all groups of all sequences, and a workgroup takes a run of them as long as every other's, whatever the lengths; a group
// that lies in one run is finished there, the others' partials are merged by tree_merge_k.
// Arithmetic: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16, one pass with a running reference of every column. With bf16 results q, P, K and V
// enter as one f16 each, a quantized value times its scale; where results are f32 (EXACT) q and P are two halves, codes stay whole numbers and their
// scales multiply fp32 results (K) or P (V), as in p1a_step.hip.
// Only the last tiles hold nodes of the tree: there a column's 32 bits of its mask are shifted out of two words.
#include "p1a_tiles.hpp"

#include <algorithm>
#include <atomic>

namespace p1a {
namespace {

constexpr int NW = 4, NTHR = NW * 64, PC = 8;                 // waves; columns of a wave folded at a time

// ---- what a sequence's rows make ----
struct shape {
    int cols, blocks, groups, bpg, cb, ks;                    // columns; blocks of columns; groups; blocks of a group; waves side by side; streams of keys
};
__host__ __device__ __forceinline__ shape shape_of(int rows, int GQA, int BC) {
    shape s;
    s.cols = rows * GQA;
    s.blocks = (s.cols + BC - 1) / BC;
    s.groups = (s.blocks + NW - 1) / NW;
    s.bpg = s.groups ? (s.blocks + s.groups - 1) / s.groups : 1;
    s.cb = s.bpg < 3 ? s.bpg : 4;
    if (s.cb < 1) s.cb = 1;
    s.ks = NW / s.cb;
    return s;
}

struct tree_params : chunk_params {
    const uint32_t * mask;                                    // [T][words]
    int words, max_groups;
};

// ---- runs of steps of equal length over the groups of all sequences (lane i of a wave counts for sequence s0 + i) ----
template <int BC> struct tree_runs {
    struct of_lane { int first, pos0, table, rows, per_group, steps; };
    of_lane first64;
    int first, end, per;
    static __device__ __forceinline__ span span_of_rows(const rows_view & R, const seq_view & v) { return span_of<32>(R, v.pos0, v.pos0 + v.count - 1); }
    static __device__ __forceinline__ of_lane look(const rows_view & R, const kv_view & pg, int GQA, int s) {
        of_lane r{0, 0, 0, 0, 0, 0};
        if (s >= R.n_seq) return r;
        const seq_view v = seq_of(R, s);
        r.table = pg.pt && pg.rtab ? pg.rtab[s] : 0;
        r.first = v.first;
        r.pos0 = v.pos0;
        r.rows = v.count;
        if (v.count > 0) {
            const shape h = shape_of(v.count, GQA, BC);
            r.per_group = max((span_of_rows(R, v).nt + h.ks - 1) / h.ks, 1);
            r.steps = r.per_group * h.groups;
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
            n += __builtin_amdgcn_readlane(lanes_up_to(x.steps), 63);
            most = max(most, x.per_group);
        }
        most = rfl((int) wave_max((float) most));             // (a group has 2^25 steps at most: the f32 next to it, 1 off in 2^24, only moves the cut)
        per = max((n + runs - 1) / runs, (most + most_runs - 2) / (most_runs - 1) + (most >> 23));
        first = run * per;
        end = min(first + per, n);
        return first < end;
    }
    // whose step `at` is: sequence, group, the group's first step, its steps. False: nobody's (row0 or pos0 were written since begin())
    struct found { int seq, group, first, steps, table; seq_view v; };
    __device__ __forceinline__ bool find(const rows_view & R, const kv_view & pg, int GQA, int at, int lane, found & f) const {
        int base = 0;
        for (int s0 = 0; s0 < R.n_seq; s0 += 64) {
            const of_lane x = s0 ? look(R, pg, GQA, s0 + lane) : first64;
            const int u = base + lanes_up_to(x.steps);
            const unsigned long long behind = __ballot(u > at);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                f.seq = s0 + l;
                f.steps = __builtin_amdgcn_readlane(x.per_group, l);
                const int start = __builtin_amdgcn_readlane(u, l) - __builtin_amdgcn_readlane(x.steps, l);
                f.group = (at - start) / f.steps;
                f.first = start + f.group * f.steps;
                f.v.first = __builtin_amdgcn_readlane(x.first, l);
                f.v.count = __builtin_amdgcn_readlane(x.rows, l);
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

template <uint32_t KT, int D, int NT, bool EXACT> struct tree_cfg {
    static constexpr bool F16 = KT == P1A_KV_F16, CODES = EXACT && !F16;      // codes as whole numbers, scales outside of the products
    static constexpr int VT_B = 2 * plane_bytes(D);           // 32 keys of V
    static constexpr int V_B = (F16 ? 2 : 1) * VT_B;
    static constexpr int TAB = CODES ? keys16<KT, D>::TAB : 0;
    static constexpr int WAVE_B = V_B + 4 * TAB * 4;          // and the scales of 2 x 16 keys of K and V
    // (the low halves of q, where registers do not hold them: a block's, its streams write the same. One tile of columns: calls of one block)
    static constexpr bool QL = CODES && NT * D >= 256;
    static constexpr int QL_B = QL ? NT * D * 32 : 0, ML_B = NW * 2 * 16 * NT * 4;
    static constexpr bool ML_OVER = 4 * TAB * 4 >= ML_B;      // references and sums go where the first wave's scales were
    static constexpr int ML_AT = ML_OVER ? V_B : NW * WAVE_B + (NT == 1 ? 1 : NW) * QL_B, LDS = NW * WAVE_B + (NT == 1 ? 1 : NW) * QL_B + (ML_OVER ? 0 : ML_B);
    static constexpr int WGS = LDS <= 80 * 1024 && !(D == 256 && NT == 2) ? 2 : 1;   // workgroups of a compute unit
    static_assert(PC * (D + 4) * 4 <= V_B, "folded columns fit where V was");
};

// bits `at` .. `at + 31` of a row's mask (at: from -31 on; what is not there is 0)
__device__ __forceinline__ uint32_t mask_bits(const uint32_t * row, int words, int at) {
    const int w = at >> 5;                                    // (-1 at the least)
    const uint32_t lo = w >= 0 && w < words ? row[w] : 0, hi = w + 1 < words ? row[w + 1] : 0;
    return __builtin_amdgcn_alignbit(hi, lo, at & 31);
}

template <uint32_t KT, int D, int NT, bool EXACT>
__global__ void __launch_bounds__(NTHR, (tree_cfg<KT, D, NT, EXACT>::WGS)) tree_k(const tree_params P) {
    using C = tree_cfg<KT, D, NT, EXACT>;
    constexpr bool F16 = C::F16, CODES = C::CODES;
    using K = typename std::conditional<F16 || CODES, keys16<KT, D>, keysd<KT, D>>::type;
    using G = group<KT, D, CODES ? 0 : 1>;
    constexpr int NB = D / 32, NDT = D / 16, NQ = EXACT ? 2 : 1, PL_B = plane_bytes(D), BC = 16 * NT;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the kv heads of a run of steps, whose rows have cache lines in common, on one XCD
    const int xcd = blockIdx.x & 7, jx = blockIdx.x >> 3, hk = jx % P.Hkv, run = jx / P.Hkv * 8 + xcd;
    if (run >= P.runs) return;
    auto tok_of = [&](int r) {
        const int t = (int) __umulhi((uint32_t) r, P.gqa_magic);
        return r - t * P.GQA >= P.GQA ? t + 1 : t;
    };
    tree_runs<BC> steps;
    steps.first = 0;
    steps.end = 1;
    steps.per = 1 << 30;
    if (P.nks > 1 && !steps.begin(P.R, P.pg, P.GQA, run, P.runs, P.nks)) return;
    char * const mine = lds + wave * C::WAVE_B;
    float * const tk = reinterpret_cast<float *>(mine + C::V_B), * const tv = tk + 2 * C::TAB;
    const size_t head_off = (size_t) hk * head_bytes(KT, D);

  for (int at_step = steps.first; at_step < steps.end;) {
    // (the lane's number anew for each group: what follows from it would be worked out ahead of the loop and kept)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, c = lane & 15, g = lane >> 4;
    typename tree_runs<BC>::found f;
    if (P.nks > 1) {
        if (!steps.find(P.R, P.pg, P.GQA, at_step, lane, f)) return;
    } else {                                                  // a group each
        f.seq = run / P.max_groups; f.group = run - f.seq * P.max_groups; f.first = 0; f.steps = 1 << 26;
        f.v = seq_of<true>(P.R, f.seq);
        f.table = P.pg.pt && P.pg.rtab ? sload_i32(P.pg.rtab + f.seq) : 0;
        if (f.v.count < 1) return;
    }
    const seq_view & sv = f.v;
    const shape sh = shape_of(sv.count, P.GQA, BC);
    if (P.nks == 1 && f.group >= sh.groups) return;
    const int run0 = f.first / steps.per, pieces = P.nks > 1 ? (f.first + f.steps - 1) / steps.per - run0 + 1 : 1, piece = P.nks > 1 ? run - run0 : 0;
    const int beside = wave & (sh.cb - 1), stream = wave / sh.cb;   // (cb: 1, 2 or 4)
    const int block = f.group * sh.bpg + beside, col0 = block * BC;
    const bool busy = beside < sh.bpg && col0 < sh.cols;
    const int R = busy ? min(sh.cols - col0, BC) : 1;         // (a wave without a block looks at column 0 and writes nothing)
    const int first_col = busy ? col0 : 0;
    auto row_index = [&](int r) { const int t = tok_of(r); return (size_t) (sv.first + t) * P.Hq + (size_t) hk * P.GQA + (r - t * P.GQA); };
    const span sp = tree_runs<BC>::span_of_rows(P.R, sv);
    const int ta = (at_step - f.first) * sh.ks, tb = P.nks > 1 ? min((min(steps.end, f.first + f.steps) - f.first) * sh.ks, sp.nt) : sp.nt;
    at_step = f.first + f.steps;
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
    typename K::raw kr[2];
    typename std::conditional<F16, none, typename group<F16 ? P1A_KV_Q8_0 : KT, D, CODES ? 0 : 1>::raw>::type vr[2];
    typename keys16<KT, D>::scales vs[2];
    auto ask_k = [&](const where & w) {
#pragma unroll
        for (int x = 0; x < 2; ++x) K::load(kr[x], (gbytes) P.kc + w.off[x], g);
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

    int i = busy ? ta + stream : tb;
    if (i < tb) {
        const where at = keys.at(sp.tile(i), keys.pages_of(sp.tile(i)));
        ask_v(at, 0);
        ask_k(at);
    }

    // ---- Q^T: columns 16 n + c ----
    constexpr int NQR = C::QL ? 1 : NQ;                       // halves in registers
    h8 qf[NT][NQR][NB];
    char * const ql = lds + NW * C::WAVE_B + beside * C::QL_B + lane * 16;
    auto q_at = [&](int n, int k, int b) { return k < NQR ? qf[n][k < NQR ? k : 0][b] : *reinterpret_cast<const h8 *>(ql + (n * NB + b) * 1024); };
    float factor[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const size_t row = row_index(first_col + min(16 * n + c, R - 1));
        h8 qq[NQ][NB];
        if constexpr (F16 || CODES) factor[n] = ldexpf(P.factor, q_columns<KT, D, NQ>(P.q, P.q_bf16, row, P.sign, g, qq));
        else {
            f4 x[NB][2];
            float most = 0.f;
            auto fetch = [&](auto as_bf16) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) x[b][e] = q4_at(P.q, as_bf16, row * D + K::dim(b, g, e));
            };
            if (P.q_bf16) fetch(std::true_type{});
            else fetch(std::false_type{});
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[b][e >> 2][e & 3]));
            const int ex = row_exponent(max_swap32(max_swap16(most)));
            factor[n] = ldexpf(P.factor, ex);
            const float by = ldexpf(P.sign, -ex);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8 r[NQ];
                halves<NQ>([&](int e) { return x[b][e >> 2][e & 3]; }, [&](int) { return by; }, r);
                qq[0][b] = r[0];
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int k = 0; k < NQR; ++k) qf[n][k][b] = qq[k][b];
            if constexpr (C::QL) *reinterpret_cast<h8 *>(ql + (n * NB + b) * 1024) = qq[NQ - 1][b];
        }
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
    for (int st = 0; i < tb; i += sh.ks, st ^= 1) {
        const int k0 = sp.tile(i) * 32;
        const bool more = i + sh.ks < tb;
        key_rows::pages pg;
        if (more) pg = keys.pages_of(sp.tile(i + sh.ks));
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
            __builtin_amdgcn_wave_barrier();
        } else if constexpr (!F16) {
#pragma unroll
            for (int x = 0; x < 2; ++x) G::store(vr[x], mine + x * PL_B, lane);
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
        // (V of this tile was asked for ahead of its K)
        if constexpr (F16) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (more) {
            const where at = keys.at(sp.tile(i + sh.ks), pg);
            ask_v(at, st ^ 1);
            ask_k(at);
        }
        // ---- what a column does not see: in front of the tree by its window, in the tree by its mask ----
        if (!(k0 + 31 <= all_hi && k0 >= all_lo)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int tok = tok_of(first_col + min(16 * n + c, R - 1)), slot = sv.pos0 + tok, from = k0 + 4 * g;
                const bool live = slot >= 0 && slot < P.R.n_ctx;
                const uint32_t * const row = P.mask + (size_t) (sv.first + tok) * P.words;
                int lo = -1, sk = 0;
                if (P.R.window != INT32_MAX) {                // (its place: as many nodes behind the first as its path has)
                    int nodes = 0;
                    for (int w = 0; 32 * w < sv.count; ++w) nodes += __popc(sv.count - 32 * w >= 32 ? row[w] : row[w] & ((1u << (sv.count - 32 * w)) - 1));
                    lo = sv.pos0 + max(nodes - 1, 0) - P.R.window - from;
                    sk = P.R.n_sink - from;
                } else lo = -1 - from;
                const int hi = live ? sv.pos0 - 1 - from : INT32_MIN;
                uint32_t bits = 0;
                const int at = k0 - sv.pos0;
                if (live && at > -32) {
                    bits = mask_bits(row, P.words, at);
                    const int left = sv.count - at;           // nodes that are there
                    bits = left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1) : 0;
                }
                bits >>= 4 * g;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 16 * x + e;             // (and 4 g)
                        s[x][n][e] = (j <= hi && (j > lo || j < sk)) || (bits >> j & 1) ? s[x][n][e] : MINUS_INF;
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
    }

    // ---- fold the streams of each block, in their order ----
    {
    asm volatile("" : "+v"(tid));
    const int c = tid & 15, g = (tid >> 4) & 3;
    auto ml = [&](int w, int which, int col) -> float & { return reinterpret_cast<float *>(lds + C::ML_AT)[(w * 2 + which) * 16 * NT + col]; };
    if constexpr (C::ML_OVER) __syncthreads();                // (until the first wave has done with its scales)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        if (g == 0) { ml(wave, 0, 16 * n + c) = ref[n]; ml(wave, 1, 16 * n + c) = l[n]; }
    }
    float * const parked = reinterpret_cast<float *>(mine);
    constexpr int OS = D + 4, D4 = D / 4;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int half = 0; half < 16; half += PC) {
            const int h0 = 16 * n + half;                     // columns h0 .. of every block
            if (n || half) __syncthreads();
            if (c >= half && c < half + PC) {
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
            for (int t = tid; t < sh.bpg * PC * D4; t += NTHR) {
                const int u = t / D4, d = 4 * (t - u * D4), b = u / PC, cc = u - b * PC, col = h0 + cc;
                const int at = (f.group * sh.bpg + b) * BC + col;             // of the sequence's columns
                if (at >= sh.cols) continue;
                float M = MINUS_INF, lt = 0.f;
                f4 acc = {0.f, 0.f, 0.f, 0.f};
                for (int k = 0; k < sh.ks; ++k) M = fmaxf(M, ml(k * sh.cb + b, 0, col));
                for (int k = 0; k < sh.ks; ++k) {
                    const int w = k * sh.cb + b;
                    const float m = ml(w, 0, col), fw = m == MINUS_INF ? 0.f : __builtin_amdgcn_exp2f(m - M), lw = ml(w, 1, col);
                    lt += m == MINUS_INF ? lw : lw * fw;      // (no maximum: 0, or NaN where scores were)
                    if (m != MINUS_INF) acc += *reinterpret_cast<const f4 *>(reinterpret_cast<const float *>(lds + w * C::WAVE_B) + cc * OS + d) * fw;
                }
                const size_t row = row_index(at);
                if (pieces > 1) {
                    if (d == 0) {
                        float * pm = P.part_ml + (row * P.nks + piece) * 2;
                        pm[0] = part_ref(M, lt);
                        pm[1] = lt;
                    }
                    if (part_ref(M, lt) != MINUS_INF) *reinterpret_cast<f4 *>(P.part_o + (row * P.nks + piece) * D + d) = acc;
                    continue;
                }
                if (P.lse && d == 0) P.lse[row] = (M + log2f(lt)) * LN2;
                f4 v = acc * (lt == 0.f ? 0.f : 1.0f / lt);   // (nothing seen: 0)
                if (P.gate) {
                    const f4 gt = *reinterpret_cast<const f4 *>(P.gate + row * D + d);
#pragma unroll
                    for (int y = 0; y < 4; ++y) v[y] *= gate_of(gt[y]);
                }
                put4(P.out, P.out_bf16, row * D + d, v);
            }
        }
    }
    if (P.nks > 1 && piece == 0 && hk == 0 && tid == 0) P.part_n[f.seq * P.max_groups + f.group] = pieces;
    __syncthreads();                                          // (what was folded is read; the next group's V goes there)
  }
}

// Partials of a row -> its result: 256 / (D / 4) rows of one sequence a workgroup, four dims a thread
struct tree_merge_params {
    rows_view R;
    const float * part_o, * part_ml, * gate;
    void * out;
    float * lse;
    int Hq, GQA, D, nks, out_bf16, BC, max_groups;
    const int * part_n;    // [n_seq][max_groups] partials of a group's rows (1: they are finished)
};
__global__ void __launch_bounds__(NTHR) tree_merge_k(const tree_merge_params P) {
    const int tpr = P.D >> 2, per = NTHR / tpr, sub = threadIdx.x / tpr, d = 4 * (threadIdx.x - sub * tpr);
    item_at at;
    if (!find_item(P.R, blockIdx.x, P.Hq, per, threadIdx.x & 63, at)) return;
    const int r = at.index * per + sub;                       // of the sequence
    if (r >= (long long) at.v.count * P.Hq) return;
    const int t = r / P.Hq, h = r - t * P.Hq;
    const shape sh = shape_of(at.v.count, P.GQA, P.BC);
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
        for (int i = 0; i < 4; ++i) v[i] *= gate_of(gt[i]);
    }
    put4(P.out, P.out_bf16, e, v);
}

template <uint32_t KT, int D, int NT, bool EXACT> int launch_cfg(const tree_params & P, unsigned grid, hipStream_t s) {
    constexpr int lds = tree_cfg<KT, D, NT, EXACT>::LDS;
    // (the attribute belongs to the function on ONE device: remembered per device, set again on another)
    static std::atomic<uint32_t> attr_set{0};
    int dev = 0;
    (void) hipGetDevice(&dev);
    const uint32_t bit = 1u << (dev & 31);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        if (hipFuncSetAttribute((const void *) tree_k<KT, D, NT, EXACT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
            (void) hipGetLastError();
            set_error("p1a_attn_tree: cannot reserve %d bytes of LDS", lds);
            return P1A_E_LAUNCH;
        }
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    tree_k<KT, D, NT, EXACT><<<grid, NTHR, lds, s>>>(P);
    return launched();
}
template <uint32_t KT, int D> int launch_d(const tree_params & P, int NT, bool exact, unsigned grid, hipStream_t s) {
    if (NT == 1) return exact ? launch_cfg<KT, D, 1, true>(P, grid, s) : launch_cfg<KT, D, 1, false>(P, grid, s);
    return exact ? launch_cfg<KT, D, 2, true>(P, grid, s) : launch_cfg<KT, D, 2, false>(P, grid, s);
}
template <uint32_t KT> int launch_kt(const tree_params & P, int D, int NT, bool exact, unsigned grid, hipStream_t s) {
    return D == 256 ? launch_d<KT, 256>(P, NT, exact, grid, s) : D == 128 ? launch_d<KT, 128>(P, NT, exact, grid, s) : launch_d<KT, 64>(P, NT, exact, grid, s);
}
// workgroups of a compute unit: as tree_cfg has it
template <uint32_t KT> int wgs_kt(int D, int NT, bool exact) {
    auto of = [&](auto d) { constexpr int X = decltype(d)::value; return NT == 1 ? exact ? tree_cfg<KT, X, 1, true>::WGS : tree_cfg<KT, X, 1, false>::WGS : exact ? tree_cfg<KT, X, 2, true>::WGS : tree_cfg<KT, X, 2, false>::WGS; };
    return D == 256 ? of(std::integral_constant<int, 256>{}) : D == 128 ? of(std::integral_constant<int, 128>{}) : of(std::integral_constant<int, 64>{});
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
    pl.NT = (long long) R.max_rows * GQA <= 16 ? 1 : 2;
    const shape sh = shape_of(R.max_rows, GQA, 16 * pl.NT);
    pl.max_groups = sh.groups;
    pl.nks = 1;
    const long long groups = (long long) R.n_seq * sh.groups;
    pl.runs = (int) groups;
    const int wgs = c.type == P1A_KV_F16 ? wgs_kt<P1A_KV_F16>(c.D, pl.NT, exact) : c.type == P1A_KV_Q8_0 ? wgs_kt<P1A_KV_Q8_0>(c.D, pl.NT, exact) : wgs_kt<P1A_KV_Q4_0>(c.D, pl.NT, exact);
    const long long slots = (long long) std::max(cus, 1) * wgs, units = groups * c.Hkv;
    const long long keys = R.window == INT32_MAX ? max_n : std::min<long long>(max_n, (long long) R.window + R.max_rows + R.n_sink);
    const long long nt = std::max<long long>(((keys + 31) / 32 + sh.ks - 1) / sh.ks, 1);
    const size_t rows = (size_t) R.T * Hq, row_bytes = (size_t) c.D * 4 + 8;
    const long long runs = std::min(std::max(slots / c.Hkv, 1LL), groups * nt), per = (groups * nt + runs - 1) / runs;
    const long long most = std::min({64LL, runs, nt + 1, (128LL << 20) / (long long) (rows * row_bytes)});
    if (most > 1 && (units + slots - 1) / slots * (nt + 3) > std::max(per, (nt + most - 2) / (most - 1)) + 8) {
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
    if (steps > 1 << 30 || grid > 0x7fffffffLL) { set_error("p1a_attn_tree: too many positions and nodes for one call"); return P1A_E_SHAPE; }
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
    const int rc = c.type == P1A_KV_F16 ? launch_kt<P1A_KV_F16>(P, c.D, pl.NT, exact, (unsigned) grid, s)
                 : c.type == P1A_KV_Q8_0 ? launch_kt<P1A_KV_Q8_0>(P, c.D, pl.NT, exact, (unsigned) grid, s) : launch_kt<P1A_KV_Q4_0>(P, c.D, pl.NT, exact, (unsigned) grid, s);
    if (rc != P1A_OK || P.nks == 1) return rc;
    const tree_merge_params M{a.R, P.part_o, P.part_ml, a.gate, a.out, a.lse, a.Hq, P.GQA, c.D, P.nks, a.out_bf16, 16 * pl.NT, pl.max_groups, P.part_n};
    tree_merge_k<<<(unsigned) item_bound(a.R, a.Hq, NTHR / (c.D / 4)), NTHR, 0, s>>>(M);
    return launched();
}

}   // namespace p1a
