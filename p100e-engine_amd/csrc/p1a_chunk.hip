// Attention of the new tokens of several sequences over their paged caches - from one token each to whole prompts, ragged, with a sliding window and
// first positions that stay visible - for gfx950.
//
// Work: a block is 128 consecutive rows of one sequence and kv head (row r: token r / GQA under q head r % GQA of the group); a workgroup of four
// waves owns one, wave w the 32 rows from 32 w on, and walks the tiles of keys that any of its rows sees: the sinks' and the window's. Calls of few
// blocks deal a block's tiles to several workgroups, whose partials a second kernel merges.
// Arithmetic: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_f16, sums in fp32, one pass with a running reference r of every row:
// P = exp2(scale log2 e S - r), O and l are sums over P and rescaled when the row's maximum comes out of [r + 8 - inf, r + 14]. Where results are f32, q and P
// are two f16 halves (EXACT) and quantized K and V two planes (p1a_tiles.hpp): 2 products for f16 caches, 3 for quantized ones (low times low is 2^-22
// of the result and left out). P runs up to 2^14, so its low halves end 2^-38 below the largest weight.
// What bounds it, heads of 256 and f16: a tile of 64 keys asks LDS for as many clocks as the matrix pipe - 256 KB, as every wave reads all of K and V, and 64 products
// of a wave: 2048 each -, and with a wave to a SIMD (O and Q fill the registers) whatever is not hidden behind that wave's own products waits: 4096 tokens of a
// document through a window of 4096 (24 / 4 heads, bf16 out) keep the pipe busy for 36 % of the time, the waves wait for 39 %; without the loads they took a fifth
// less. They take 508 to 600 us by card, 700 to 820 TFLOP/s (a large product of the vendor's library: 1130, 370 us at that rate); eight prompts of 77 ... 2003
// tokens 280 to 310. (p1a_prefill.hip, a wave to a SIMD too, shares V between two waves, 1536 clocks of LDS, and reaches 1.1 PFLOP/s.)
#include "p1a_tiles.hpp"

#include <algorithm>
#include <atomic>

namespace p1a {
namespace {

constexpr int BM = 128, NTHR = 256;

template <uint32_t KT, int D, bool EXACT> struct chunk_cfg {
    static constexpr int NPL = group_planes(KT, EXACT);
    // keys of a tile, by what registers hold: scores of this tile and the next, P, and a quantized tile on its way
    static constexpr int BN = D >= 128 && (EXACT || KT != P1A_KV_F16) ? 32 : 64;
    static constexpr int NG = BN / 16, G_B = NPL * plane_bytes(D), STAGE_B = 2 * NG * G_B;
};

template <uint32_t KT, int D, bool EXACT>
__global__ void __launch_bounds__(NTHR, D <= 128 ? 2 : 1) chunk_k(const chunk_params P) {
    using C = chunk_cfg<KT, D, EXACT>;
    using G = group<KT, D, C::NPL>;
    constexpr int BN = C::BN, NG = C::NG, G_B = C::G_B, PL_B = plane_bytes(D), NPL = C::NPL;
    constexpr int NKS = D / 16, NDT = D / 32, NH = BN / 32, NQ = EXACT ? 2 : 1, PF_K = NPL == 2 ? 1 : EXACT ? 2 : 4, PF_V = NPL == 2 ? 1 : EXACT ? 2 : 3;
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, g = lane >> 5;
    // kv heads side by side (their XCDs), then the splits of a block, then blocks
    const int item = blockIdx.x / P.Hkv, hk = blockIdx.x - item * P.Hkv, bi = item / P.nks, ksp = item - bi * P.nks;
    item_at at;
    if (!find_item(P.R, bi, P.GQA, BM, lane, at)) return;
    const int nrows = at.v.count * P.GQA, row0 = (at.of - 1 - at.index) * BM;   // (the blocks that see most first)
    const int wrow0 = row0 + 32 * wave, wrows = min(32, nrows - wrow0);
    auto tok_of = [&](int r) {                                // (the multiplication is at most one short)
        const int t = (int) __umulhi((uint32_t) r, P.gqa_magic);
        return r - t * P.GQA >= P.GQA ? t + 1 : t;
    };
    auto row_index = [&](int r) { const int t = tok_of(r); return (size_t) (at.v.first + t) * P.Hq + (size_t) hk * P.GQA + (r - t * P.GQA); };
    const bool live = c < wrows;
    const int my_row = wrow0 + min(c, max(wrows, 1) - 1), my_tok = tok_of(min(my_row, nrows - 1));
    int my_pos = at.v.pos0 + my_tok;
    if (!live || my_pos < 0 || my_pos >= P.R.n_ctx) my_pos = -1;   // sees nothing
    const size_t my_index = row_index(min(my_row, nrows - 1));

    const span sp = span_of<BN>(P.R, at.v.pos0 + tok_of(row0), at.v.pos0 + tok_of(min(row0 + BM, nrows) - 1));
    const int tps = (sp.nt + P.nks - 1) / P.nks, ta = min(ksp * tps, sp.nt), tb = min(ta + tps, sp.nt);
    // positions that every row of the wave sees: up to all_hi, from all_lo on (rows stand at consecutive positions; none where one of them sees nothing)
    const int all_hi = __builtin_amdgcn_readlane(my_pos, 0), last_pos = __builtin_amdgcn_readlane(my_pos, max(wrows, 1) - 1);
    const int all_lo = all_hi < 0 || last_pos < 0 ? INT32_MAX : P.R.window == INT32_MAX ? 0 : max(last_pos - P.R.window + 1, 0);

    // ---- where rows of the cache are ----
    const int32_t * const ptab = P.pg.pt ? P.pg.pt + (P.pg.rtab ? sload_i32(P.pg.rtab + at.seq) : 0) : nullptr;
    const size_t head_off = (size_t) hk * head_bytes(KT, D);
    // BN = 64: wave w fills group w of K and V; 32: groups 0 and 1 of K (waves 0, 1) and of V (waves 2, 3)
    constexpr bool BOTH = BN == 64;
    const int grp = BOTH ? wave : wave & 1, my_key = 16 * grp + G::key(lane);
    const bool my_v = !BOTH && wave >= 2;
    auto pos_of = [&](int tile) { return seen_or_near<BN>(sp, tile * BN, tile * BN + my_key); };
    auto page_of = [&](int tile) { return ptab ? ptab[pos_of(tile) >> P.pg.psh] : 0; };
    auto row_of = [&](int tile, int page) {
        const int j = pos_of(tile);
        return head_off + (ptab ? (size_t) page * P.pg.pstride + (size_t) (j & ((1 << P.pg.psh) - 1)) * P.pg.rowb : (size_t) j * P.pg.rowb);
    };
    auto k_groups = [&](int st) { return lds + st * C::STAGE_B; };
    auto v_groups = [&](int st) { return lds + st * C::STAGE_B + NG * G_B; };

    // ---- Q^T operands: lane (row c, half g) holds dims 16 ks + 8 g .. + 7 ----
    h8 qf[NQ][NKS];
    float factor = P.factor;
    auto load_q = [&] {
        f4 x[NKS][2];
        float most = 0.f;
        auto fetch = [&](auto as_bf16) {
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) x[ks][e] = q4_at(P.q, as_bf16, my_index * D + 16 * ks + 8 * g + 4 * e);
        };
        if (P.q_bf16) fetch(std::true_type{});
        else fetch(std::false_type{});
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[ks][e >> 2][e & 3]));
        const int ex = row_exponent(max_swap32(most));
        factor = ldexpf(factor, ex);
        const float by = ldexpf(P.sign, -ex);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            h8 r[NQ];
            halves<NQ>([&](int e) { return x[ks][e >> 2][e & 3]; }, [&](int) { return by; }, r);
#pragma unroll
            for (int k = 0; k < NQ; ++k) {
                qf[k][ks] = r[k];
                // (in accumulation registers, where the products read it as it is: what vector instructions work on has the others)
                if constexpr (D == 256) asm volatile("" : "+a"(qf[k][ks]));
            }
        }
    };

    f16x o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    float ref = MINUS_INF, l = 0.f;

    const k_frag kf(lane, G_B);
    const v_frag vf(lane);
    // (stage: its place in LDS as a number the compiler does not see through - offsets from it fit the instructions, those from the start do not)
    auto stage_of = [&](int st) {
        int at = st * C::STAGE_B;
        asm volatile("" : "+s"(at));
        return (const char *) lds + at;
    };
    auto k_read = [&](const char * stage, int k, int pl) { return kf.read(stage + 2 * (k / NKS) * G_B + pl * PL_B, k % NKS); };
    auto v_read = [&](const char * stage, int f, int pl) { return vf.read(stage + NG * G_B + (f / NDT) * G_B + pl * PL_B, f % NDT); };

    // ---- S^T of one tile: product k of NH * NKS ----
    auto s_product = [&](f16x (&s)[NH], int k, const h8 (&a)[NPL]) {
        const int u = k / NKS, ks = k % NKS;
        if (ks == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
        }
        s[u] = mfma32(a[0], qf[0][ks], s[u]);
        if constexpr (EXACT) s[u] = mfma32(a[0], qf[NQ - 1][ks], s[u]);
        if constexpr (NPL == 2) s[u] = mfma32(a[NPL - 1], qf[0][ks], s[u]);
    };
    // what a row does not see, where a row of the wave does not see all of the tile
    auto mask = [&](f16x (&s)[NH], int k0) {
        const int from = k0 + 4 * g;
        int hi = my_pos - from, lo = max(my_pos - k0, 0) - P.R.window - 4 * g, sk = P.R.n_sink - from;
        asm volatile("" : "+v"(hi), "+v"(lo), "+v"(sk));      // (or the comparisons would be made ahead of the branch, for every tile)
#pragma unroll
        for (int u = 0; u < NH; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = 32 * u + mfma_row(i, 0);        // (and 4 g: a number the comparison holds itself)
                s[u][i] = j <= hi && (j > lo || j < sk) ? s[u][i] : MINUS_INF;
            }
    };
    float top = -MINUS_INF;
    asm volatile("" : "+s"(top));
    auto most_of = [&](const f16x (&s)[NH]) {
        float m = MINUS_INF;
#pragma unroll
        for (int u = 0; u < NH; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) m = larger(m, s[u][i], top);
        return m;
    };
    auto whole = [&](int k0) { return k0 + BN - 1 <= all_hi && k0 >= all_lo; };
    float mx = MINUS_INF;                                     // the row's largest score of the tile in hand

    constexpr int NPC = (BOTH ? 2 : 1) * G::PIECES;           // loads of a step
    // ---- a step: P of this tile beside the products S^T of the next one, then O^T beside the next one's maximum. The loads of K two tiles on and V one
    // tile on are under way meanwhile ----
    auto step = [&](int st, int next, f16x (&s)[NH], f16x (&sn)[NH], auto && piece) __attribute__((always_inline)) {
        const char * const here = stage_of(st), * const after = stage_of(st ^ 1);
        const bool fresh = ref == MINUS_INF, move = mx > (fresh ? MINUS_INF : ref + (HEAD + STEP));
        if (__builtin_expect(__any(move), 0)) {
            const float to = move ? mx - HEAD : ref, alpha = fresh ? 1.f : __builtin_amdgcn_exp2f(ref - to);   // (fresh: nothing accumulated)
            ref = to;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
        }
        const float nr = ref == MINUS_INF ? 0.f : -ref;       // (a row that has seen nothing: exp2(-inf))
        constexpr int NK = NH * NKS, NF = NG * NDT, NV = NH * 16;
        h8 pb[NQ][2 * NH];
        float ls[2] = {0.f, 0.f};
        // (operands from LDS are asked for a few products ahead, and no further: registers)
        h8 fr[PF_K][NPL];
#pragma unroll
        for (int k = 0; k < PF_K; ++k)
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) fr[k][pl] = k_read(after, k, pl);
        static_assert(NPC <= NK);
        each<NK>([&](auto k) __attribute__((always_inline)) {
            h8 a[NPL];
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) {
                a[pl] = fr[k % PF_K][pl];
                if (k + PF_K < NK) fr[k % PF_K][pl] = k_read(after, k + PF_K, pl);
            }
            s_product(sn, k, a);
            // (a load now and then: one behind the other they would hold the wave for as long as the compute unit takes for all of them)
            if constexpr (k * NPC % NK < NPC) piece(std::integral_constant<int, k * NPC / NK>{});
#pragma unroll
            for (int v = k * NV / NK / 2 * 2; v < (k + 1) * NV / NK / 2 * 2; v += 2) {   // pairs of values of P
                const int u = v >> 4, i = v & 15;
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[u][i], factor, nr)), p1 = __builtin_amdgcn_exp2f(fmaf(s[u][i + 1], factor, nr));
                ls[0] += p0;
                ls[1] += p1;
                asm volatile("" : "+v"(ls[0]), "+v"(ls[1]));  // (here: put off, all of P would stay in registers)
                h2 h = __builtin_convertvector(f2w{p0, p1}, h2);
                asm("" : "+v"(h));
                pb[0][2 * u + (i >> 3)][i & 7] = h[0];
                pb[0][2 * u + (i >> 3)][(i & 7) + 1] = h[1];
                if constexpr (EXACT) {
                    pb[NQ - 1][2 * u + (i >> 3)][i & 7] = (half_t) (p0 - (float) h[0]);
                    pb[NQ - 1][2 * u + (i >> 3)][(i & 7) + 1] = (half_t) (p1 - (float) h[1]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        l += ls[0] + ls[1];
        h8 fv[PF_V][NPL];
#pragma unroll
        for (int f = 0; f < PF_V; ++f)
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) fv[f][pl] = v_read(here, f, pl);
        mx = MINUS_INF;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int ps = f / NDT, dt = f % NDT;
            h8 a[NPL];
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl) {
                a[pl] = fv[f % PF_V][pl];
                if (f + PF_V < NF) fv[f % PF_V][pl] = v_read(here, f + PF_V, pl);
            }
            o[dt] = mfma32(a[0], pb[0][ps], o[dt]);
            if constexpr (EXACT) o[dt] = mfma32(a[0], pb[NQ - 1][ps], o[dt]);
            if constexpr (NPL == 2) o[dt] = mfma32(a[NPL - 1], pb[0][ps], o[dt]);
#pragma unroll
            for (int v = f * NV / NF; v < (f + 1) * NV / NF; ++v) mx = larger(mx, sn[v >> 4][v & 15], top);
            asm volatile("" : "+v"(mx));
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_expect(!whole(next * BN), 0)) {
            mask(sn, next * BN);
            mx = most_of(sn);
        }
        mx = max_swap32(mx) * factor;
    };

    // ---- the walk. Stage i & 1 holds K of tile i and V of tile i; page-table entries are asked for a tile ahead of the rows ----
    // 64-key tiles: a wave has its group of K and of V; 32: one of the two
    typename G::raw rk, rv;
    const gbytes k_from = (gbytes) (my_v ? P.vc : P.kc), v_from = (gbytes) P.vc;
    // load y of those of a step: K of its tile + 2 into stage k_st, V of its tile + 1 into the other one
    auto piece = [&](auto y, int k_st, size_t row_k, size_t row_v) __attribute__((always_inline)) {
        if constexpr (BOTH && y >= G::PIECES) G::template piece<y - G::PIECES>(rv, v_from + row_v, v_groups(k_st ^ 1) + grp * G_B, lane);
        else G::template piece<y>(rk, k_from + (my_v ? row_v : row_k), (my_v ? v_groups(k_st ^ 1) : k_groups(k_st)) + grp * G_B, lane);
    };
    auto put = [&](int k_st) {                                // (what came through registers)
        if constexpr (!G::DIRECT) {
            G::store(rk, (my_v ? v_groups(k_st ^ 1) : k_groups(k_st)) + grp * G_B, lane);
            if constexpr (BOTH) G::store(rv, v_groups(k_st ^ 1) + grp * G_B, lane);
        }
    };
    auto done = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    if (ta < tb) {
        auto tile = [&](int i) { return sp.tile(min(i, tb - 1)); };          // (past the last: that one once more, unused)
        int page = page_of(tile(ta)), page1 = page_of(tile(ta + 1));
        size_t row_v = row_of(tile(ta), page), row_k = row_of(tile(ta + 1), page1);
        page = page_of(tile(ta + 2));
        // K of the first tile into stage 0 (quantized: and V into stage 1, where nobody looks at it), then K of the second and V of the first
        each<G::DIRECT ? G::PIECES : NPC>([&](auto y) __attribute__((always_inline)) { piece(y, 0, row_v, row_v); });
        if constexpr (!G::DIRECT) put(0);
        each<NPC>([&](auto y) __attribute__((always_inline)) { piece(y, 1, row_k, row_v); });
        load_q();
        if constexpr (!G::DIRECT) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else done();
        f16x sa[NH], sb[NH];
        if (wrows > 0) {
#pragma unroll
            for (int k = 0; k < NH * NKS; ++k) {
                h8 a[NPL];
#pragma unroll
                for (int pl = 0; pl < NPL; ++pl) a[pl] = k_read(lds, k, pl);
                s_product(sa, k, a);
            }
            if (!whole(tile(ta) * BN)) mask(sa, tile(ta) * BN);
            mx = max_swap32(most_of(sa)) * factor;
        }
        put(1);
        done();
        // tile i: K(i + 1) and V(i) are there; K(i + 2) goes where K(i) was, V(i + 1) where V(i - 1) was
        auto turn = [&](int i, int st, f16x (&s)[NH], f16x (&sn)[NH]) __attribute__((always_inline)) {
            row_v = row_k;
            row_k = row_of(tile(i + 2), page);
            page = page_of(tile(i + 3));
            if (wrows > 0) step(st, tile(i + 1), s, sn, [&](auto y) __attribute__((always_inline)) { piece(y, st, row_k, row_v); });
            else each<NPC>([&](auto y) __attribute__((always_inline)) { piece(y, st, row_k, row_v); });
            put(st);
            done();
        };
        for (int i = ta;;) {
            turn(i, 0, sa, sb);
            if (++i == tb) break;
            turn(i, 1, sb, sa);
            if (++i == tb) break;
        }
    }

    // ---- results: lane (row c, half g) holds dims 32 dt + 8 (i / 4) + 4 g + i % 4 ----
    l += __shfl_xor(l, 32);
    if (!live) return;
    if (P.nks > 1) {
        float * ml = P.part_ml + (my_index * P.nks + ksp) * 2;
        if (g == 0) { ml[0] = part_ref(ref, l); ml[1] = l; }
        if (part_ref(ref, l) == MINUS_INF) return;            // (nothing seen: the merge does not look at it)
        float * po = P.part_o + (my_index * P.nks + ksp) * D;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<f4 *>(po + 32 * dt + 8 * q + 4 * g) = f4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
        return;
    }
    const float inv = my_pos < 0 ? 0.f : 1.0f / l;
    if (P.lse && g == 0) P.lse[my_index] = (ref + log2f(l)) * LN2;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const size_t e = my_index * D + 32 * dt + 8 * q + 4 * g;
            f4 v = f4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]} * inv;
            if (P.gate) {
                const f4 gt = *reinterpret_cast<const f4 *>(P.gate + e);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] *= gate_of(gt[i]);
            }
            put4(P.out, P.out_bf16, e, v);
        }
}

// Partials of a row -> its result: 256 / (D / 4) rows of one sequence a workgroup, four dims a thread
struct chunk_merge_params {
    rows_view R;
    const float * part_o, * part_ml, * gate;
    void * out;
    float * lse;
    int Hq, D, nks, out_bf16;
    const int * part_n;    // few rows: partials that each sequence has (1: its rows are finished), or null: nks
};
__global__ void __launch_bounds__(NTHR) chunk_merge_k(const chunk_merge_params P) {
    const int tpr = P.D >> 2, per = NTHR / tpr, sub = threadIdx.x / tpr, d = 4 * (threadIdx.x - sub * tpr);
    item_at at;                                               // (whose rows they are: as the kernels that left the partials find it, whatever row0 holds)
    if (!find_item(P.R, blockIdx.x, P.Hq, per, threadIdx.x & 63, at)) return;
    const int r = at.index * per + sub;                       // of the sequence
    if (r >= (long long) at.v.count * P.Hq) return;
    const long long row = (long long) at.v.first * P.Hq + r;
    const int n = P.part_n ? min(P.part_n[at.seq], P.nks) : P.nks;
    if (n < 2) return;                                        // (finished already)
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
    const int pos = at.v.pos0 + r / P.Hq;
    if (P.lse && d == 0) P.lse[row] = (M + log2f(l)) * LN2;
    f4 v = acc * (pos < 0 || pos >= P.R.n_ctx ? 0.f : 1.0f / l);
    const size_t e = (size_t) row * P.D + d;
    if (P.gate) {
        const f4 gt = *reinterpret_cast<const f4 *>(P.gate + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= gate_of(gt[i]);
    }
    put4(P.out, P.out_bf16, e, v);
}

template <uint32_t KT, int D, bool EXACT> int launch_cfg(const chunk_params & P, unsigned grid, hipStream_t s) {
    constexpr int lds = 2 * chunk_cfg<KT, D, EXACT>::STAGE_B;
    // (the attribute belongs to the function on ONE device: remembered per device, set again on another)
    static std::atomic<uint32_t> attr_set{0};
    int dev = 0;
    (void) hipGetDevice(&dev);
    const uint32_t bit = 1u << (dev & 31);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        if (hipFuncSetAttribute((const void *) chunk_k<KT, D, EXACT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
            (void) hipGetLastError();
            set_error("p1a_attn_chunk: cannot reserve %d bytes of LDS", lds);
            return P1A_E_LAUNCH;
        }
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    chunk_k<KT, D, EXACT><<<grid, NTHR, lds, s>>>(P);
    return launched();
}
template <uint32_t KT, int D> int launch_d(const chunk_params & P, bool exact, unsigned grid, hipStream_t s) {
    return exact ? launch_cfg<KT, D, true>(P, grid, s) : launch_cfg<KT, D, false>(P, grid, s);
}
template <uint32_t KT> int launch_kt(const chunk_params & P, int D, bool exact, unsigned grid, hipStream_t s) {
    return D == 256 ? launch_d<KT, 256>(P, exact, grid, s) : D == 128 ? launch_d<KT, 128>(P, exact, grid, s) : launch_d<KT, 64>(P, exact, grid, s);
}

// the most items of `unit` that the sequences' rows times `mul` can make (as find_item counts them)
long long item_bound(const rows_view & R, int mul, int unit) {
    const long long each = ((long long) R.max_rows * mul + unit - 1) / unit * R.n_seq;
    return R.row0 ? std::min(each, (long long) R.T * mul / unit + R.n_seq) : each;
}
// the most blocks the rows can make
long long block_bound(const rows_view & R, int GQA) { return item_bound(R, GQA, BM); }

}   // namespace

// How a call is dealt out, from its host numbers and the device. Up to 32 rows of a sequence under a kv head take the kernel of p1a_step.hip (one token over
// 260 keys, 4 / 1 heads of 64: 7 us, as a block 9 and 2 of merging; 32 tokens through 4096 keys, 24 / 4 of 256, q8_0: 52 + 5, as blocks 164 + 5).
//   blocks of rows: the number of workgroups that share a block's keys minimises rounds of workgroups x (64-key tiles of a workgroup + 3 for its set-up and
//     results), and 3 for a merge (four turns of 17 ... 150 tokens through a window of 2048, 32 / 8 of 128, q4_0: 52 + 8 us, unsplit 110; 24 sequences of
//     1 ... 500 tokens over 500 ... 7000 keys, f16: 147 + 19, unsplit 225).
//   few rows: as many runs of 128-key steps as there are places for workgroups, unless one for each sequence takes no longer than a run, its
//     set-up (3), a second sequence's (2) and the merge (3) (the 32 tokens: 52 + 5 us, a workgroup for each sequence 109).
// Partials take 64 MB (few rows) and 256 MB (blocks) at most: fewer to a row where there are many rows, none where two would be more. They go by T, rows of no
// sequence among them.
chunk_plan plan_chunk(const p1a_kv & c, const rows_view & R, int Hq, int max_n, int cus) {
    const int GQA = Hq / c.Hkv;
    chunk_plan pl{};
    pl.few = (long long) R.max_rows * GQA <= 32 ? (R.max_rows * GQA + 15) / 16 : 0;
    pl.runs = R.n_seq;
    const int step = pl.few ? 128 : 64;
    const bool two = c.D <= 128 || (pl.few == 1 && c.type != P1A_KV_F16);   // two workgroups to a compute unit
    const long long units = (pl.few ? R.n_seq : block_bound(R, GQA)) * c.Hkv, slots = (long long) std::max(cus, 1) * (two ? 2 : 1);
    const long long keys = R.window == INT32_MAX ? max_n : std::min<long long>(max_n, (long long) R.window + std::min(R.max_rows, BM / GQA + 1) + R.n_sink);
    const long long nt = std::max<long long>((keys + step - 1) / step, 1);
    const size_t rows = (size_t) R.T * Hq, row_bytes = (size_t) c.D * 4 + 8;
    if (pl.few) {
        pl.nks = 1;
        const long long runs = std::min(std::max(slots / c.Hkv, 1LL), R.n_seq * nt), per = (R.n_seq * nt + runs - 1) / runs;
        const long long most = std::min({64LL, runs, nt + 1, (64LL << 20) / (long long) (rows * row_bytes)});
        if (most > 1 && (units + slots - 1) / slots * (nt + 3) > std::max(per, (nt + most - 2) / (most - 1)) + 8) {
            pl.runs = (int) runs;
            pl.nks = (int) most;
        }
    } else {
        auto cost = [&](long long k) { return (units * k + slots - 1) / slots * ((nt + k - 1) / k + 3) + (k > 1 ? 3 : 0); };
        long long best = 1;
        for (long long k = 2; k <= std::min({64LL, nt, (256LL << 20) / (long long) (rows * row_bytes), 0xffffffLL / units}); ++k) if (cost(k) < cost(best)) best = k;
        pl.nks = (int) best;
    }
    if (pl.nks > 1) {
        pl.bytes_n = pl.few ? ((size_t) R.n_seq * 4 + 255) & ~(size_t) 255 : 0;
        pl.bytes_ml = (rows * pl.nks * 8 + 255) & ~(size_t) 255;
        pl.bytes_o = rows * pl.nks * c.D * 4;
    }
    return pl;
}

int launch_chunk(const p1a_kv & c, const chunk_args & a, hipStream_t s) {
    chunk_params P;
    P.q = a.q; P.out = a.out; P.gate = a.gate; P.lse = a.lse;
    P.kc = (const char *) c.k; P.vc = (const char *) c.v; P.pg = view_of(c); P.R = a.R;
    P.Hq = a.Hq; P.Hkv = c.Hkv; P.GQA = a.Hq / c.Hkv;
    P.gqa_magic = (uint32_t) (P.GQA == 1 ? (1ull << 32) - 1 : (1ull << 32) / (unsigned) P.GQA);
    P.factor = a.scale == 0.f ? 1.f : (a.scale < 0 ? -a.scale : a.scale) * LOG2E;
    P.sign = a.scale == 0.f ? 0.f : a.scale < 0 ? -1.f : 1.f;
    P.q_bf16 = a.q_bf16; P.out_bf16 = a.out_bf16;
    const chunk_plan pl = plan_chunk(c, a.R, a.Hq, a.max_n, cu_count());
    P.nks = pl.nks; P.runs = pl.runs;
    P.part_o = P.part_ml = nullptr; P.part_n = nullptr;
    const size_t rows = (size_t) a.R.T * a.Hq;
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
    const long long grid = pl.few ? 0 : block_bound(a.R, P.GQA) * P.nks * c.Hkv;   // (up to 2^23 blocks of rows and one more for each of 2^22 pairs: below 2^24)
    const bool exact = !a.out_bf16 || a.lse;
    const int rc = pl.few ? launch_step(c, P, pl.few, exact, s) : c.type == P1A_KV_F16 ? launch_kt<P1A_KV_F16>(P, c.D, exact, (unsigned) grid, s)
                 : c.type == P1A_KV_Q8_0 ? launch_kt<P1A_KV_Q8_0>(P, c.D, exact, (unsigned) grid, s) : launch_kt<P1A_KV_Q4_0>(P, c.D, exact, (unsigned) grid, s);
    if (rc != P1A_OK || P.nks == 1) return rc;
    const chunk_merge_params M{a.R, P.part_o, P.part_ml, a.gate, a.out, a.lse, a.Hq, c.D, P.nks, a.out_bf16, pl.few ? P.part_n : nullptr};
    chunk_merge_k<<<(unsigned) item_bound(a.R, a.Hq, NTHR / (c.D / 4)), NTHR, 0, s>>>(M);
    return launched();
}

}   // namespace p1a
