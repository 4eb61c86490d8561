// Attention weight per cache position (gfx950): mass[s][h][j] += sum over a call's rows t and the heads i of kv head h of exp(scale q_ti . k_j - lse_ti).
// No two waves add to the same entry, no atomic orders the sums; weights and sums in fp32, q in two f16 halves.
//
// Few rows (32 columns a sequence at most), mass_step_k: reading K is what it costs. Runs of steps of equal length as in p1a_step.hip; a wave holds q and
// walks tiles of 32 keys, K straight into the operands of v_mfma_f32_16x16x32_f16, codes as whole numbers; a key's weights are added over the 16 lanes of its
// columns and its entry written at once.
// Many rows, mass_k: a wave owns 32 NU keys - their rows stay in its registers as operands of v_mfma_f32_32x32x16_f16, quantized ones in two planes
// (p1a_tiles.hpp) - and walks the rows of q that may see them, 32 at a time; a key's sum stays with one lane until the end. The workgroup's eight
// waves (256 NU keys) share the rows: fetched, brought to two halves and put into LDS once for all; with NU = 2 a half read from LDS feeds two products
// (one: LDS gives 128 bytes a clock and eight waves would ask for 128). Two workgroups of four waves a compute unit, which brought each row twice and had no
// registers left to ask for it ahead, took 417 us for four prompts of 300 ... 2003 tokens (24 / 4 heads of 256, f16); this takes 260 to 280. Where there are too few
// keys to fill the device, workgroups share the rows of a block of keys too, leave their sums, and mass_add_k adds them in order.
// What bounds it: the matrix pipe (2 products for f16 caches, 3 for quantized ones; 144 us of the 270 at a large product's rate) and, hardly beside it
// with two waves a SIMD, the exponentials and the rows' halves; over long caches (64 rows over 30011 keys, 32 / 8 heads of 128: 57 us) 8 us of
// a workgroup's 28 before its first product.
// Few rows: 32 sequences of 1000 ... 8190 keys (24 / 4 of 256, q8_0) 36 us, 4.5 TB/s of K and totals.
#include "p1a_tiles.hpp"

#include <algorithm>
#include <atomic>

namespace p1a {
namespace {

constexpr int NW = 4, NTHR = NW * 64, QR = 32;                // waves; rows of q at a time

struct mass_params {
    const void * q;
    const float * lse;
    float * mass;
    float * part;          // [splits][n_seq][Hkv][pld]: sums of the positions of the list of tiles, in its order
    const char * kc;
    kv_view pg;
    rows_view R;
    int Hq, Hkv, GQA, ld, pld, q_bf16;
    uint32_t gqa_magic;
    float factor, sign;
    int runs;              // few rows: workgroups of a kv head
    int blocks, splits;    // many rows: blocks of keys, workgroups that share the rows of one
};
__device__ __forceinline__ int token_of(const mass_params & P, int r) {   // (the multiplication is at most one short)
    const int t = (int) __umulhi((uint32_t) r, P.gqa_magic);
    return r - t * P.GQA >= P.GQA ? t + 1 : t;
}

// ---- few rows ----
template <int CTRL> __device__ __forceinline__ float add_dpp(float x) { return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true)); }
// over 16 lanes, in every one of them
__device__ __forceinline__ float add16(float x) { return add_dpp<0x140>(add_dpp<0x141>(add_dpp<0x4E>(add_dpp<0xB1>(x)))); }

template <uint32_t KT, int D, int NT>
__global__ void __launch_bounds__(NTHR, D == 256 && NT == 2 ? 1 : 2) mass_step_k(const mass_params P) {
    using K = keys16<KT, D>;
    constexpr int NB = D / 32;
    __shared__ __attribute__((aligned(16))) float tables[K::F16 ? 4 : NW * 2 * K::TAB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int xcd = blockIdx.x & 7, jx = blockIdx.x >> 3, hk = jx % P.Hkv, run = jx / P.Hkv * 8 + xcd;
    if (run >= P.runs) return;
    step_runs<NW> steps;
    if (!steps.begin(P.R, P.pg, run, P.runs, 1 << 30)) return;
    float * const tk = tables + (K::F16 ? 0 : wave * 2 * K::TAB);
    const size_t head_off = (size_t) hk * head_bytes(KT, D);

    for (int at_step = steps.first; at_step < steps.end;) {
        typename step_runs<NW>::found f;
        if (!steps.find(P.R, P.pg, at_step, lane, f)) return;
        const seq_view & sv = f.v;
        const int R = min(sv.count * P.GQA, 16 * NT);
        const span sp = step_runs<NW>::span_of_rows(P.R, sv);
        const int ta = (at_step - f.first) * NW, tb = min((min(steps.end, f.first + f.steps) - f.first) * NW, sp.nt);
        at_step = f.first + f.steps;
        const key_rows keys{sp, P.pg, P.pg.pt ? P.pg.pt + f.table : nullptr, head_off, c};
        float * const mass = P.mass + ((size_t) f.seq * P.Hkv + hk) * P.ld;
        // this lane's entry of a tile (the first eight lanes of a group write its eight keys), or -1
        auto entry = [&](int tile) {
            const int j = tile * 32 + 16 * (c >> 2) + 4 * g + (c & 3);
            return c < 8 && j <= sp.pmax && (j >= sp.lo || j < sp.ns) && j < P.ld ? j : -1;
        };
        typename K::raw kr[2];
        float old = 0.f;
        auto ask = [&](int tile, const key_rows::pages & e) {
            const key_rows::where at = keys.at(tile, e);
#pragma unroll
            for (int x = 0; x < 2; ++x) K::load(kr[x], (gbytes) P.kc + at.off[x], g);
            const int j = entry(tile);
            old = j >= 0 ? mass[j] : 0.f;
        };
        int i = ta + wave;
        if (i < tb) ask(sp.tile(i), keys.pages_of(sp.tile(i)));

        h8 qf[NT][2][NB];
        float factor[NT], lse[NT];
        int pos[NT], first_pos = INT32_MAX, last_pos = -1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = 16 * n + c, rr = min(r, R - 1), t = token_of(P, rr);
            const size_t row = (size_t) (sv.first + t) * P.Hq + (size_t) hk * P.GQA + (rr - t * P.GQA);
            factor[n] = ldexpf(P.factor, q_columns<KT, D, 2>(P.q, P.q_bf16, row, P.sign, g, qf[n]));
            const float z = P.lse[row];
            lse[n] = -z * LOG2E;
            pos[n] = sv.pos0 + t;
            if (r >= R || pos[n] < 0 || pos[n] >= P.R.n_ctx || z == MINUS_INF) pos[n] = -1;   // sees nothing
            first_pos = min(first_pos, pos[n]);
            last_pos = max(last_pos, pos[n]);
            __builtin_amdgcn_sched_barrier(0);
        }

        for (; i < tb; i += NW) {
            const int tile = sp.tile(i), k0 = tile * 32;
            const bool more = i + NW < tb;
            key_rows::pages pg;
            if (more) pg = keys.pages_of(sp.tile(i + NW));
            if constexpr (!K::F16) {
#pragma unroll
                for (int x = 0; x < 2; ++x) K::put(tk + x * K::TAB, kr[x].d, c, g);
                __builtin_amdgcn_wave_barrier();
            }
            f4 s[2][NT];
            K::template scores<NT, 2>(kr, [&](int n, int k, int b) { return qf[n][k][b]; }, tk, g, s);
            const float before = old;
            if (more) ask(sp.tile(i + NW), pg);
            const bool all = __all(k0 + 31 <= first_pos && k0 > last_pos - P.R.window);   // (every column sees every key)
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 0.f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int at = k0 + 4 * g, hi = pos[n] - at, lo = max(pos[n] - k0, 0) - P.R.window - 4 * g, sk = P.R.n_sink - at;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][n][e & 3], factor[n], lse[n]));
                    const int j = 16 * (e >> 2) + (e & 3);    // (and 4 g)
                    w[e] += all || (j <= hi && (j > lo || j < sk)) ? x : 0.f;
                }
            }
            float mine = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = add16(w[e]);
                if (c == e) mine = x;
            }
            const int j = entry(tile);
            if (j >= 0) mass[j] = before + mine;
        }
    }
}

// ---- many rows ----
constexpr int MW = 8, MTHR = MW * 64;                         // waves of a workgroup
template <uint32_t KT, int D> struct mass_cfg {
    static constexpr int NPL = group_planes(KT, true), NU = NPL == 2 && D == 256 ? 1 : 2, BK = MW * 32 * NU;
    static constexpr int G_B = NPL * plane_bytes(D);
    static constexpr int AT_ONCE = std::min(2 * NU, 16384 / G_B);            // groups of 16 keys of a wave on their way to its registers: 128 KB of LDS
    static constexpr int K_B = MW * AT_ONCE * G_B;
    static constexpr int Q_B = 2 * 2 * plane_bytes(D);        // 32 rows in two halves
    static constexpr int ROWS_AT = std::max(K_B, 4 * Q_B), LDS = ROWS_AT + 4 * QR * 12;   // (the rows go where the keys were)
};

template <uint32_t KT, int D>
__global__ void __launch_bounds__(MTHR, 2) mass_k(const mass_params P) {
    using C = mass_cfg<KT, D>;
    using G = group<KT, D, C::NPL>;
    constexpr int NPL = C::NPL, NU = C::NU, G_B = C::G_B, PL_B = plane_bytes(D), NKS = D / 16, NJ = (D + 127) / 128, TB = MW * NU;   // TB: tiles of a block
    extern __shared__ __attribute__((aligned(16))) char lds[];
    struct row_info { float factor, lse; int pos; };
    row_info * const info = reinterpret_cast<row_info *>(lds + C::ROWS_AT);   // [4][QR]

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // kv heads side by side, then the splits of a block, then blocks (those of the first keys, which most rows see, ahead)
    const int hk = blockIdx.x % P.Hkv, item = blockIdx.x / P.Hkv, split = item % P.splits, bx = item / P.splits, seq = blockIdx.y;
    const seq_view sv = seq_of<true>(P.R, seq);
    if (sv.count < 1) return;
    const span sp = span_of<32>(P.R, sv.pos0, sv.pos0 + sv.count - 1);   // tiles of 32 keys: a wave's NU are consecutive ones of the list
    const int32_t * const ptab = P.pg.pt ? P.pg.pt + (P.pg.rtab ? sload_i32(P.pg.rtab + seq) : 0) : nullptr;
    const size_t head_off = (size_t) hk * head_bytes(KT, D);
    const int nrows = sv.count * P.GQA;
    const size_t entries = (size_t) seq * P.Hkv + hk;
    float * const mass = P.splits > 1 ? P.part + ((size_t) split * P.R.n_seq * P.Hkv + entries) * P.pld : P.mass + entries * P.ld;

    for (int b = bx * TB; b < sp.nt; b += P.blocks * TB) {
    // (the lane's number anew for each block, and once more for the sums: what follows from it would be worked out ahead of the loop and kept)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int c = lane & 31, g = lane >> 5;
    // Rows of q as the operand's columns. Wave w brings rows 4 w .. 4 w + 3 of the 32: lane (row lane % 4, chunk 16 j + lane / 4; heads of 64: twice)
    auto qrow_of = [&] { return 4 * wave + (lane & 3); };
    auto qchunk_of = [&] { return (lane >> 2) & (D / 8 - 1); };
    struct rows_raw { u4 x[NJ][2]; float lse; int pos; };
    auto fetch_rows = [&](rows_raw & r, int r0) {
        const int qrow = qrow_of(), qchunk = qchunk_of(), row = min(r0 + qrow, nrows - 1), t = token_of(P, row);
        const size_t i = (size_t) (sv.first + t) * P.Hq + (size_t) hk * P.GQA + (row - t * P.GQA);
        // (as they are in memory: whatever looked at them here would wait for them here)
        const gbytes from = (gbytes) P.q + (i * D + 8 * qchunk) * (P.q_bf16 ? 2 : 4);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (P.q_bf16) r.x[j][0] = gload<u4>(from + 256 * j);
            else {
                r.x[j][0] = gload<u4>(from + 512 * j);
                r.x[j][1] = gload<u4>(from + 512 * j + 16);
            }
        }
        r.lse = P.lse[i];
        r.pos = sv.pos0 + t;
        if (r0 + qrow >= nrows || r.pos < 0 || r.pos >= P.R.n_ctx) r.pos = -1;   // sees nothing
    };
    auto put_rows = [&](const rows_raw & r, int st) {
        const int qrow = qrow_of(), qchunk = qchunk_of();
        float most = 0.f, x[NJ][8];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t half = r.x[j][0][e >> 1];
                x[j][e] = __builtin_bit_cast(float, P.q_bf16 ? (e & 1 ? half & 0xffff0000u : half << 16) : r.x[j][e >> 2][e & 3]);
                most = fmaxf(most, fabsf(x[j][e]));
            }
        most = fmaxf(most, __shfl_xor(most, 4));
        most = fmaxf(most, __shfl_xor(most, 8));
        most = max_swap32(max_swap16(most));
        const int ex = row_exponent(most);
        const float by = ldexpf(P.sign, -ex);
        char * const to = lds + st * C::Q_B + (qrow >> 4) * PL_B;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            h8 y[2];
            halves<2>([&](int e) { return x[j][e]; }, [&](int) { return by; }, y);
            char * const at = to + chunk_at(qrow & 15, 16 * j + qchunk);
            *reinterpret_cast<h8 *>(at) = y[0];
            *reinterpret_cast<h8 *>(at + 2 * PL_B) = y[1];
        }
        if (lane < 4) info[st * QR + qrow] = row_info{ldexpf(P.factor, ex), -r.lse * LOG2E, r.lse == MINUS_INF ? -1 : r.pos};
    };

        // ---- this wave's keys, AT_ONCE groups of 16 at a time through LDS ----
        h8 kr[NU][NPL][NKS];
        int tile[NU];
        size_t from[2 * NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            tile[u] = sp.tile(min(b + wave * NU + u, sp.nt - 1));
#pragma unroll
            for (int x = 0; x < 2; ++x) from[2 * u + x] = head_off + kv_off_tab(P.pg, ptab, seen_or_near<32>(sp, tile[u] * 32, tile[u] * 32 + 16 * x + G::key(lane)));
        }
        char * const to = lds + wave * C::AT_ONCE * G_B;
#pragma unroll
        for (int x0 = 0; x0 < 2 * NU; x0 += C::AT_ONCE) {
#pragma unroll
            for (int x = x0; x < x0 + C::AT_ONCE; ++x) {
                if constexpr (G::DIRECT) G::load((gbytes) P.kc + from[x], to + (x - x0) * G_B, lane);
                else {
                    typename G::raw raw;
                    G::load(raw, (gbytes) P.kc + from[x], lane);
                    G::store(raw, to + (x - x0) * G_B, lane);
                }
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
            const k_frag kf(C::AT_ONCE > 1 ? lane : lane & ~16, G_B);        // (one at a time: row c % 16 of the group that is there)
            if (C::AT_ONCE > 1 || (c >> 4) == x0) {
#pragma unroll
                for (int u = x0 / 2; u < (x0 + C::AT_ONCE + 1) / 2; ++u)
#pragma unroll
                    for (int pl = 0; pl < NPL; ++pl)
#pragma unroll
                        for (int ks = 0; ks < NKS; ++ks) kr[u][pl][ks] = kf.read(to + (2 * u - (C::AT_ONCE > 1 ? x0 : 2 * u)) * G_B + pl * PL_B, ks);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
        }
        float acc[NU][16];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[u][i] = 0.f;
        // rows ahead of the block's first key see none of them; rows whose window begins behind its last one neither, unless there are sinks in it
        const int k_first = sp.tile(b) * 32;
        const int ra = max(k_first - sv.pos0, 0) * P.GQA / QR;
        const long long k_gone = (long long) sp.tile(min(b + TB, sp.nt) - 1) * 32 + 31 + P.R.window - sv.pos0;
        const int rows_end = b < sp.nst || k_gone >= sv.count ? nrows : max((int) k_gone, 0) * P.GQA;
        const int rb = (rows_end + QR - 1) / QR, per = (max(rb - ra, 0) + P.splits - 1) / P.splits;   // this split's share of them
        int r0 = (ra + split * per) * QR;
        const int r1 = min((ra + (split + 1) * per) * QR, rb * QR);
        // Step i reads the rows in place i % 4 and brings those of step i + 2, so that the waves meet after every second step only: one's
        // products run beside another's exponentials (309 -> 285 us for four prompts)
        rows_raw rr;
        if (r0 < r1) fetch_rows(rr, r0);
        __syncthreads();                                      // (the rows go where the keys were)
        if (r0 < r1) put_rows(rr, 0);
        if (r0 + QR < r1) fetch_rows(rr, r0 + QR);
        if (r0 + QR < r1) put_rows(rr, 1);
        __syncthreads();
        for (int st = 0; r0 < r1; r0 += QR, st = (st + 1) & 3) {
            asm volatile("" : "+v"(lane));                    // (anew for each step: registers)
            const int c = lane & 31, g = lane >> 5;
            const k_frag qfr(lane, PL_B);
            const bool more = r0 + 2 * QR < r1;
            if (more) fetch_rows(rr, r0 + 2 * QR);
            const row_info my = info[st * QR + c];
            f16x s[NU];
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
            const char * const rows = lds + st * C::Q_B;
            h8 qn[2] = {qfr.read(rows, 0), qfr.read(rows + 2 * PL_B, 0)};
            bool all[NU];                                     // every row of the 32 sees every key of the tile
#pragma unroll
            for (int u = 0; u < NU; ++u) all[u] = __all(my.pos >= tile[u] * 32 + 31 && tile[u] * 32 > my.pos - P.R.window);
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {                // (the next step's halves of q on their way, no more: registers)
                const h8 q0 = qn[0], q1 = qn[1];
                if (ks + 1 < NKS) {
                    qn[0] = qfr.read(rows, ks + 1);
                    qn[1] = qfr.read(rows + 2 * PL_B, ks + 1);
                }
#pragma unroll
                for (int u = 0; u < NU; ++u) s[u] = mfma32(kr[u][0][ks], q0, s[u]);
#pragma unroll
                for (int u = 0; u < NU; ++u) s[u] = mfma32(kr[u][0][ks], q1, s[u]);
                if constexpr (NPL == 2) {
#pragma unroll
                    for (int u = 0; u < NU; ++u) s[u] = mfma32(kr[u][NPL - 1][ks], q0, s[u]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int k0 = tile[u] * 32;
                if (__builtin_expect(!all[u], 0)) {
                    const int at = k0 + 4 * g;
                    int hi = my.pos - at, lo = max(my.pos - k0, 0) - P.R.window - 4 * g, sk = P.R.n_sink - at;
                    asm volatile("" : "+v"(hi), "+v"(lo), "+v"(sk));   // (or the comparisons would be made ahead of the branch, for every tile)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = mfma_row(i, 0);         // (and 4 g: a number the comparison holds itself)
                        const float w = __builtin_amdgcn_exp2f(fmaf(s[u][i], my.factor, my.lse));
                        acc[u][i] += j <= hi && (j > lo || j < sk) ? w : 0.f;
                        asm volatile("" : "+v"(acc[u][i]));   // (one at a time: conditions take two scalar registers each)
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[u][i] += __builtin_amdgcn_exp2f(fmaf(s[u][i], my.factor, my.lse));
                }
            }
            if (more) put_rows(rr, (st + 2) & 3);
            if (st & 1) __syncthreads();
        }
        // ---- sums over the 32 rows' lanes; lane i of a half adds value i to its key ----
        asm volatile("" : "+v"(lane));
        {
        const int c = lane & 31, g = lane >> 5;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            float mine = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float x = add16(acc[u][i]);
                x += __shfl_xor(x, 16);
                if (c == i) mine = x;
            }
            const int i = b + wave * NU + u, at = mfma_row(c & 15, g), j = tile[u] * 32 + at;
            const bool seen = j <= sp.pmax && (j >= sp.lo || j < sp.ns) && j < P.ld;
            if (c < 16 && i < sp.nt && seen) {
                if (P.splits > 1) mass[i * 32 + at] = mine;   // (i is at most the tile's number)
                else mass[j] += mine;
            }
        }
        }
        __syncthreads();                                      // (the next keys go where the rows were)
    }
}

// the splits' sums, in order, onto the totals of the positions that some row sees
__global__ void __launch_bounds__(256) mass_add_k(const mass_params P) {
    const int x = blockIdx.x * 256 + threadIdx.x, hk = blockIdx.y, seq = blockIdx.z;
    const seq_view sv = seq_of<true>(P.R, seq);
    if (sv.count < 1 || x >= P.pld) return;
    const span sp = span_of<32>(P.R, sv.pos0, sv.pos0 + sv.count - 1);
    const int j = sp.tile(x >> 5) * 32 + (x & 31);
    if (x >> 5 >= sp.nt || j > sp.pmax || !(j >= sp.lo || j < sp.ns) || j >= P.ld) return;
    const size_t entries = (size_t) seq * P.Hkv + hk, step = (size_t) P.R.n_seq * P.Hkv * P.pld;
    const float * const part = P.part + entries * P.pld + x;
    float sum = 0.f;
    for (int k = 0; k < P.splits; ++k) sum += part[k * step];
    P.mass[entries * P.ld + j] += sum;
}

template <class F> int launch_big(F kernel, std::atomic<uint32_t> & attr_set, int lds, const mass_params & P, dim3 grid, hipStream_t s) {
    int dev = 0;
    (void) hipGetDevice(&dev);
    const uint32_t bit = 1u << (dev & 31);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        if (hipFuncSetAttribute((const void *) kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
            (void) hipGetLastError();
            set_error("p1a_attn_mass: cannot reserve %d bytes of LDS", lds);
            return P1A_E_LAUNCH;
        }
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    kernel<<<grid, MTHR, lds, s>>>(P);
    return launched();
}
template <uint32_t KT, int D> int launch_d(const mass_params & P, int few, dim3 grid, hipStream_t s) {
    static std::atomic<uint32_t> attr_set{0};
    if (!few) return launch_big(mass_k<KT, D>, attr_set, mass_cfg<KT, D>::LDS, P, grid, s);
    if (few == 1) mass_step_k<KT, D, 1><<<grid, NTHR, 0, s>>>(P);
    else mass_step_k<KT, D, 2><<<grid, NTHR, 0, s>>>(P);
    return launched();
}
template <uint32_t KT> int launch_kt(const mass_params & P, int D, int few, dim3 grid, hipStream_t s) {
    return D == 256 ? launch_d<KT, 256>(P, few, grid, s) : D == 128 ? launch_d<KT, 128>(P, few, grid, s) : launch_d<KT, 64>(P, few, grid, s);
}

}   // namespace

// How a call is dealt out, from its host numbers and the device. Up to 32 rows of a sequence under a kv head: runs of steps, as many as there are places for
// workgroups (32 sequences of 1000 ... 8190 keys, 24 / 4 heads of 256, q8_0: 36 us; as blocks of keys 88). More: blocks of keys. Their rows are split in
// pieces of four times 32 and more while that leaves compute units without a workgroup, of eight times while there are no more than four workgroups to each,
// of 16 times up to eight workgroups - setting one up costs what three or four times 32 rows do, and the last of unequal ones are waited for:
//   64 tokens over 3001 keys (32 / 8 heads of 128, f16; whole calls) 29 us unsplit, 23 in two; 256 over 3001 53 in two, 35 in four, 39 in eight;
//   256 over 30011 177 in two, 197 in four; four prompts (24 / 4 of 256) 1240 unsplit, 475 in one or two, 335 in three, 270 in seven.
// Partial sums take 256 MB at most: as many splits as fit.
mass_plan plan_mass(const p1a_kv & c, const rows_view & R, int Hq, int max_n, int ld, int cus) {
    const int GQA = Hq / c.Hkv;
    const bool planes = c.type != P1A_KV_F16;
    mass_plan pl{};
    pl.few = (long long) R.max_rows * GQA <= 32 ? (R.max_rows * GQA + 15) / 16 : 0;
    // (a descriptor without positions: as if there were one)
    const long long keys = std::max(1LL, R.window == INT32_MAX ? max_n : std::min<long long>(max_n, (long long) R.window + R.max_rows + R.n_sink + 64));
    const long long places = std::max(cus, 1);
    pl.splits = 1;
    if (pl.few) {
        pl.runs = (int) std::max(1LL, std::min(places * (c.D == 256 ? 2 : 4) / c.Hkv, R.n_seq * ((keys + 127) / 128)));
        return pl;
    }
    const int BK = MW * 32 * (planes && c.D == 256 ? 1 : 2);
    pl.blocks = (int) std::min<long long>((keys + BK - 1) / BK, 65536 / c.Hkv + 1);
    const long long units = (long long) pl.blocks * c.Hkv * R.n_seq, tiles = ((long long) R.max_rows * GQA + QR - 1) / QR;
    pl.splits = (int) std::min(32LL, std::max({1LL, std::min(places / units, tiles / 4), std::min(4 * places / units, tiles / 8), std::min(8 * places / units, tiles / 16)}));
    // (positions of a sequence's tiles: what n_ctx allows, as max_n may be less than what there is)
    pl.pld = (int) std::min<long long>(ld, R.window == INT32_MAX ? R.n_ctx : std::min<long long>(R.n_ctx, (long long) R.window + R.max_rows + R.n_sink) + 96);
    const size_t each = (size_t) R.n_seq * c.Hkv * pl.pld * 4;
    pl.splits = (int) std::max(1LL, std::min<long long>(pl.splits, (256LL << 20) / (long long) std::max<size_t>(each, 1)));
    if (pl.splits > 1) pl.bytes = pl.splits * each;
    return pl;
}

int launch_mass(const p1a_kv & c, const mass_args & a, hipStream_t s) {
    mass_params P;
    P.q = a.q; P.lse = a.lse; P.mass = a.mass; P.kc = (const char *) c.k; P.pg = view_of(c); P.R = a.R;
    P.Hq = a.Hq; P.Hkv = c.Hkv; P.GQA = a.Hq / c.Hkv; P.ld = a.ld; P.q_bf16 = a.q_bf16;
    P.gqa_magic = (uint32_t) (P.GQA == 1 ? (1ull << 32) - 1 : (1ull << 32) / (unsigned) P.GQA);
    P.factor = a.scale == 0.f ? 1.f : (a.scale < 0 ? -a.scale : a.scale) * LOG2E;
    P.sign = a.scale == 0.f ? 0.f : a.scale < 0 ? -1.f : 1.f;
    const mass_plan pl = plan_mass(c, a.R, a.Hq, a.max_n, a.ld, cu_count());
    P.runs = pl.runs; P.blocks = pl.blocks; P.splits = pl.splits; P.pld = pl.pld; P.part = nullptr;
    if (pl.splits > 1) {
        if (a.scratch && !((uintptr_t) a.scratch & 255) && a.scratch_bytes >= pl.bytes) P.part = (float *) a.scratch;
        else {
            float * unused;
            if (!split_scratch(s, kept_bytes(pl.bytes), kept_bytes(1), P.part, unused)) return P1A_E_SCRATCH;
        }
    }
    const dim3 grid = pl.few ? dim3((unsigned) ((pl.runs + 7) / 8 * 8 * c.Hkv)) : dim3((unsigned) (pl.blocks * c.Hkv * pl.splits), a.R.n_seq);
    const int rc = c.type == P1A_KV_F16 ? launch_kt<P1A_KV_F16>(P, c.D, pl.few, grid, s)
                 : c.type == P1A_KV_Q8_0 ? launch_kt<P1A_KV_Q8_0>(P, c.D, pl.few, grid, s) : launch_kt<P1A_KV_Q4_0>(P, c.D, pl.few, grid, s);
    if (rc != P1A_OK || pl.splits == 1) return rc;
    mass_add_k<<<dim3((pl.pld + 255) / 256, c.Hkv, a.R.n_seq), 256, 0, s>>>(P);
    return launched();
}

}   // namespace p1a
