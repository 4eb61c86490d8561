// Attention of few rows a sequence - single tokens, drafts to verify - over bounded caches: p1a_attn_chunk where a sequence's rows under a kv head are at
// most 32, and so one or two tiles of 16 columns.
//
// Work: steps of 128 keys, counted through over the sequences of a kv head; a workgroup of four waves takes a run of them, as long as every other
// workgroup's - a sequence's end, the next one and its beginning, if need be. (Equal shares of every sequence: 32 sequences of 300 ... 32768 keys through a window
// of 4096 left a third of the device idle at the end.) Within a sequence each wave walks tiles of 32 keys of its own, 4 apart; nothing is
// shared and nothing waited for until the waves' results are folded. A sequence that lies in one run is finished there, the others' partials are
// merged by chunk_merge_k. (p1a_chunk.hip's blocks, whose waves share tiles and split rows, would leave three waves of four idle here.)
// Arithmetic: S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16. K is read straight into the operand; codes of quantized caches stay whole numbers,
// exact in f16. K's scales multiply the fp32 result of a block; V's multiply P (fp32) ahead of the product, P d being what is cut into f16 halves. q and
// P (P d) are two halves where results are f32, one where they are bf16 (EXACT). d enters as d / 2^E with E the largest exponent of a scale so far
// - O is counted in 2^E - so that halves of P d do not end where f16 does.
// V goes through LDS (16 keys of a dim lie in 16 rows): f16 straight there, two tiles a wave, codes through registers. While a tile's weights
// and results are worked out the next one is on its way; its page-table entries were asked for ahead of the scores.
// What bounds it: reading K and V (f16: 32 tokens of sequences of 300 ... 32768 keys through a window of 4096, 24 / 4 heads of 256, 78 us a call, 67 at the rate of a copy),
// and over quantized caches the vector instructions that unpack codes and cut P d into halves anew for every 32 dims: the same over q8_0 52 us and 5.4 of
// merging, 35 at the rate of a copy; bf16 results, one half, 11 % less.
#include "p1a_tiles.hpp"

#include <atomic>

namespace p1a {
namespace {

constexpr int NW = 4, NTHR = NW * 64, PC = 8;                 // waves; columns folded at a time

template <uint32_t KT, int D, int NT, bool EXACT> struct step_cfg {
    static constexpr bool F16 = KT == P1A_KV_F16;
    static constexpr int VT_B = 2 * plane_bytes(D);           // 32 keys of V
    static constexpr int V_B = (F16 ? 2 : 1) * VT_B;
    static constexpr int TAB = keys16<KT, D>::TAB;
    static constexpr int WAVE_B = V_B + 4 * TAB * 4;          // and the scales of 2 x 16 keys of K and V
    // (the low halves of q, where registers do not hold them: the same for every wave, each writes all of them)
    static constexpr bool QL = EXACT && NT * D >= (F16 ? 512 : 256);
    static constexpr int ML_B = NW * 2 * 16 * NT * 4, LDS = NW * WAVE_B + (QL ? NT * D * 32 : 0) + (4 * TAB * 4 >= ML_B ? 0 : ML_B);
    static constexpr int ML_AT = 4 * TAB * 4 >= ML_B ? V_B : LDS - ML_B;      // (the first wave's scales are done with by then)
    static_assert(PC * (D + 4) * 4 <= V_B, "folded columns fit where V was");
};

template <uint32_t KT, int D, int NT, bool EXACT>
__global__ void __launch_bounds__(NTHR, D == 256 && (KT == P1A_KV_F16 || NT == 2) ? 1 : 2) step_k(const chunk_params P) {
    using C = step_cfg<KT, D, NT, EXACT>;
    using K = keys16<KT, D>;
    using G = group<KT, D, C::F16 ? 1 : 0>;
    constexpr bool F16 = C::F16;
    constexpr int NB = D / 32, NDT = D / 16, NQ = EXACT ? 2 : 1, PL_B = plane_bytes(D);
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // the kv heads of a run of steps, whose rows have cache lines in common, on one XCD
    const int xcd = blockIdx.x & 7, jx = blockIdx.x >> 3, hk = jx % P.Hkv, run = jx / P.Hkv * 8 + xcd;
    if (run >= P.runs) return;
    auto tok_of = [&](int r) {
        const int t = (int) __umulhi((uint32_t) r, P.gqa_magic);
        return r - t * P.GQA >= P.GQA ? t + 1 : t;
    };
    step_runs<NW> steps;
    steps.first = 0;
    steps.end = 1;
    steps.per = 1 << 30;
    if (P.nks > 1 && !steps.begin(P.R, P.pg, run, P.runs, P.nks)) return;
    char * const mine = lds + wave * C::WAVE_B;
    float * const tk = reinterpret_cast<float *>(mine + C::V_B), * const tv = tk + 2 * C::TAB;
    const size_t head_off = (size_t) hk * head_bytes(KT, D);

  for (int at_step = steps.first; at_step < steps.end;) {
    // (the lane's number anew for each sequence, and once more for the fold: what follows from it would be worked out ahead of the loop and kept, 40 registers)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, c = lane & 15, g = lane >> 4;
    // whose step that is, and the sequence's runs, which of them this is
    typename step_runs<NW>::found f;
    if (P.nks > 1) {
        if (!steps.find(P.R, P.pg, at_step, lane, f)) return;
    } else {                                                    // a sequence each
        f.seq = run; f.first = 0; f.steps = 1 << 24;
        f.v = seq_of<true>(P.R, run);
        f.table = P.pg.pt && P.pg.rtab ? sload_i32(P.pg.rtab + run) : 0;
        if (f.v.count < 1) return;
    }
    const seq_view & sv = f.v;
    const int run0 = f.first / steps.per, pieces = P.nks > 1 ? (f.first + f.steps - 1) / steps.per - run0 + 1 : 1, piece = P.nks > 1 ? run - run0 : 0;
    const int R = min(sv.count * P.GQA, 16 * NT);
    auto row_index = [&](int r) { const int t = tok_of(r); return (size_t) (sv.first + t) * P.Hq + (size_t) hk * P.GQA + (r - t * P.GQA); };
    const span sp = step_runs<NW>::span_of_rows(P.R, sv);
    const int ta = (at_step - f.first) * NW, tb = P.nks > 1 ? min((min(steps.end, f.first + f.steps) - f.first) * NW, sp.nt) : sp.nt;
    at_step = f.first + f.steps;
    // positions that all rows see
    const bool odd = sv.pos0 < 0 || sv.pos0 + sv.count > P.R.n_ctx;
    const int all_hi = odd ? -1 : sv.pos0, all_lo = P.R.window == INT32_MAX ? 0 : sp.pmax - P.R.window + 1;

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
    typename K::raw kr[2];
    typename K::scales vs[2];
    struct none {};
    typename std::conditional<F16, none, typename group<F16 ? P1A_KV_Q8_0 : KT, D, 0>::raw>::type vr[2];
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
                K::load_scales(vs[x], (gbytes) P.vc + w.off[x], g);
            }
        }
    };

    int i = ta + wave;
    where at;
    if (i < tb) {
        at = keys.at(sp.tile(i), keys.pages_of(sp.tile(i)));
        if constexpr (F16) ask_v(at, 0);
        if constexpr (F16 || NT * D <= 128) ask_k(at);
    }

    // ---- Q^T: columns 16 n + c ----
    constexpr int NQR = C::QL ? 1 : NQ;                       // halves in registers
    h8 qf[NT][NQR][NB];
    char * const ql = lds + NW * C::WAVE_B + lane * 16;
    auto q_at = [&](int n, int k, int b) { return k < NQR ? qf[n][k < NQR ? k : 0][b] : *reinterpret_cast<const h8 *>(ql + (n * NB + b) * 1024); };
    float factor[NT];
    int pos[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = 16 * n + c, rr = min(r, R - 1);
        h8 qq[NQ][NB];
        factor[n] = ldexpf(P.factor, q_columns<KT, D, NQ>(P.q, P.q_bf16, row_index(rr), P.sign, g, qq));
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int k = 0; k < NQR; ++k) qf[n][k][b] = qq[k][b];
            if constexpr (C::QL) *reinterpret_cast<h8 *>(ql + (n * NB + b) * 1024) = qq[NQ - 1][b];
        }
        pos[n] = sv.pos0 + tok_of(rr);
        if (pos[n] < 0 || pos[n] >= P.R.n_ctx) pos[n] = -1;   // sees nothing
        __builtin_amdgcn_sched_barrier(0);
    }

    if (i < tb) {                                             // (what registers hold not ahead of Q)
        if constexpr (!F16) ask_v(at, 0);
        if constexpr (!F16 && NT * D > 128) ask_k(at);
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
    for (int st = 0; i < tb; i += NW, st ^= 1) {
        const int k0 = sp.tile(i) * 32;
        const bool more = i + NW < tb;
        key_rows::pages pg;
        if (more) pg = keys.pages_of(sp.tile(i + NW));
        // ---- V's codes and the scales into LDS ----
        if constexpr (!F16) {
            float dm = 0.f;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < K::NSC; ++y) dm = fmaxf(dm, fabsf(K::scale(vs[x], y)));
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
                K::put(tk + x * C::TAB, kr[x].d, c, g);
                K::put(tv + x * C::TAB, vs[x], c, g, -E);
                G::store(vr[x], mine + x * PL_B, lane);
            }
            __builtin_amdgcn_wave_barrier();
        }
        // ---- S^T ----
        f4 s[2][NT];
        K::template scores<NT, NQ>(kr, q_at, tk, g, s);
        // (V of this tile was asked for ahead of its K)
        if constexpr (F16) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (more) {
            const where at = keys.at(sp.tile(i + NW), pg);
            ask_v(at, st ^ 1);
            ask_k(at);
        }
        // ---- softmax ----
        if (!(k0 + 31 <= all_hi && k0 >= all_lo)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int from = k0 + 4 * g;
                int hi = pos[n] - from, lo = max(pos[n] - k0, 0) - P.R.window - 4 * g, sk = P.R.n_sink - from;
                asm volatile("" : "+v"(hi), "+v"(lo), "+v"(sk));   // (or the comparisons would be made ahead of the branch, for every tile)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 16 * x + e;                // (and 4 g)
                        s[x][n][e] = j <= hi && (j > lo || j < sk) ? s[x][n][e] : MINUS_INF;
                    }
            }
        }
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
        // ---- O^T += V^T (P d) ----
        const char * const vt = mine + (F16 ? st * C::VT_B : 0);
        // (a block's scales and rows of V^T are asked for a block ahead)
        struct block { f4 d[2]; h4 a[2][2]; };
        auto read = [&](int b) {
            block r;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (!F16) r.d[x] = *reinterpret_cast<const f4 *>(tv + x * C::TAB + b * 16 + 4 * g);
#pragma unroll
                for (int y = 0; y < 2; ++y) r.a[y][x] = v_read(vt + x * PL_B, 2 * b + y);
            }
            return r;
        };
        h8 pb[NT][NQ];
        block next = read(0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const block now = next;
            if (b + 1 < NB) next = read(b + 1);
            if (!F16 || b == 0) {
#pragma unroll
                for (int n = 0; n < NT; ++n) halves<NQ>([&](int e) { return p[n][e]; }, [&](int e) { return F16 ? 1.f : now.d[e >> 2][e & 3]; }, pb[n]);
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

    // ---- fold the waves, in wave order ----
    {
    asm volatile("" : "+v"(tid));
    const int c = tid & 15, g = (tid >> 4) & 3;
    auto ml = [&](int w, int which, int col) -> float & { return reinterpret_cast<float *>(lds + C::ML_AT)[(w * 2 + which) * 16 * NT + col]; };
    if constexpr (C::ML_AT < C::WAVE_B) __syncthreads();      // (until the first wave has done with them)
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
            const int h0 = 16 * n + half, he = min(h0 + PC, R);
            if (h0 >= R) break;
            if (h0) __syncthreads();
            if (c >= half && c < half + PC) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) {
                    f4 v = o[n][dt];
                    if constexpr (!F16) {
#pragma unroll
                        for (int y = 0; y < 4; ++y) v[y] = ldexpf(v[y], E);
                    }
                    *reinterpret_cast<f4 *>(parked + (c - half) * OS + 16 * dt + 4 * g) = v;
                }
            }
            __syncthreads();
            for (int t = tid; t < (he - h0) * D4; t += NTHR) {
                const int cc = t / D4, d = 4 * (t - cc * D4), col = h0 + cc;
                float m[NW], M = MINUS_INF, lt = 0.f;
                f4 a[NW], acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    a[w] = *reinterpret_cast<const f4 *>(reinterpret_cast<const float *>(lds + w * C::WAVE_B) + cc * OS + d);
                    m[w] = ml(w, 0, col);
                    M = fmaxf(M, m[w]);
                }
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float f = m[w] == MINUS_INF ? 0.f : __builtin_amdgcn_exp2f(m[w] - M);
                    lt += ml(w, 1, col) * f;
                    acc += a[w] * f;
                }
                const size_t row = row_index(col);
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
                const int at = sv.pos0 + tok_of(col);
                f4 v = acc * (at < 0 || at >= P.R.n_ctx ? 0.f : 1.0f / lt);
                if (P.gate) {
                    const f4 gt = *reinterpret_cast<const f4 *>(P.gate + row * D + d);
#pragma unroll
                    for (int y = 0; y < 4; ++y) v[y] *= gate_of(gt[y]);
                }
                put4(P.out, P.out_bf16, row * D + d, v);
            }
        }
    }
    if (P.nks > 1 && piece == 0 && hk == 0 && tid == 0) P.part_n[f.seq] = pieces;
    __syncthreads();                                          // (what was folded is read; the next sequence's V goes there)
  }
}

template <uint32_t KT, int D, int NT, bool EXACT> int launch_cfg(const chunk_params & P, unsigned grid, hipStream_t s) {
    constexpr int lds = step_cfg<KT, D, NT, EXACT>::LDS;
    static std::atomic<uint32_t> attr_set{0};
    int dev = 0;
    (void) hipGetDevice(&dev);
    const uint32_t bit = 1u << (dev & 31);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        if (hipFuncSetAttribute((const void *) step_k<KT, D, NT, EXACT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
            (void) hipGetLastError();
            set_error("p1a_attn_chunk: cannot reserve %d bytes of LDS", lds);
            return P1A_E_LAUNCH;
        }
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    step_k<KT, D, NT, EXACT><<<grid, NTHR, lds, s>>>(P);
    return launched();
}
template <uint32_t KT, int D> int launch_d(const chunk_params & P, int NT, bool exact, unsigned grid, hipStream_t s) {
    if (NT == 1) return exact ? launch_cfg<KT, D, 1, true>(P, grid, s) : launch_cfg<KT, D, 1, false>(P, grid, s);
    return exact ? launch_cfg<KT, D, 2, true>(P, grid, s) : launch_cfg<KT, D, 2, false>(P, grid, s);
}
template <uint32_t KT> int launch_kt(const chunk_params & P, int D, int NT, bool exact, unsigned grid, hipStream_t s) {
    return D == 256 ? launch_d<KT, 256>(P, NT, exact, grid, s) : D == 128 ? launch_d<KT, 128>(P, NT, exact, grid, s) : launch_d<KT, 64>(P, NT, exact, grid, s);
}

}   // namespace

int launch_step(const p1a_kv & c, const chunk_params & P, int NT, bool exact, hipStream_t s) {
    const long long grid = (P.runs + 7LL) / 8 * 8 * c.Hkv;
    if (grid > 0x7fffffffLL) { set_error("p1a_attn_chunk: too many rows for one call"); return P1A_E_SHAPE; }
    return c.type == P1A_KV_F16 ? launch_kt<P1A_KV_F16>(P, c.D, NT, exact, (unsigned) grid, s)
         : c.type == P1A_KV_Q8_0 ? launch_kt<P1A_KV_Q8_0>(P, c.D, NT, exact, (unsigned) grid, s) : launch_kt<P1A_KV_Q4_0>(P, c.D, NT, exact, (unsigned) grid, s);
}

}   // namespace p1a
