// Attention weight per cache position (gfx950): mass[s][h][j] += sum over a call's rows t and the heads i of kv head h of exp(scale q_ti . k_j - lse_ti).
//
// Work: a wave owns 32 NU keys of one sequence and kv head - their rows stay in its registers as matrix operands - and walks the rows of q that may see
// them, 32 at a time; a key's sum stays with one lane until the end, so no two waves add to the same entry and no atomic orders the sums. The
// workgroup's four waves (128 NU keys) share the rows: fetched, brought to two f16 halves and put into LDS once for all.
// Arithmetic: S^T = K Q^T on v_mfma_f32_32x32x16_f16 with q in two halves and quantized keys in two planes (p1a_tiles.hpp): 2 products for f16 caches,
// 3 for quantized ones; weights and sums in fp32.
// What bounds it: few rows - reading K once; many - the matrix pipe, 16 vector instructions a product for the weights beside it.
#include "p1a_tiles.hpp"

#include <algorithm>
#include <atomic>

namespace p1a {
namespace {

constexpr int NTHR = 256, QR = 32;                            // rows of q at a time

struct mass_params {
    const void * q;
    const float * lse;
    float * mass;
    const char * kc;
    kv_view pg;
    rows_view R;
    int Hq, Hkv, GQA, ld, q_bf16;
    uint32_t gqa_magic;
    float factor, sign;
};

template <uint32_t KT, int D, int NU> struct mass_cfg {
    static constexpr int NPL = group_planes(KT, true), G_B = NPL * plane_bytes(D);
    static constexpr int K_B = 4 * 2 * G_B;                   // 32 keys of every wave
    static constexpr int Q_B = 2 * 2 * plane_bytes(D);        // 32 rows in two halves
    static constexpr int LDS = std::max(K_B, 2 * Q_B) + 2 * QR * 12;   // (the rows go where the keys were)
};

template <uint32_t KT, int D, int NU>
__global__ void __launch_bounds__(NTHR, D <= 128 ? 2 : 1) mass_k(const mass_params P) {
    using C = mass_cfg<KT, D, NU>;
    using G = group<KT, D, C::NPL>;
    constexpr int NPL = C::NPL, G_B = C::G_B, PL_B = plane_bytes(D), NKS = D / 16, NJ = D / 64, BK = 128 * NU;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    struct row_info { float factor, lse; int pos; };
    row_info * const info = reinterpret_cast<row_info *>(lds + std::max(C::K_B, 2 * C::Q_B));   // [2][QR]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, g = lane >> 5;
    const int hk = blockIdx.x % P.Hkv, bx = blockIdx.x / P.Hkv, seq = blockIdx.y;
    const seq_view sv = seq_of<true>(P.R, seq);
    if (sv.count < 1) return;
    const span sp = span_of<32>(P.R, sv.pos0, sv.pos0 + sv.count - 1);   // tiles of 32 keys: a wave's NU are consecutive ones of the list
    const int32_t * const ptab = P.pg.pt ? P.pg.pt + (P.pg.rtab ? sload_i32(P.pg.rtab + seq) : 0) : nullptr;
    const size_t head_off = (size_t) hk * head_bytes(KT, D);
    const int nrows = sv.count * P.GQA;
    auto tok_of = [&](int r) {
        const int t = (int) __umulhi((uint32_t) r, P.gqa_magic);
        return r - t * P.GQA >= P.GQA ? t + 1 : t;
    };
    const k_frag kf(lane, G_B), qfr(lane, PL_B);
    float * const mass = P.mass + ((size_t) seq * P.Hkv + hk) * P.ld;

    // Rows of q as the operand's columns. Wave w brings rows 8 w .. 8 w + 7 of the 32: lane (row lane % 8, chunk 8 j + lane / 8)
    const int qrow = 8 * wave + (lane & 7);
    struct rows_raw { f4 x[NJ][2]; float lse; int pos; };
    auto fetch_rows = [&](rows_raw & r, int r0) {
        const int row = min(r0 + qrow, nrows - 1), t = tok_of(row);
        const size_t i = (size_t) (sv.first + t) * P.Hq + (size_t) hk * P.GQA + (row - t * P.GQA);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) r.x[j][e] = q4_at(P.q, P.q_bf16, i * D + (8 * j + (lane >> 3)) * 8 + 4 * e);
        r.lse = P.lse[i];
        r.pos = sv.pos0 + t;
        if (r0 + qrow >= nrows || r.pos < 0 || r.pos >= P.R.n_ctx || r.lse == MINUS_INF) r.pos = -1;   // sees nothing
    };
    auto put_rows = [&](const rows_raw & r, int st) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(r.x[j][e >> 2][e & 3]));
        most = fmaxf(most, __shfl_xor(most, 8));
        most = max_swap32(max_swap16(most));
        const int ex = row_exponent(most);
        const float by = ldexpf(P.sign, -ex);
        char * const to = lds + st * C::Q_B + (qrow >> 4) * PL_B;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            h8 y[2];
            halves<2>([&](int e) { return r.x[j][e >> 2][e & 3]; }, [&](int) { return by; }, y);
            char * const at = to + chunk_at(qrow & 15, 8 * j + (lane >> 3));
            *reinterpret_cast<h8 *>(at) = y[0];
            *reinterpret_cast<h8 *>(at + 2 * PL_B) = y[1];
        }
        if (lane < 8) info[st * QR + qrow] = row_info{ldexpf(P.factor, ex), -r.lse * LOG2E, r.pos};
    };

    for (int b = bx * 4 * NU; b < sp.nt; b += gridDim.x / P.Hkv * 4 * NU) {
        // ---- this wave's keys ----
        h8 kr[NU][NPL][NKS];
        int tile[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            tile[u] = sp.tile(min(b + wave * NU + u, sp.nt - 1));
            char * const to = lds + wave * 2 * G_B;
            typename std::conditional<G::DIRECT, int, typename group<KT == P1A_KV_F16 ? P1A_KV_Q8_0 : KT, D, NPL>::raw>::type raw[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int j = seen_or_near<32>(sp, tile[u] * 32, tile[u] * 32 + 16 * x + G::key(lane));
                const size_t row = head_off + kv_off_tab(P.pg, ptab, j);
                if constexpr (G::DIRECT) G::load((gbytes) P.kc + row, to + x * G_B, lane);
                else G::load(raw[x], (gbytes) P.kc + row, lane);
            }
            if constexpr (!G::DIRECT) {
#pragma unroll
                for (int x = 0; x < 2; ++x) G::store(raw[x], to + x * G_B, lane);
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int pl = 0; pl < NPL; ++pl)
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) kr[u][pl][ks] = kf.read(to + pl * PL_B, ks);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
        }
        float acc[NU][16];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[u][i] = 0.f;
        // rows ahead of the block's first key see none of them
        const int k_first = sp.tile(b) * 32;
        int r0 = max(k_first - sv.pos0, 0) * P.GQA / QR * QR;
        // rows whose window begins behind its last one neither, unless there are sinks in it
        const long long k_gone = (long long) sp.tile(min(b + 4 * NU, sp.nt) - 1) * 32 + 31 + P.R.window - sv.pos0;
        const int r1 = b < sp.nst || k_gone >= sv.count ? nrows : max((int) k_gone, 0) * P.GQA;
        rows_raw rr;
        if (r0 < r1) fetch_rows(rr, r0);
        __syncthreads();                                      // (the rows go where the keys were)
        if (r0 < r1) put_rows(rr, 0);
        __syncthreads();
        for (int st = 0; r0 < r1; r0 += QR, st ^= 1) {
            const bool more = r0 + QR < r1;
            if (more) fetch_rows(rr, r0 + QR);
            const row_info my = info[st * QR + c];
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int k0 = tile[u] * 32;
                f16x s;
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
                for (int ks = 0; ks < NKS; ++ks) {
                    const h8 q0 = qfr.read(lds + st * C::Q_B, ks), q1 = qfr.read(lds + st * C::Q_B + 2 * PL_B, ks);
                    s = mfma32(kr[u][0][ks], q0, s);
                    s = mfma32(kr[u][0][ks], q1, s);
                    if constexpr (NPL == 2) s = mfma32(kr[u][NPL - 1][ks], q0, s);
                }
                if (!__all(my.pos >= k0 + 31 && k0 > my.pos - P.R.window)) {   // (else every row of the 32 sees every key of the tile)
                    const int hi = my.pos - k0, lo = max(hi, 0) - P.R.window, sk = P.R.n_sink - k0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int j = mfma_row(i, g);
                        if (j <= hi && (j > lo || j < sk)) acc[u][i] += __builtin_amdgcn_exp2f(fmaf(s[i], my.factor, my.lse));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[u][i] += __builtin_amdgcn_exp2f(fmaf(s[i], my.factor, my.lse));
                }
            }
            if (more) put_rows(rr, st ^ 1);
            __syncthreads();
        }
        // ---- sums over the 32 rows' lanes; lane i of a half adds value i to its key ----
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            float mine = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float x = acc[u][i];
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) x += __shfl_xor(x, d);
                if (c == i) mine = x;
            }
            const int j = tile[u] * 32 + mfma_row(c & 15, g);
            const bool seen = j <= sp.pmax && (j >= sp.lo || j < sp.ns) && j < P.ld;
            if (c < 16 && b + wave * NU + u < sp.nt && seen) mass[j] += mine;
        }
        __syncthreads();                                      // (the next keys go where the rows were)
    }
}

template <uint32_t KT, int D, int NU> int launch_cfg(const mass_params & P, dim3 grid, hipStream_t s) {
    constexpr int lds = mass_cfg<KT, D, NU>::LDS;
    static std::atomic<uint32_t> attr_set{0};
    int dev = 0;
    (void) hipGetDevice(&dev);
    const uint32_t bit = 1u << (dev & 31);
    if (!(attr_set.load(std::memory_order_acquire) & bit)) {
        if (hipFuncSetAttribute((const void *) mass_k<KT, D, NU>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
            (void) hipGetLastError();
            set_error("p1a_attn_mass: cannot reserve %d bytes of LDS", lds);
            return P1A_E_LAUNCH;
        }
        attr_set.fetch_or(bit, std::memory_order_release);
    }
    mass_k<KT, D, NU><<<grid, NTHR, lds, s>>>(P);
    return launched();
}
template <uint32_t KT> int launch_kt(const mass_params & P, int D, dim3 grid, hipStream_t s) {
    return D == 256 ? launch_cfg<KT, 256, 1>(P, grid, s) : D == 128 ? launch_cfg<KT, 128, 1>(P, grid, s) : launch_cfg<KT, 64, 1>(P, grid, s);
}

}   // namespace

int launch_mass(const p1a_kv & c, const void * q, bool q_bf16, const float * lse, float * mass, int ld, const rows_view & R, int Hq, float scale, int max_n, hipStream_t s) {
    mass_params P;
    P.q = q; P.lse = lse; P.mass = mass; P.kc = (const char *) c.k; P.pg = view_of(c); P.R = R;
    P.Hq = Hq; P.Hkv = c.Hkv; P.GQA = Hq / c.Hkv; P.ld = ld; P.q_bf16 = q_bf16;
    P.gqa_magic = (uint32_t) (P.GQA == 1 ? (1ull << 32) - 1 : (1ull << 32) / (unsigned) P.GQA);
    P.factor = scale == 0.f ? 1.f : (scale < 0 ? -scale : scale) * LOG2E;
    P.sign = scale == 0.f ? 0.f : scale < 0 ? -1.f : 1.f;
    // a workgroup for every 128 keys that a sequence may have seen (one that understates them: each takes several)
    const long long keys = R.window == INT32_MAX ? max_n : std::min<long long>(max_n, (long long) R.window + R.max_rows + R.n_sink + 64);
    const unsigned nb = (unsigned) std::min<long long>((keys + 127) / 128, 65536 / c.Hkv + 1);
    const dim3 grid(nb * c.Hkv, R.n_seq);
    return c.type == P1A_KV_F16 ? launch_kt<P1A_KV_F16>(P, c.D, grid, s) : c.type == P1A_KV_Q8_0 ? launch_kt<P1A_KV_Q8_0>(P, c.D, grid, s) : launch_kt<P1A_KV_Q4_0>(P, c.D, grid, s);
}

}   // namespace p1a
