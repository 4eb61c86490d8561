// What the kernels over bounded caches share (internal header): whose a call's rows are and what they see, and tiles of 16 keys in LDS.
#pragma once
#include "p1a_common.hpp"

#include <type_traits>
#include <utility>

namespace p1a {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float MINUS_INF = -__builtin_inff();

// f(0), f(1) ... f(N - 1), each with its number as a constant
template <int... I, typename F> __device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F && f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F> __device__ __forceinline__ void each(F && f) { each_of(std::make_integer_sequence<int, N>{}, f); }

// ---- rows of several sequences (p1a_rows as the kernels take it) ----
struct rows_view {
    const int32_t * row0, * pos0;
    int T, n_seq, max_rows, per, p0;   // per: rows of a sequence without row0
    int window, n_sink;                // window: INT32_MAX for none (n_sink 0 then)
    int n_ctx;
};
struct seq_view { int first, count, pos0; };   // rows first .. first + count - 1, the first of them at position pos0
// (whatever the device arrays hold: rows inside 0 .. T, positions where adding a row to one does not overflow)
// (UNIFORM: every lane asks for the same sequence - scalar loads, and what follows from them stays in scalar registers)
template <bool UNIFORM = false> __device__ __forceinline__ seq_view seq_of(const rows_view & R, int s) {
    auto at = [](const int32_t * p) { return UNIFORM ? sload_i32(p) : *p; };
    seq_view v;
    v.first = R.row0 ? min(max(at(R.row0 + s), 0), R.T) : s * R.per;
    v.count = min(R.row0 ? max(min(at(R.row0 + s + 1), R.T) - v.first, 0) : R.per, R.max_rows);
    v.pos0 = min(max(R.pos0 ? at(R.pos0 + s) : R.p0, -(1 << 30)), R.n_ctx);
    return v;
}
// sums over the lanes up to this one
__device__ __forceinline__ int lanes_up_to(int u) {
    u += __builtin_amdgcn_update_dpp(0, u, 0x111, 0xf, 0xf, true);
    u += __builtin_amdgcn_update_dpp(0, u, 0x112, 0xf, 0xf, true);
    u += __builtin_amdgcn_update_dpp(0, u, 0x114, 0xf, 0xf, true);
    u += __builtin_amdgcn_update_dpp(0, u, 0x118, 0xf, 0xf, true);
    u += __builtin_amdgcn_update_dpp(0, u, 0x142, 0xa, 0xf, false);
    u += __builtin_amdgcn_update_dpp(0, u, 0x143, 0xc, 0xf, false);
    return u;
}
// Item b of a list that holds ceil(count * mul / unit) items of each sequence, in order: whose it is, and which of them; false: there are fewer.
// Every lane of the wave calls, with the same b.
struct item_at { int seq, index, of; seq_view v; };
__device__ __forceinline__ bool find_item(const rows_view & R, int b, int mul, int unit, int lane, item_at & at) {
    if (!R.row0) {
        at.of = (R.max_rows * mul + unit - 1) / unit;          // (max_rows is at most per)
        at.seq = b / at.of;
        at.index = b - at.seq * at.of;
        if (at.seq >= R.n_seq) return false;
        at.v = seq_of<true>(R, at.seq);
        return true;
    }
    for (int s0 = 0; s0 < R.n_seq; s0 += 64) {
        const int s = s0 + lane;
        const int n = s < R.n_seq ? (int) (((long long) seq_of(R, s).count * mul + unit - 1) / unit) : 0;
        const int u = lanes_up_to(n);
        const unsigned long long behind = __ballot(u > b);
        if (behind) {
            const int l = __builtin_ctzll(behind);
            at.seq = s0 + l;
            at.of = __builtin_amdgcn_readlane(n, l);
            at.index = b - (__builtin_amdgcn_readlane(u, l) - at.of);
            at.v = seq_of<true>(R, at.seq);
            return true;
        }
        b -= __builtin_amdgcn_readlane(u, 63);
    }
    return false;
}

// The positions that rows at pmin .. pmax of one sequence see, in tiles of BN: the sinks' tiles, then the window's
struct span {
    int pmax, lo, ns;                  // visible: lo .. pmax and 0 .. ns - 1
    int nst, tw0, nt;                  // tiles of sinks, first tile of the window, all tiles (0: nothing is seen)
    __device__ __forceinline__ int tile(int i) const { return i < nst ? i : tw0 + (i - nst); }
};
template <int BN> __device__ __forceinline__ span span_of(const rows_view & R, int pmin, int pmax) {
    span s;
    pmin = max(pmin, 0);
    s.pmax = min(pmax, R.n_ctx - 1);
    s.lo = R.window == INT32_MAX ? 0 : max(pmin - R.window + 1, 0);
    s.ns = max(min(R.n_sink, s.pmax + 1), 0);
    s.nst = (s.ns + BN - 1) / BN;
    s.tw0 = max(s.lo / BN, s.nst);
    s.nt = pmin > s.pmax ? 0 : s.nst + max(s.pmax / BN - s.tw0 + 1, 0);
    return s;
}
// Position j of the tile that starts at k0 or, where nothing sees j, one of the tile that is seen: its row is fetched in its place, so that no
// page-table entry and no memory behind one is read that the call may not know
template <int BN> __device__ __forceinline__ int seen_or_near(const span & s, int k0, int j) {
    if (j > s.pmax) return s.pmax;
    if (j < s.lo && j >= s.ns) return k0 + BN > s.lo ? s.lo : s.ns - 1;
    return j;
}

// ---- rows of q as operands: two halves whose sum is the f32 value ----
// A row is brought below 1 by a power of two first (its inverse goes into the factor of the scores), so that the low halves do not end where f16 does.
// (Not above 2^100: the factor stays a number above zero.)
__device__ __forceinline__ int row_exponent(float most) { return most > 0.f && most < __builtin_inff() ? max(__builtin_amdgcn_frexp_expf(most), -100) : 0; }

// x(0 .. 7) * y(0 .. 7) in f16 halves: the rounded products, and (NQ = 2) what the rounding left, rounded itself
typedef float f2w __attribute__((ext_vector_type(2)));
template <int NQ, class X, class Y> __device__ __forceinline__ void halves(X && x, Y && y, h8 (&out)[NQ]) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x0 = x(2 * e), y0 = y(2 * e), x1 = x(2 * e + 1), y1 = y(2 * e + 1);
        h2 h = __builtin_convertvector(f2w{x0 * y0, x1 * y1}, h2);
        asm("" : "+v"(h));                                    // (one conversion of both, not one more of each for the rest)
        hi[e] = __builtin_bit_cast(uint32_t, h);
        if constexpr (NQ == 2) lo[e] = __builtin_bit_cast(uint32_t, h2{(half_t) fmaf(x0, y0, -(float) h[0]), (half_t) fmaf(x1, y1, -(float) h[1])});
    }
    out[0] = __builtin_bit_cast(h8, u4{hi[0], hi[1], hi[2], hi[3]});
    if constexpr (NQ == 2) out[NQ - 1] = __builtin_bit_cast(h8, u4{lo[0], lo[1], lo[2], lo[3]});
}

// ---- tiles of 16 keys in LDS ----
// A group is 16 keys of one kv head as f16, in one plane or - where a quantized value has to keep all its 18 bits - two, whose sum it is. A plane
// is cut into blocks of 1 KB, four 16-byte chunks (32 dims) of the 16 keys: chunk x of key k lies in block x / 4 at (x % 4) * 256 + (k ^ 4 (x % 4)) * 16. A
// block is what one global_load_lds_dwordx4 moves (64 lanes x 16 bytes to consecutive LDS), 64 bytes of each of 16 rows; a lane's key is the same in every
// block, so it needs one page-table entry and one address a tile, whatever the pages' length. The operand of S^T = K Q^T reads 16 keys of a chunk, 256 bytes
// on end; the transposing read of V^T takes 4 keys of the four chunks of a block, which the exclusive or puts side by side in the banks.
typedef const __attribute__((address_space(1))) char * gbytes;
template <typename T> __device__ __forceinline__ T gload(gbytes p) { return *(const __attribute__((address_space(1))) T *) p; }
typedef u4 u4_a4 __attribute__((aligned(4)));
typedef u4 u4_a2 __attribute__((aligned(2)));
typedef unsigned u2w __attribute__((ext_vector_type(2)));
typedef u2w u2_a4 __attribute__((aligned(4)));

constexpr int group_planes(uint32_t kt, bool exact) { return exact && kt != P1A_KV_F16 ? 2 : 1; }
constexpr int plane_bytes(int D) { return 16 * 2 * D; }

__device__ __forceinline__ uint32_t lds_at(const char * p) { return (uint32_t) (size_t) (const __attribute__((address_space(3))) char *) p; }
__device__ __forceinline__ int chunk_at(int key, int x) { return (x >> 2) * 1024 + (x & 3) * 256 + ((key ^ (4 * (x & 3))) * 16); }

// 4 codes in the bytes of w (biased so that byte - off is the code) times d: rounded to f16, and what the rounding left (exact: the product is a
// multiple of 2^-24 of at most 18 bits)
// NPL = 0: the code itself.
template <int NPL> __device__ __forceinline__ void times4(uint32_t w, float off, h2 d, uint32_t * hi, uint32_t * lo) {
    const h2 o = {(half_t) off, (half_t) off};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, k ? 0x04030402u : 0x04010400u)) - o;
        const h2 p = NPL == 0 ? c : c * d;
        hi[k] = __builtin_bit_cast(uint32_t, p);
        if constexpr (NPL == 2) lo[k] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, d, -p));
    }
}

// ... the codes alone
__device__ __forceinline__ void codes4(uint32_t w, float off, uint32_t * c) {
    const h2 o = {(half_t) off, (half_t) off};
#pragma unroll
    for (int k = 0; k < 2; ++k) c[k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, k ? 0x04030402u : 0x04010400u)) - o);
}

// A wave's part in filling one group: every lane stands for one key (row) of it
template <uint32_t KT, int D, int NPL> struct group;

template <int D, int NPL> struct group<P1A_KV_F16, D, NPL> {
    static constexpr bool DIRECT = true;
    static __device__ __forceinline__ int key(int lane) { return (lane & 15) ^ (4 * (lane >> 4)); }
    static constexpr int PIECES = D / 32;                     // loads of a group
    struct raw {};
    // load j, straight to LDS: complete when vmcnt says so. (The instruction adds its offset to both addresses. s_nop: one
    // instruction has to stand between the write of M0 and a load that goes by it, and the compiler does not look in here.)
    template <int j> static __device__ __forceinline__ void piece(raw &, gbytes row, char * to, int lane) {
        asm volatile("s_add_u32 m0, %1, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:%3" :: "v"(row + (lane >> 4) * 16), "s"(__builtin_amdgcn_readfirstlane(lds_at(to))), "i"(960 * j), "i"(64 * j)
                     : "memory", "m0", "scc");
    }
    static __device__ __forceinline__ void load(gbytes row, char * to, int lane) {
        raw r;
        each<PIECES>([&](auto j) __attribute__((always_inline)) { piece<j>(r, row, to, lane); });
    }
};

template <int D, int NPL> struct group<P1A_KV_Q8_0, D, NPL> {
    static constexpr bool DIRECT = false;
    static constexpr int NJ = D / 64, NB = D / 32;            // loads of 16 codes a lane; blocks of a row
    static constexpr int PIECES = NJ + 1;
    struct raw { u4 w[NJ]; uint32_t d[NB / 2]; };
    static __device__ __forceinline__ int key(int lane) { return lane & 15; }
    static __device__ __forceinline__ void load(raw & r, gbytes row, int lane) {
        each<PIECES>([&](auto j) __attribute__((always_inline)) { piece<j>(r, row, nullptr, lane); });
    }
    template <int j> static __device__ __forceinline__ void piece(raw & r, gbytes row, char *, int lane) {
        if constexpr (j < NJ) r.w[j] = gload<u4_a4>(row + 2 * NB + (4 * j + (lane >> 4)) * 16);
        else if constexpr (NB == 8) { const u4 t = gload<u4_a4>(row); r.d[0] = t[0]; r.d[1] = t[1]; r.d[2] = t[2]; r.d[3] = t[3]; }
        else if constexpr (NB == 4) { const u2w t = gload<u2_a4>(row); r.d[0] = t[0]; r.d[1] = t[1]; }
        else r.d[0] = gload<uint32_t>(row);
    }
    static __device__ __forceinline__ void store(const raw & r, char * to, int lane) {
        const int q = lane >> 4, k = lane & 15;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {                        // codes of part 4 j + q: block 2 j + q / 2, chunks 8 j + 2 q and the next
            const uint32_t s = q & 2 ? r.d[j] >> 16 : r.d[j] & 0xffff;
            const h2 d = __builtin_bit_cast(h2, s | (s << 16));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                u4 hi, lo;
                uint32_t h[4], l[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) times4<NPL>(r.w[j][2 * x + e] ^ 0x80808080u, 1152.f, d, h + 2 * e, l + 2 * e);
                hi = u4{h[0], h[1], h[2], h[3]};
                char * at = to + chunk_at(k, 8 * j + 2 * q + x);
                *reinterpret_cast<u4 *>(at) = hi;
                if constexpr (NPL == 2) { lo = u4{l[0], l[1], l[2], l[3]}; *reinterpret_cast<u4 *>(at + plane_bytes(D)) = lo; }
            }
        }
    }
};

template <int D, int NPL> struct group<P1A_KV_Q4_0, D, NPL> {
    static constexpr bool DIRECT = false;
    static constexpr int NB = D / 32, NJ = (NB + 3) / 4;      // blocks of a row; of a lane
    static constexpr int PIECES = NJ;
    struct raw { u4 w[NJ]; uint32_t d[NJ]; };
    static __device__ __forceinline__ int key(int lane) { return lane & 15; }
    template <int j> static __device__ __forceinline__ void piece(raw & r, gbytes row, char *, int lane) {
        const gbytes b = row + min(4 * j + (lane >> 4), NB - 1) * 18;
        r.d[j] = gload<uint16_t>(b);
        r.w[j] = gload<u4_a2>(b + 2);
    }
    static __device__ __forceinline__ void load(raw & r, gbytes row, int lane) {
        each<PIECES>([&](auto j) __attribute__((always_inline)) { piece<j>(r, row, nullptr, lane); });
    }
    static __device__ __forceinline__ void store(const raw & r, char * to, int lane) {
        const int k = lane & 15;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int b = 4 * j + (lane >> 4);
            if (NB % 4 && b >= NB) break;
            const h2 d = __builtin_bit_cast(h2, r.d[j] | (r.d[j] << 16));
#pragma unroll
            for (int x = 0; x < 4; ++x) {                     // values 8 x ..: bytes 8 (x & 1) .., low nibbles, then high ones
                uint32_t h[4], l[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t w = r.w[j][2 * (x & 1) + e];
                    times4<NPL>((x & 2 ? w >> 4 : w) & 0x0f0f0f0fu, 1032.f, d, h + 2 * e, l + 2 * e);
                }
                char * at = to + chunk_at(k, 4 * b + x);
                *reinterpret_cast<u4 *>(at) = u4{h[0], h[1], h[2], h[3]};
                if constexpr (NPL == 2) *reinterpret_cast<u4 *>(at + plane_bytes(D)) = u4{l[0], l[1], l[2], l[3]};
            }
        }
    }
};

// The 32 keys of groups 2 u and 2 u + 1 as rows of a 32 x 16 operand: lane (row c, half g) reads chunk 2 ks + g of key c in step ks. base: what of
// the address depends on the lane, for even and odd steps
struct k_frag {
    int base[2];
    __device__ __forceinline__ k_frag(int lane, int group_bytes) {
        const int c = lane & 31, g = lane >> 5;
#pragma unroll
        for (int o = 0; o < 2; ++o) base[o] = (c >> 4) * group_bytes + chunk_at(c & 15, 2 * o + g);
    }
    __device__ __forceinline__ h8 read(const char * groups, int ks) const { return *reinterpret_cast<const h8 *>(groups + base[ks & 1] + (ks >> 1) * 1024); }
};
// V^T as a 32 x 16 operand: lane (row c: dim 32 dt + c, half g) gets keys 4 g .. 4 g + 3 and 8 + 4 g .. of one group - the order in which the result
// of S^T holds its 16 keys
struct v_frag {
    int base[2];
    __device__ __forceinline__ v_frag(int lane) {
        const int g = lane >> 5, i16 = lane & 15, kk = i16 >> 2, jq = i16 & 3, x = 2 * ((lane >> 4) & 1) + (jq >> 1);
#pragma unroll
        for (int o = 0; o < 2; ++o) base[o] = chunk_at(4 * g + kk + 8 * o, x) + (jq & 1) * 8;
    }
    __device__ __forceinline__ h8 read(const char * grp, int dt) const {
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4 __attribute__((address_space(3))) *) (grp + base[0] + dt * 1024));
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s4 __attribute__((address_space(3))) *) (grp + base[1] + dt * 1024));
        const h4 a = __builtin_bit_cast(h4, lo), b = __builtin_bit_cast(h4, hi);
        return h8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
};

__device__ __forceinline__ f16x mfma32(h8 a, h8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// the larger of two numbers, in one instruction (fmaxf has to make a NaN quiet first). top: infinity, in a register the compiler knows nothing about
__device__ __forceinline__ float larger(float a, float b, float top) { return __builtin_amdgcn_fmed3f(a, b, top); }
// row of value i of a lane (half g) of a 32 x 32 result
__device__ __forceinline__ constexpr int mfma_row(int i, int g) { return 8 * (i >> 2) + 4 * g + (i & 3); }

// 4 consecutive values of a row of q, as f32
__device__ __forceinline__ f4 q4_at(const void * q, bool bf16, size_t i) {
    if (!bf16) return *(const __attribute__((address_space(1))) f4 *) ((gbytes) q + 4 * i);
    const u2w w = *(const __attribute__((address_space(1))) u2w *) ((gbytes) q + 2 * i);
    return f4{__builtin_bit_cast(float, w[0] << 16), __builtin_bit_cast(float, w[0] & 0xffff0000u), __builtin_bit_cast(float, w[1] << 16), __builtin_bit_cast(float, w[1] & 0xffff0000u)};
}
// f32 -> bf16, to nearest, ties to even (a NaN stays one)
__device__ __forceinline__ uint32_t bf16_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return x == x ? (u + 0x7fffu + ((u >> 16) & 1)) >> 16 : 0x7fc0u;
}

// ---- 16 keys straight from memory as the rows of a 16 x 32 operand ----
// Lane (key c = lane % 16, group g = lane / 16) reads the 8 values of each 32-dim block that it feeds to the products: 16, 8 or 4 bytes, 64, 32 or 16 on
// end for a key. Codes enter as the whole numbers they are (exact in f16); a block's scale multiplies its fp32 result, from a table in LDS that
// turns scales by key into scales by result (lane group g holds keys 4 g ..).
template <uint32_t KT, int D> struct keys16 {
    static constexpr bool F16 = KT == P1A_KV_F16, Q8 = KT == P1A_KV_Q8_0;
    static constexpr int NB = D / 32, NSC = (NB + 3) / 4, SC = Q8 ? 2 : 18;   // blocks; scales a lane fetches; their distance
    static constexpr int TAB = F16 ? 0 : NB * 16;             // floats of the table
    typedef uint32_t u1_a2 __attribute__((aligned(2)));
    static constexpr bool PAIRS = Q8 && NB == 8;              // two scales side by side in one load
    struct scales { uint16_t s[F16 || PAIRS ? 1 : NSC]; uint32_t two; };
    // the block of a lane's scale x (lanes without a block of their own repeat the last one)
    static __device__ __forceinline__ int block(int x, int g) { return PAIRS ? 2 * g + x : min(4 * x + g, NB - 1); }
    struct raw {
        u4 w[F16 ? NB : 1];
        u2w w8[Q8 ? NB : 1];
        uint32_t w4[!F16 && !Q8 ? NB : 1];
        scales d;
    };
    // dims of the 8 slots of lane group g in a block: two runs of four
    static __device__ __forceinline__ int dims(int g, int half) { return F16 || Q8 ? 8 * g + 4 * half : 4 * g + 16 * half; }
    static __device__ __forceinline__ void load_scales(scales & r, gbytes row, int g) {
        if constexpr (PAIRS) r.two = gload<uint32_t>(row + 4 * g);
        else if constexpr (!F16) {
#pragma unroll
            for (int x = 0; x < NSC; ++x) r.s[x] = gload<uint16_t>(row + block(x, g) * SC);
        }
    }
    static __device__ __forceinline__ void load(raw & r, gbytes row, int g) {
        load_scales(r.d, row, g);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if constexpr (F16) r.w[b] = gload<u4>(row + 64 * b + 16 * g);
            else if constexpr (Q8) r.w8[b] = gload<u2_a4>(row + 2 * NB + 32 * b + 8 * g);
            else r.w4[b] = gload<u1_a2>(row + 18 * b + 2 + 4 * g);
        }
    }
    static __device__ __forceinline__ float scale(const scales & r, int x) { return (float) (PAIRS ? __builtin_bit_cast(h2, r.two)[x & 1] : __builtin_bit_cast(half_t, r.s[PAIRS ? 0 : x])); }
    static __device__ __forceinline__ void put(float * table, const scales & r, int c, int g, int shift = 0) {
        if constexpr (!F16) {
#pragma unroll
            for (int x = 0; x < NSC; ++x) table[block(x, g) * 16 + c] = ldexpf(scale(r, x), shift);
        }
    }
    static __device__ __forceinline__ h8 operand(const raw & r, int b) {
        if constexpr (F16) return __builtin_bit_cast(h8, r.w[b]);
        else {
            uint32_t a[4];
            if constexpr (Q8) {
                codes4(r.w8[b][0] ^ 0x80808080u, 1152.f, a);
                codes4(r.w8[b][1] ^ 0x80808080u, 1152.f, a + 2);
            } else {
                codes4(r.w4[b] & 0x0f0f0f0fu, 1032.f, a);
                codes4((r.w4[b] >> 4) & 0x0f0f0f0fu, 1032.f, a + 2);
            }
            return __builtin_bit_cast(h8, u4{a[0], a[1], a[2], a[3]});
        }
    }
    // S^T of two times 16 keys and NT tiles of 16 columns: value i of lane (column c, group g) is key 4 g + i. q(n, k, b): half k of block b of tile n's
    // operand. (Both halves side by side, and a block's scales asked for a block ahead: a product's result and LDS take a hundred clocks and more.)
    template <int NT, int NQ, class Q> static __device__ __forceinline__ void scores(const raw (&r)[2], Q && q, const float * table, int g, f4 (&s)[2][NT]) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int n = 0; n < NT; ++n) s[x][n] = f4{0.f, 0.f, 0.f, 0.f};
        f4 d[2], dn[2];
        auto fetch = [&](int b) {
            if constexpr (!F16) {
#pragma unroll
                for (int x = 0; x < 2; ++x) dn[x] = *reinterpret_cast<const f4 *>(table + x * TAB + b * 16 + 4 * g);
            }
        };
        fetch(0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if constexpr (!F16) {
                d[0] = dn[0];
                d[1] = dn[1];
                if (b + 1 < NB) fetch(b + 1);
            }
            h8 a[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) a[x] = operand(r[x], b);
            f4 t[2][NT];
#pragma unroll
            for (int k = 0; k < NQ; ++k)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const h8 qq = q(n, k, b);
#pragma unroll
                    for (int x = 0; x < 2; ++x) t[x][n] = mfma16(a[x], qq, k ? t[x][n] : F16 ? s[x][n] : f4{0.f, 0.f, 0.f, 0.f});
                }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if constexpr (F16) s[x][n] = t[x][n];
                    else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[x][n][i] = fmaf(t[x][n][i], d[x][i], s[x][n][i]);
                        asm volatile("" : "+v"(s[x][n]));     // (here: put off behind the next branch, every block's t and d would stay in registers)
                    }
                }
        }
    }
};
// 16 columns of q for it: lane (column c, group g). Returns the factor's exponent (the same in the column's four lanes)
template <uint32_t KT, int D, int NQ> __device__ __forceinline__ int q_columns(const void * q, bool bf16, size_t row, float sign, int g, h8 (&qf)[NQ][D / 32]) {
    constexpr int NB = D / 32;
    f4 x[NB][2];
    auto fetch = [&](auto as_bf16) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[b][e] = q4_at(q, as_bf16, row * D + 32 * b + keys16<KT, D>::dims(g, e));
    };
    if (bf16) fetch(std::true_type{});
    else fetch(std::false_type{});
    float most = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[b][e >> 2][e & 3]));
    const int ex = row_exponent(max_swap32(max_swap16(most)));
    const float by = ldexpf(sign, -ex);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        h8 r[NQ];
        halves<NQ>([&](int e) { return x[b][e >> 2][e & 3]; }, [&](int) { return by; }, r);
#pragma unroll
        for (int k = 0; k < NQ; ++k) qf[k][b] = r[k];
    }
    return ex;
}

// ---- few rows a sequence: steps of 32 TPS keys, counted through over the sequences, in runs of equal length ----
// A sequence with rows has one step at least. Lane i of a wave counts for sequence s0 + i and keeps what it found out about the first 64 (all of
// them, mostly).
template <int TPS> struct step_runs {
    // first row, its position, where the page-table row begins; rows (32 at most) and steps (2^30 positions: 2^23 and one) share a register - the first row may be
    // anything up to 2^30
    struct of_lane {
        int first, pos0, table, work;
        static __host__ __device__ __forceinline__ int both(int steps, int rows) { return steps << 6 | rows; }
        __host__ __device__ __forceinline__ int steps() const { return work >> 6; }
        __host__ __device__ __forceinline__ int rows() const { return work & 63; }
    };
    of_lane first64;
    int first, end, per;                                      // this run's steps; steps of a run
    static __device__ __forceinline__ span span_of_rows(const rows_view & R, const seq_view & v) { return span_of<32>(R, v.pos0, v.pos0 + v.count - 1); }
    static __device__ __forceinline__ of_lane look(const rows_view & R, const kv_view & pg, int s) {
        of_lane r{0, 0, 0, 0};
        if (s >= R.n_seq) return r;
        const seq_view v = seq_of(R, s);
        r.table = pg.pt && pg.rtab ? pg.rtab[s] : 0;
        r.first = v.first;
        r.pos0 = v.pos0;
        r.work = v.count < 1 ? 0 : r.both(max((span_of_rows(R, v).nt + TPS - 1) / TPS, 1), v.count);
        return r;
    }
    // run number `run` of `runs`; no sequence in more than `most_runs` of them. False: there is nothing for it
    __device__ __forceinline__ bool begin(const rows_view & R, const kv_view & pg, int run, int runs, int most_runs) {
        const int lane = threadIdx.x & 63;
        first64 = look(R, pg, lane);
        int n = 0, most = 0;
        for (int s0 = 0; s0 < R.n_seq; s0 += 64) {
            const int x = s0 ? look(R, pg, s0 + lane).steps() : first64.steps();
            n += __builtin_amdgcn_readlane(lanes_up_to(x), 63);
            most = max(most, x);
        }
        most = rfl((int) wave_max((float) most));             // (2^24 steps at most: exact)
        per = max((n + runs - 1) / runs, (most + most_runs - 2) / (most_runs - 1));
        first = run * per;
        end = min(first + per, n);
        return first < end;
    }
    // the sequence that holds step `at` (of begin()'s run), where its steps begin and how many it has. False: none does - row0 or pos0 have been
    // written since begin() read them
    struct found { int seq, first, steps, table; seq_view v; };
    __device__ __forceinline__ bool find(const rows_view & R, const kv_view & pg, int at, int lane, found & f) const {
        int base = 0;
        for (int s0 = 0; s0 < R.n_seq; s0 += 64) {
            const of_lane x = s0 ? look(R, pg, s0 + lane) : first64;
            const int u = base + lanes_up_to(x.steps());
            const unsigned long long behind = __ballot(u > at);
            if (behind) {
                const int l = __builtin_ctzll(behind);
                const of_lane at_l{0, 0, 0, __builtin_amdgcn_readlane(x.work, l)};
                f.seq = s0 + l;
                f.steps = at_l.steps();
                f.first = __builtin_amdgcn_readlane(u, l) - f.steps;
                f.v.first = __builtin_amdgcn_readlane(x.first, l);
                f.v.count = at_l.rows();
                f.v.pos0 = __builtin_amdgcn_readlane(x.pos0, l);
                f.table = __builtin_amdgcn_readlane(x.table, l);
                return true;
            }
            base = __builtin_amdgcn_readlane(u, 63);
        }
        return false;
    }
};
// The rows of a lane's keys: key c of each half of a tile of 32
struct key_rows {
    const span & sp;
    const kv_view & pg;
    const int32_t * ptab;
    size_t head_off;
    int c;
    struct pages { int p[2]; };
    struct where { size_t off[2]; };
    __device__ __forceinline__ int pos(int tile, int x) const { return seen_or_near<32>(sp, tile * 32, tile * 32 + 16 * x + c); }
    __device__ __forceinline__ pages pages_of(int tile) const {
        pages r;
#pragma unroll
        for (int x = 0; x < 2; ++x) r.p[x] = ptab ? ptab[pos(tile, x) >> pg.psh] : 0;
        return r;
    }
    __device__ __forceinline__ where at(int tile, const pages & e) const {
        where r;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int j = pos(tile, x);
            r.off[x] = head_off + (ptab ? (size_t) e.p[x] * pg.pstride + (size_t) (j & ((1 << pg.psh) - 1)) * pg.rowb : (size_t) j * pg.rowb);
        }
        return r;
    }
};

// ---- attention of chunks: what its kernels share ----
constexpr float HEAD = 8.f, STEP = 6.f;                       // log2 of P at the row's maximum: HEAD when the reference moves, at most HEAD + STEP
struct chunk_params {
    const void * q;
    void * out;
    const float * gate;
    float * lse;
    const char * kc;
    const char * vc;
    kv_view pg;
    rows_view R;
    int Hq, Hkv, GQA;
    uint32_t gqa_magic;    // floor(2^32 / GQA) (2^32 - 1 for GQA = 1)
    float factor, sign;    // scores are factor * (sign q . k), in log2 units; factor > 0
    int q_bf16, out_bf16;
    int nks;               // partials of a row: workgroups of a block, or the most runs that a sequence of few rows may lie in
    int runs;              // few rows: workgroups of a kv head
    int * part_n;          // few rows: [n_seq] runs that the sequence lies in
    float * part_o;        // [T * Hq][nks][D], relative to r
    float * part_ml;       // [T * Hq][nks][2]: r, l
};
// A row that sees something has itself to see: whether it sees nothing (result 0, log-sum-exp -inf) is a matter of its position. Where q holds a NaN or an infinity
// all its scores may be NaN: no maximum, so r = -inf as if nothing had been seen, but l is NaN, and result and log-sum-exp become that. As a partial such a row
// says so with a reference of 0.
__device__ __forceinline__ float part_ref(float r, float l) { return r == MINUS_INF && !(l == 0.f) ? 0.f : r; }
__device__ __forceinline__ float gate_of(float g) { return 1.0f / (1.0f + expf(-g)); }
// four results of a row, at element i of out
__device__ __forceinline__ void put4(void * out, bool bf16, size_t i, f4 v) {
    if (!bf16) *(__attribute__((address_space(1))) f4 *) ((__attribute__((address_space(1))) char *) out + 4 * i) = v;
    else *(__attribute__((address_space(1))) u2w *) ((__attribute__((address_space(1))) char *) out + 2 * i) =
        u2w{bf16_of(v[0]) | bf16_of(v[1]) << 16, bf16_of(v[2]) | bf16_of(v[3]) << 16};
}

// host side (p1a_api.hip)
// What the library's own buffers are asked for where a call has these bytes: the next power of two. A buffer that is replaced stays allocated (a recorded graph may
// hold it), and there is room for so many only: calls that grow row by row replace it a dozen times, not each time.
inline size_t kept_bytes(size_t bytes) {
    size_t n = 64 << 10;
    while (n < bytes) n *= 2;
    return n;
}
struct chunk_args {
    const void * q; void * out; const float * gate; float * lse;
    bool q_bf16, out_bf16;
    rows_view R;
    int Hq, max_n;
    float scale;
    void * scratch; size_t scratch_bytes;
};
int launch_chunk(const p1a_kv & c, const chunk_args & a, hipStream_t s);
struct chunk_plan {
    int few;                           // tiles of 16 columns that hold a sequence's rows under a kv head (p1a_step.hip), or 0
    int nks, runs;                     // as in chunk_params
    size_t bytes_n, bytes_ml, bytes_o; // scratch (0: no partials), in this order
};
chunk_plan plan_chunk(const p1a_kv & c, const rows_view & R, int Hq, int max_n, int cus);
int launch_step(const p1a_kv & c, const chunk_params & P, int NT, bool exact, hipStream_t s);
struct mass_args {
    const void * q; bool q_bf16; const float * lse; float * mass;
    int ld;
    rows_view R;
    int Hq, max_n;
    float scale;
    void * scratch; size_t scratch_bytes;
};
struct mass_plan { int few, runs, blocks, splits, pld; size_t bytes; };   // (few as in chunk_plan; pld: positions of a partial row; bytes of scratch)
mass_plan plan_mass(const p1a_kv & c, const rows_view & R, int Hq, int max_n, int ld, int cus);
int launch_mass(const p1a_kv & c, const mass_args & a, hipStream_t s);
constexpr long long MOST_GROUPS = (1LL << 32) / 256 - 1;     // workgroups of 256 threads that one launch holds
struct tree_plan {
    int NT, max_groups;                // tiles of 16 columns of a wave; groups of waves' columns that a sequence may have
    int nks, runs;                     // as in chunk_params
    size_t bytes_n, bytes_ml, bytes_o; // scratch (0: no partials), in this order
};
tree_plan plan_tree(const p1a_kv & c, const rows_view & R, int Hq, int max_n, bool exact, int cus);
int launch_tree(const p1a_kv & c, const chunk_args & a, const uint32_t * mask, int words, hipStream_t s);
int launch_tree_rows(const int32_t * parent, const rows_view & R, uint32_t * mask, int words, int32_t * pos, int32_t * slot, hipStream_t s);
int launch_tree_commit(const p1a_kv * layers, int n_layers, const rows_view & R, const int32_t * n_accept, const int32_t * path, int ld_path, hipStream_t s);
struct verify_args {
    const void * target, * draft;
    size_t ld_target, ld_draft;
    const int32_t * token, * parent;
    const float * temp, * u, * u_next;
    int32_t * n_accept, * path, * next;
    rows_view R;
    int V, ld_path, max_children;
    bool target_bf16, draft_bf16, logits, distinct;
    void * scratch; size_t scratch_bytes;
};
struct verify_plan { int stretches; size_t at[16], bytes; };   // stretches of a row; where the parts of the scratch begin (p1a_verify.hip), and all of it
verify_plan plan_verify(const rows_view & R, int V, bool logits, bool draft);
int launch_verify(const verify_args & a, hipStream_t s);
int launch_evict_select(const float * mass, int ld, int n_seq, int Hkv, const int32_t * n_dev, int n, int budget, int n_sink, int n_recent, int32_t * keep, hipStream_t s);
int launch_kv_compact(const p1a_kv & c, const int32_t * keep, int n_seq, int budget, const float * mass, float * mass_out, int ld, hipStream_t s);

}   // namespace p1a
