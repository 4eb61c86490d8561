// Eviction from a cache by accumulated attention weight (gfx950): which positions stay, and moving their rows to the front of the sequence's pages.
#include "p1a_tiles.hpp"

namespace p1a {
namespace {

// ---- which positions stay ----
// One workgroup per (sequence, kv head): the want-th largest of the positions between the sinks and the last ones by radix selection, 8 bits of the
// value a pass - until what shares the digits so far is wanted as a whole -, then one pass that lists what is above it, and of what equals it the first
// ones, in order. A thread holds 16 consecutive values of a part of 16384; longer rows are read again for each pass (from L2). Counts go to 32 copies of
// the histogram, one for every other lane: values of one order of magnitude share their first digit, and additions to one address wait for each other.
// What bounds it: one compute unit's vector instructions a row, some 15 a value and pass: 1100 positions 8 us, 8190 14, 100003 72. (Eleven bits a pass,
// fewer passes, values kept in registers or LDS or asked for ahead took 92 to 145 there; several workgroups a row, their counts in scratch, have not
// been built: eight rows leave 248 compute units idle.)
constexpr int STHR = 1024, PER = 16, PART = STHR * PER;

// larger values have larger keys; -0 is 0, a NaN is below everything
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x == x ? u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u) : 0u;
}

__global__ void __launch_bounds__(STHR) select_k(const float * mass, int ld, const int32_t * n_dev, int n_host, int budget, int n_sink, int n_recent, int32_t * keep_) {
    constexpr int COPIES = 32, HS = COPIES + 1;
    __shared__ uint32_t hist[256 * HS];
    __shared__ uint32_t count[256];
    __shared__ uint32_t wsum[STHR / 64];
    __shared__ uint32_t found[3];                             // digit, how many of it are still wanted, how many there are
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.x, s = blockIdx.y;
    const size_t row = (size_t) s * gridDim.x + h;
    const float * const m = mass + row * ld;
    int32_t * const keep = keep_ + row * budget;
    const int n = min(max(n_dev ? n_dev[s] : n_host, 0), ld);
    if (n <= budget) {
        for (int i = tid; i < budget; i += STHR) keep[i] = i < n ? i : -1;
        return;
    }
    const int a = n_sink, b = n - n_recent, want = budget - n_sink - n_recent;   // (b - a > want)
    for (int i = tid; i < n_sink; i += STHR) keep[i] = i;
    for (int i = tid; i < n_recent; i += STHR) keep[budget - n_recent + i] = b + i;
    if (want == 0) return;
    const int parts = (b - a + PART - 1) / PART;
    uint32_t key[PER];
    int held = -1;
    auto hold = [&](int part) {                               // (a key past the end: 0)
        if (held == part) return;
        held = part;
        const int i0 = a + part * PART + tid * PER;
        if (i0 + PER <= b) {
#pragma unroll
            for (int x = 0; x < PER; x += 4) {
                const u4 v = gload<u4_a4>((gbytes) (m + i0 + x));
#pragma unroll
                for (int e = 0; e < 4; ++e) key[x + e] = key_of(__builtin_bit_cast(float, (uint32_t) v[e]));
            }
        } else {
#pragma unroll
            for (int x = 0; x < PER; ++x) key[x] = i0 + x < b ? key_of(m[i0 + x]) : 0u;
        }
    };
    uint32_t prefix = 0, left = (uint32_t) want, low = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256 * HS; i += STHR) hist[i] = 0;
        __syncthreads();
        for (int part = 0; part < parts; ++part) {
            hold(part);
            // (keys past the end are 0 and count as such: the last digit looked at then seems to hold more than are there, never fewer than are wanted)
            uint32_t * const mine = hist + (lane & 31);
            if (shift == 24) {
#pragma unroll
                for (int x = 0; x < PER; ++x) atomicAdd(&mine[(key[x] >> 24) * HS], 1u);
            } else {
#pragma unroll
                for (int x = 0; x < PER; ++x)
                    if ((key[x] ^ prefix) >> (shift + 8) == 0) atomicAdd(&mine[((key[x] >> shift) & 255) * HS], 1u);
            }
        }
        __syncthreads();
        {
            uint32_t t = 0;
#pragma unroll
            for (int x = 0; x < COPIES / 4; ++x) t += hist[(tid >> 2) * HS + (tid & 3) * (COPIES / 4) + x];
            t += __shfl_xor(t, 1);
            t += __shfl_xor(t, 2);
            if ((tid & 3) == 0) count[tid >> 2] = t;
        }
        __syncthreads();
        if (wave == 0) {                                      // lane l: digits 255 - 4 l .. 252 - 4 l, the largest first
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) { c[x] = count[255 - 4 * lane - x]; sum += c[x]; }
            uint32_t upto = sum;
            for (int d = 1; d < 64; d <<= 1) { const uint32_t y = __shfl_up(upto, d); if (lane >= d) upto += y; }
            uint32_t before = upto - sum;
            if (before < left && left <= upto) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (before < left && left <= before + c[x]) { found[0] = 255 - 4 * lane - x; found[1] = left - before; found[2] = c[x]; }
                    before += c[x];
                }
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        left = found[1];
        low = found[2] == left ? prefix : prefix + 1;         // (no value has the largest key)
        if (low == prefix) break;
        __syncthreads();
    }
    // from `low` on: all; equal to `prefix` below it: the first `left`
    uint32_t gt0 = 0, eq0 = 0;                                // of the parts behind
    for (int part = 0; part < parts; ++part) {
        hold(part);
        const int i0 = a + part * PART + tid * PER, live = b - i0;
        uint32_t mine = 0;                                    // from `low` on, and equal in the upper half
#pragma unroll
        for (int x = 0; x < PER; ++x)
            if (x < live) mine += key[x] >= low ? 1u : key[x] == prefix ? 0x10000u : 0u;
        uint32_t upto = mine;
        for (int d = 1; d < 64; d <<= 1) { const uint32_t y = __shfl_up(upto, d); if (lane >= d) upto += y; }
        if (lane == 63) wsum[wave] = upto;
        __syncthreads();
        uint32_t before = upto - mine, all = 0;
        for (int w = 0; w < STHR / 64; ++w) { const uint32_t y = wsum[w]; all += y; if (w < wave) before += y; }
        uint32_t gt = gt0 + (before & 0xffff), eq = eq0 + (before >> 16);
#pragma unroll
        for (int x = 0; x < PER; ++x) {
            if (x >= live) break;
            const bool above = key[x] >= low, equal = !above && key[x] == prefix;
            if (above || (equal && eq < left)) keep[n_sink + gt + min(eq, left)] = i0 + x;
            gt += above;
            eq += equal;
        }
        gt0 += all & 0xffff;
        eq0 += all >> 16;
        __syncthreads();
    }
}

// ---- moving what stays ----
// A row k only ever receives a row from behind it, so one workgroup that walks k upwards - fetch a stretch of rows, wait until every wave has, write
// it - never loses one, without a copy. What is split over workgroups is the row: a slice of its bytes moves on its own. (The slices of a row go to
// one XCD, whose L2 holds their common lines.) One workgroup more per (sequence, kv head) moves the row of totals.
template <int W> struct word_of;
template <> struct word_of<16> { typedef u4 type; };
template <> struct word_of<8> { typedef u2w type; };
template <> struct word_of<4> { typedef uint32_t type; };
template <> struct word_of<2> { typedef uint16_t type; };

struct move_params {
    char * kc, * vc;
    kv_view pg;
    const int32_t * keep;
    const float * mass;
    float * mass_out;
    int n_seq, Hkv, budget, ld, n_ctx, hb;
    int words, per_sh, slices;   // words of a head's row; log2 of those of a slice; slices of a row
    int units;                   // (sequence, kv head, K or V), then (sequence, kv head) for the totals
};
constexpr int MTHR = 1024, DEPTH = 4;
__device__ __forceinline__ void all_fetched() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int W> __global__ void __launch_bounds__(MTHR) move_k(const move_params P) {
    typedef typename word_of<W>::type word;
    typedef __attribute__((address_space(1))) word * gword;
    const int xcd = blockIdx.x & 7, lin = blockIdx.x >> 3, unit = lin / P.slices * 8 + xcd, slice = lin % P.slices, tid = threadIdx.x;
    const int rows = P.n_seq * P.Hkv;
    if (unit >= P.units) return;
    if (unit >= 2 * rows) {                                   // totals
        if (slice) return;
        const int r = unit - 2 * rows;
        const int32_t * const keep = P.keep + (size_t) r * P.budget;
        const float * const m = P.mass + (size_t) r * P.ld;
        float * const to = P.mass_out + (size_t) r * P.ld;
        const int last = min(P.budget, P.ld);
        for (int k0 = 0; k0 < last; k0 += MTHR * DEPTH) {
            float x[DEPTH];
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int k = k0 + d * MTHR + tid, j = k < last ? keep[k] : -1;
                x[d] = j >= k && j < P.ld ? m[j] : 0.f;
            }
            all_fetched();
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) if (k0 + d * MTHR + tid < last) to[k0 + d * MTHR + tid] = x[d];
        }
        for (int k = last + tid; k < P.ld; k += MTHR) to[k] = 0.f;
        return;
    }
    const int v = unit >= rows, r = unit - v * rows, s = r / P.Hkv, h = r - s * P.Hkv;
    const int32_t * const keep = P.keep + (size_t) r * P.budget;
    const int32_t * const ptab = P.pg.pt ? P.pg.pt + (P.pg.rtab ? P.pg.rtab[s] : 0) : nullptr;
    char * const base = (v ? P.vc : P.kc) + (size_t) h * P.hb;
    const int per = 1 << P.per_sh, w = slice * per + (tid & (per - 1)), rpi = MTHR >> P.per_sh;
    const bool mine = w < P.words;
    // Three things in a row - which position, its page, its bytes - asked for in one go, of three stretches: positions two ahead, pages one
    auto kept = [&](int (&src)[DEPTH], int k0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int k = k0 + d * rpi + (tid >> P.per_sh);
            src[d] = mine && k < P.budget ? keep[k] : -1;
        }
    };
    auto moves = [&](int from, int k) { return from > k && from < P.n_ctx; };
    auto pages = [&](const int (&src)[DEPTH], int (&fp)[DEPTH], int (&tp)[DEPTH], int k0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int k = k0 + d * rpi + (tid >> P.per_sh);
            const bool go = moves(src[d], k);
            fp[d] = go && ptab ? ptab[src[d] >> P.pg.psh] : 0;
            tp[d] = go && ptab ? ptab[k >> P.pg.psh] : 0;
        }
    };
    auto where = [&](int j, int page) {
        return (ptab ? (size_t) page * P.pg.pstride + (size_t) (j & ((1 << P.pg.psh) - 1)) * P.pg.rowb : (size_t) j * P.pg.rowb) + (size_t) w * W;
    };
    const int step = rpi * DEPTH;
    int src[DEPTH], next[DEPTH], fp[DEPTH], tp[DEPTH];
    kept(src, 0);
    kept(next, step);
    pages(src, fp, tp, 0);
    for (int k0 = 0; k0 < P.budget; k0 += step) {
        word x[DEPTH];
        size_t to[DEPTH];
        bool go[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int k = k0 + d * rpi + (tid >> P.per_sh);
            go[d] = moves(src[d], k);
            if (go[d]) x[d] = *(gword) (base + where(src[d], fp[d]));
            to[d] = where(k, tp[d]);
        }
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) src[d] = next[d];
        pages(src, fp, tp, k0 + step);
        kept(next, k0 + 2 * step);
        all_fetched();
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) if (go[d]) *(gword) (base + to[d]) = x[d];
    }
}

}   // namespace

int launch_evict_select(const float * mass, int ld, int n_seq, int Hkv, const int32_t * n_dev, int n, int budget, int n_sink, int n_recent, int32_t * keep, hipStream_t s) {
    select_k<<<dim3(Hkv, n_seq), STHR, 0, s>>>(mass, ld, n_dev, n, budget, n_sink, n_recent, keep);
    return launched();
}

int launch_kv_compact(const p1a_kv & c, const int32_t * keep, int n_seq, int budget, const float * mass, float * mass_out, int ld, hipStream_t s) {
    move_params P;
    P.kc = (char *) c.k; P.vc = (char *) c.v; P.pg = view_of(c); P.keep = keep; P.mass = mass; P.mass_out = mass_out;
    P.n_seq = n_seq; P.Hkv = c.Hkv; P.budget = budget; P.ld = ld; P.n_ctx = c.n_ctx;
    P.hb = (int) head_bytes(c.type, c.D);
    const size_t al = (size_t) c.k | (size_t) c.v | (size_t) P.hb | P.pg.rowb | (c.pt ? c.pstride : 0);
    const int W = al & 15 ? al & 7 ? al & 3 ? 2 : 4 : 8 : 16;
    P.words = P.hb / W;
    // slices of 64 bytes, or down to 16 while that leaves compute units without a workgroup
    int bytes = 64;
    const long long rows = 2LL * n_seq * c.Hkv;
    while (bytes > 16 && rows * ((P.hb + bytes - 1) / bytes) < cu_count()) bytes /= 2;
    P.per_sh = __builtin_ctz((unsigned) (bytes / W > 1 ? bytes / W : 1));
    P.slices = (P.words + (1 << P.per_sh) - 1) >> P.per_sh;
    P.units = (mass ? 3 : 2) * n_seq * c.Hkv;
    const unsigned grid = (unsigned) ((P.units + 7) / 8 * 8 * P.slices);
    if (W == 16) move_k<16><<<grid, MTHR, 0, s>>>(P);
    else if (W == 8) move_k<8><<<grid, MTHR, 0, s>>>(P);
    else if (W == 4) move_k<4><<<grid, MTHR, 0, s>>>(P);
    else move_k<2><<<grid, MTHR, 0, s>>>(P);
    return launched();
}

}   // namespace p1a
