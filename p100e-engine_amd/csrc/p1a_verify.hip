// Which drafted tokens stand, and the token behind them (p1a_tree_verify).
//
// The decision at a node needs its row's distribution at the children's tokens and, after a rejection, the sum of what is left over the whole vocabulary. With
// left = max(p - a q, 0) throughout (a: the sum of mass / (1 - gone) over the rejections so far) a rejection only moves the number a, and a node's
// outcome does not depend on how the walk came there: all nodes decide at once, in as many rounds as a node has children, and the walk follows what they decided.
//   stats_k   logits: every row in stretches of 4096 values, a workgroup each: the largest, where it is, the sum of exp((l - largest) / temp)
//   decide_k  a workgroup per sequence: every node tests its first child (without a draft: all of them, as a rejection takes one known weight out); the walk
//   sums_k    a launch for each further child of a node: nodes that the walk may still reach take the last round's sum, test a child, and sum what a rejection leaves
//   left_k    the last node's row: what is left, a stretch a workgroup
//   pick_k    a workgroup per sequence: the stretch where the running sum passes u, and the value in it (logits without a draft: at decide_k's end, as
//             stats_k has summed every stretch and only those with a rejected token are summed again)
// stats_k and left_k are bound by the memory that they read (160 rows of 151936 f32 logits: 23 us, 4.2 TB/s; what is left in 32 of them and the draft's: 11 us, 3.6 TB/s), the
// others by chains of dependent loads (decide_k 8 us, a round of sums_k 6, pick_k 6 ... 8): what does not depend on one another is asked for at once.
// A kernel's end is what makes its sums known: with workgroups that count themselves and a last one that goes on, each had to make its writes visible to the other
// XCDs' caches, and 32 chains over 151936 logits took 112 us instead of 48.
// Sums, exponentials and comparisons are made in 64 bits: with 32 one draw in some hundreds would take the neighbouring token. 2^x comes from a table of 256 powers
// and three terms (2e-13 of the value: a draw in 10^7), 12 64-bit instructions a value; the table is a constant of the program, since making it in every workgroup
// took 5 us of each kernel. A sum's order is fixed by its place, so the same call gives the same tokens.
#include "p1a_tiles.hpp"

#include <algorithm>

namespace p1a {
namespace {

constexpr int VTHR = 256, PER = 16, STRETCH = VTHR * PER;     // values of a thread, of a workgroup
constexpr int NODES = P1A_TREE_NODES;

// A node that waits for its sum, all in one place: what a round asks for first
struct alignas(16) pending {
    double a, gone;
    int node, child, state, token;                            // the child under test, its token and its number
    float u;
    int next, unused[2];                                      // the child behind it (-1: none)
};

struct verify_params {
    const char * target, * draft;
    size_t ld_target, ld_draft;                               // in values
    const int32_t * token, * parent;
    const float * temp, * u, * u_next;
    int32_t * n_accept, * path, * next;
    rows_view R;
    int V, stretches, ld_path, max_children;
    int target_bf16, draft_bf16, logits, distinct;
    // scratch
    double * st_sum;       // [T][stretches] sum of a stretch, relative to its largest
    float * st_max;        // [T][stretches]
    int * st_arg;          // [T][stretches]
    double * row_z;        // [T] logits: 1 / the row's sum
    float * row_max;       // [T] the row's largest
    int * row_arg;         // [T] where it is
    double * node_a;       // [T]
    int * node_state;      // [T] accepted child, NONE, or WAITS for its sum
    pending * wait[2];     // [T] a sequence's nodes that wait, from its first row on: two of them (a round reads one and writes the other)
    double * sums[2];      // [T][stretches] of a round; sums[0] then [n_seq][stretches] of the last row
    int16_t * sibling;     // [T] next child of the same parent
    int * n_waiting;       // [n_seq]
    int * last_row;        // [n_seq] the row that the token is drawn from (-1: none)
    double * last_a;       // [n_seq]
};
enum { NONE = -1, WAITS = -2 };

// ---- 2^x for x <= 0 ----
// 2^x = 2^n 2^(k / 256) 2^f: a power from a table in LDS, and 1 + f ln 2 + ... for |f| <= 1 / 512 - up to the third power 1.4e-13 of the value
struct powers { double of[256]; };
constexpr powers powers_of_2() {                              // 2^(k / 256) = exp(k ln 2 / 256), 18 terms of the series in Horner's form
    powers t{};
    for (int k = 0; k < 256; ++k) {
        const double f = k * (0.6931471805599453094 / 256);
        double p = 1.0;
        for (int i = 18; i >= 1; --i) p = 1.0 + f / i * p;
        t.of[k] = p;
    }
    return t;
}
__device__ const powers POWERS = powers_of_2();
__device__ __forceinline__ void fill(powers & t) {
    t.of[threadIdx.x] = POWERS.of[threadIdx.x];
    __syncthreads();
}
// (x: 256 times the exponent. A NaN: 0)
__device__ __forceinline__ double exp2_256(double x, const powers & t) {
    x = fmax(x, -281600.0);                                   // (below 2^-1074: 0)
    const double n = __builtin_rint(x), f = x - n;
    const int k = (int) n;
    constexpr double L = 0.6931471805599453094 / 256;
    return ldexp(t.of[k & 255] * fma(fma(fma(f, L * L * L / 6, L * L / 2), f, L), f, 1.0), k >> 8);
}
constexpr double LOG2E_256 = 256 * 1.4426950408889634074;

__device__ __forceinline__ double probability(float q) { return q > 0.f ? (double) q : 0.0; }   // (a NaN: 0)
// What logits weigh beside the largest of them, `most`, times z: by = 256 log2 e / temp (below 0: the one at `arg`, with certainty)
struct softmax {
    double by, z;
    float most;
    int arg;
    __device__ __forceinline__ softmax(double by_, float most_, int arg_, double z_) : by(by_), z(z_), most(most_), arg(arg_) {}
    // (what is decided once for a row stands outside of its values: f(how) with how(l, j) the weight of value j, l)
    template <class F> __device__ __forceinline__ void with(const powers & t, F && f) const {
        const float m = most;
        const double b = by, c = most, s = z;
        const int g = arg;
        if (by < 0.0) f([=](float, int j) { return j == g ? 1.0 : 0.0; });
        else if (m == MINUS_INF) f([](float, int) { return 0.0; });
        else if (m == -MINUS_INF) f([=](float l, int) { return l == m ? s : 0.0; });   // (infinite ones share everything)
        else f([=, &t](float l, int) { return exp2_256(((double) l - c) * b, t) * s; });   // (the difference first: a product with a small temperature rounds by whole powers)
    }
};
// 256 log2 e / temp of a sequence's logits; below 0: the largest one, with certainty
__device__ __forceinline__ double by_of(const verify_params & P, int seq) {
    if (!P.temp) return LOG2E_256;
    const float t = P.temp[seq];
    return t > 0.f ? LOG2E_256 / (double) t : -1.0;
}
__device__ __forceinline__ float value_at(const char * p, size_t i, bool bf16) {
    typedef const __attribute__((address_space(1))) uint16_t * g16;
    typedef const __attribute__((address_space(1))) float * g32;
    return bf16 ? __builtin_bit_cast(float, (uint32_t) ((g16) p)[i] << 16) : ((g32) p)[i];
}
// a thread's 16 values of the stretch from j0 on: value e is number place(e) of the row
struct places {
    int j0, tid;
    bool bf16;
    __device__ __forceinline__ int of(int e) const { return bf16 ? j0 + (e >> 3) * (VTHR * 8) + tid * 8 + (e & 7) : j0 + (e >> 2) * (VTHR * 4) + tid * 4 + (e & 3); }
};
// (Both types leave the values in the order of `at`, that of the target's type; `none` behind the row's end. A type is asked for once, not for each value.)
template <class At> __device__ __forceinline__ void load_each(float (&x)[PER], const char * row, bool bf16, At && at, int V, float none) {
    auto all = [&](auto type) {
#pragma unroll
        for (int e = 0; e < PER; ++e) x[e] = value_at(row, min(at(e), V - 1), type.value);
    };
    if (bf16) all(std::true_type{});
    else all(std::false_type{});
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] = at(e) < V ? x[e] : none;
}
template <int N> __device__ __forceinline__ void load_words(float * x, gbytes p, std::true_type) {      // N values of bf16, 8 a load
#pragma unroll
    for (int k = 0; k < N / 8; ++k) {
        const u4 w = gload<u4_a2>(p + 16 * k);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[8 * k + e] = __builtin_bit_cast(float, e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    }
}
template <int N> __device__ __forceinline__ void load_words(float * x, gbytes p, std::false_type) {     // of f32, 4 a load
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
        const u4 w = gload<u4_a4>(p + 16 * k);
#pragma unroll
        for (int e = 0; e < 4; ++e) { const uint32_t v = w[e]; x[4 * k + e] = __builtin_bit_cast(float, v); }   // (of an element itself the compiler casts the first)
    }
}
__device__ __forceinline__ void load16(float (&x)[PER], const char * row, bool bf16, const places & at, int V, float none) {
    if (at.j0 + STRETCH > V || bf16 != at.bf16) load_each(x, row, bf16, [&](int e) { return at.of(e); }, V, none);
    else if (bf16) {
#pragma unroll
        for (int k = 0; k < 2; ++k) load_words<8>(x + 8 * k, (gbytes) row + 2 * (size_t) at.of(8 * k), std::true_type{});
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) load_words<4>(x + 4 * k, (gbytes) row + 4 * (size_t) at.of(4 * k), std::false_type{});
    }
}
// the same of values j0 .. on end
__device__ __forceinline__ void load_run(float (&x)[PER], const char * row, bool bf16, int j0, int V, float none) {
    if (j0 + PER > V) load_each(x, row, bf16, [&](int e) { return j0 + e; }, V, none);
    else if (bf16) load_words<PER>(x, (gbytes) row + 2 * (size_t) j0, std::true_type{});
    else load_words<PER>(x, (gbytes) row + 4 * (size_t) j0, std::false_type{});
}

// sums over the lanes up to this one, over the wave and over the workgroup (those the same in every thread). Lanes are moved by vector instructions: through LDS the
// six steps of a sum took half a microsecond
template <int CTRL, int ROWS> __device__ __forceinline__ double moved(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t l = __builtin_amdgcn_update_dpp(0, (int) (uint32_t) u, CTRL, ROWS, 0xf, false), h = __builtin_amdgcn_update_dpp(0, (int) (u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t) h << 32 | l);
}
__device__ __forceinline__ double sum_up_to(double x) {
    x += moved<0x111, 0xf>(x);                                // lanes 1, 2, 4, 8 below, of the row of 16
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);                                // the row before's last, for rows 1 and 3
    x += moved<0x143, 0xc>(x);                                // lane 31, for rows 2 and 3
    return x;
}
__device__ __forceinline__ double wave_sum(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, sum_up_to(x));
    const uint32_t l = __builtin_amdgcn_readlane((int) (uint32_t) u, 63), h = __builtin_amdgcn_readlane((int) (u >> 32), 63);
    return __builtin_bit_cast(double, (uint64_t) h << 32 | l);
}
__device__ __forceinline__ double group_sum(double x, double * lds) {
    x = wave_sum(x);
    __syncthreads();
    if (!(threadIdx.x & 63)) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// the sequence that has row t, or -1. Every lane of the wave calls
__device__ __forceinline__ int seq_of_row(const rows_view & R, int t) {
    if (!R.row0) return R.per && t / R.per < R.n_seq && t % R.per < R.max_rows ? t / R.per : -1;
    for (int s0 = 0; s0 < R.n_seq; s0 += 64) {
        const int s = s0 + (int) (threadIdx.x & 63);
        bool has = false;
        if (s < R.n_seq) {
            const seq_view v = seq_of(R, s);
            has = t >= v.first && t < v.first + min(v.count, NODES);
        }
        const unsigned long long b = __ballot(has);
        if (b) return s0 + __builtin_ctzll(b);
    }
    return -1;
}

__global__ void __launch_bounds__(VTHR) stats_k(const verify_params P) {
    __shared__ float wm[VTHR / 64];
    __shared__ int wi[VTHR / 64];
    __shared__ double ws[VTHR / 64];
    __shared__ powers pw;
    const int t = blockIdx.x / P.stretches, z = blockIdx.x - t * P.stretches, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float x[PER];
    const places at{z * STRETCH, tid, P.target_bf16 != 0};
    load16(x, P.target + (size_t) t * P.ld_target * (P.target_bf16 ? 2 : 4), P.target_bf16, at, P.V, MINUS_INF);
    const int seq = seq_of_row(P.R, t);
    if (seq < 0) return;
    const double by = by_of(P, seq);
    fill(pw);
    float m = MINUS_INF;
#pragma unroll
    for (int e = 0; e < PER; ++e) m = fmaxf(m, x[e]);         // (NaN: not looked at)
    m = wave_max(m);
    int arg = INT32_MAX;
    if (by < 0.0) {                                           // the lowest place of the largest
#pragma unroll
        for (int e = PER - 1; e >= 0; --e) arg = x[e] == m ? at.of(e) : arg;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) arg = min(arg, __shfl_xor(arg, d));
    }
    if (lane == 0) { wm[wave] = m; wi[wave] = arg; }
    __syncthreads();
    m = wm[0]; arg = wi[0];
#pragma unroll
    for (int w = 1; w < VTHR / 64; ++w) {
        arg = wm[w] > m ? wi[w] : wm[w] == m ? min(arg, wi[w]) : arg;
        m = fmaxf(m, wm[w]);
    }
    double s = 0.0;
    if (by >= 0.0) {
        softmax(by, m, 0, 1.0).with(pw, [&](auto weight) {
#pragma unroll
            for (int e = 0; e < PER; ++e) s += weight(x[e], 0);
        });
        s = group_sum(s, ws);
    }
    if (tid == 0) {
        const size_t i = (size_t) t * P.stretches + z;
        P.st_sum[i] = s;
        P.st_max[i] = m;
        P.st_arg[i] = arg;
    }
}

// ---- what a workgroup knows about its sequence while it decides ----
struct tree_lds {
    int16_t up[NODES];                                        // parent, of nodes whose token there is
    int first[NODES];                                         // first child (none: NODES); then the child under test
    int sibling[NODES], token[NODES];                         // next child of the same parent
    int state[NODES];
    bool again[NODES];                                        // an elder sibling has the same token
    float value[NODES], q[NODES], u[NODES];                   // what the parent's rows hold of the token; its number
    float most[NODES];                                        // of the nodes' rows: the largest logit, where it is, 1 / the sum
    int arg[NODES];
    double z[NODES], gone[NODES];
    int waiting, length;
};

// A rejection of the child with the draft's probability q, of `mass`: what a and gone become. False: nothing is left to test another child with
__device__ __forceinline__ bool reject(const verify_params & P, double mass, double q, double & a, double & gone) {
    const double rest = 1.0 - gone;
    if (!(rest > 0.0)) return false;
    a += mass / rest;
    if (P.distinct) gone += q;
    return mass > 0.0 && 1.0 - gone > 0.0;                    // (no mass: nothing changes from here on and nobody is accepted; nothing to draw from: passed over)
}
__device__ __forceinline__ bool accept(double u, double mass, double p, double q, double a, double gone) { return u * (q / (1.0 - gone)) * mass < fmax(p - a * q, 0.0); }

// What one kernel reads of another's nodes stays in the call's rows even where two sequences of row0 share some, and each leaves its own there
__device__ __forceinline__ int row_in(const verify_params & P, int row) { return min(max(row, 0), P.R.T - 1); }

// f(weight) for a row: weight(l, j) of its value j, l
template <class F> __device__ __forceinline__ void with_row(const verify_params & P, int seq, int row, const powers & pw, F && f) {
    if (!P.logits) f([](float l, int) { return probability(l); });
    else softmax(by_of(P, seq), P.row_max[row], P.row_arg[row], P.row_z[row]).with(pw, f);
}

// ---- the last row of a sequence ----
struct last_lds {
    double ws[VTHR / 64], scan[VTHR];
    uint32_t out[STRETCH / 32];                               // values of a stretch that are taken out
    uint32_t touched[256 / 32];                               // stretches that have some
    int first[VTHR / 64], last[VTHR / 64];
};
// without a draft every child of the last node was rejected: f(token) for each
template <class F> __device__ __forceinline__ void rejected(const verify_params & P, const seq_view & v, int me, F && f) {
    if (P.draft) return;
    for (int i = me + 1 + (int) threadIdx.x; i < min(v.count, NODES); i += VTHR) {
        const int x = P.token[v.first + i];
        if (x >= 0 && x < P.V && (P.parent ? P.parent[v.first + i] : i - 1) == me) f(x);
    }
}
__device__ __forceinline__ void take_out(const verify_params & P, const seq_view & v, int me, int j0, last_lds & T) {
    for (int i = threadIdx.x; i < STRETCH / 32; i += VTHR) T.out[i] = 0;
    __syncthreads();
    rejected(P, v, me, [&](int x) { if (x >= j0 && x < j0 + STRETCH) atomicOr(&T.out[(x - j0) >> 5], 1u << ((x - j0) & 31)); });
    __syncthreads();
}
// what is left of a stretch (some), or all of it
__device__ __forceinline__ double sum_of(const verify_params & P, int seq, const seq_view & v, int t, double a, int z, bool some, const powers & pw, last_lds & T) {
    float x[PER], y[PER];
    const places at{z * STRETCH, (int) threadIdx.x, P.target_bf16 != 0};
    const bool draft = some && P.draft && a > 0.0;
    load16(x, P.target + (size_t) t * P.ld_target * (P.target_bf16 ? 2 : 4), P.target_bf16, at, P.V, MINUS_INF);
    if (draft) load16(y, P.draft + (size_t) t * P.ld_draft * (P.draft_bf16 ? 2 : 4), P.draft_bf16, at, P.V, 0.f);
    if (some && !P.draft) take_out(P, v, t - v.first, z * STRETCH, T);
    double s = 0.0;
    with_row(P, seq, t, pw, [&](auto weight) {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int j = at.of(e), i = j - z * STRETCH;
            const double p = weight(x[e], j);
            s += draft ? fmax(p - a * probability(y[e]), 0.0) : some && !P.draft && (T.out[i >> 5] >> (i & 31) & 1) ? 0.0 : p;
        }
    });
    return group_sum(s, T.ws);
}

__global__ void __launch_bounds__(VTHR) left_k(const verify_params P) {
    __shared__ powers pw;
    __shared__ last_lds T;
    const int seq = blockIdx.x / P.stretches, z = blockIdx.x - seq * P.stretches;
    const int t = P.last_row[seq];
    if (t < 0) return;
    if (P.logits) fill(pw);
    const double s = sum_of(P, seq, seq_of<true>(P.R, seq), t, P.last_a[seq], z, true, pw, T);
    if (threadIdx.x == 0) P.sums[0][(size_t) seq * P.stretches + z] = s;
}

// The token behind the last node's row t, with the number u. known: `mine` is the sum of stretch number tid; otherwise (logits, no draft) they are in st_sum, but for those that
// something is taken out of
__device__ __forceinline__ void pick(const verify_params & P, int seq, const seq_view & v, int t, double a, bool known, double mine, double u, const powers & pw, last_lds & T) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // ---- the stretch: one a thread (there are 256 at most) ----
    if (!known) {
        const double by = by_of(P, seq);
        const size_t at = (size_t) t * P.stretches;
        if (tid < P.stretches) {
            if (by < 0.0) mine = P.row_arg[t] >= 0 && P.row_arg[t] / STRETCH == tid ? 1.0 : 0.0;
            else softmax(by, P.row_max[t], 0, P.row_z[t]).with(pw, [&](auto weight) { mine = P.st_sum[at + tid] * weight(P.st_max[at + tid], 0); });
        }
        if (tid < 256 / 32) T.touched[tid] = 0;
        __syncthreads();
        rejected(P, v, t - v.first, [&](int x) { atomicOr(&T.touched[(x / STRETCH) >> 5], 1u << (x / STRETCH & 31)); });
        __syncthreads();
        for (int w = 0; w < 256 / 32; ++w)
            for (uint32_t bits = T.touched[w]; bits; bits &= bits - 1) {
                const int z = 32 * w + __builtin_ctz(bits);
                const double s = sum_of(P, seq, v, t, a, z, true, pw, T);
                if (tid == z) mine = s;
            }
    }
    bool some = group_sum(mine, T.ws) > 0.0;
    if (!some)                                                // nothing left: from p
        for (int z = 0; z < P.stretches; ++z) {
            const double s = sum_of(P, seq, v, t, a, z, false, pw, T);
            if (tid == z) mine = s;
        }
    auto running = [&](double x) {                            // sums over the threads up to this one
        __syncthreads();
        x = sum_up_to(x);
        if (lane == 63) T.ws[wave] = x;
        __syncthreads();
        for (int w = 0; w < wave; ++w) x += T.ws[w];
        return x;
    };
    const double upto = running(mine);
    T.scan[tid] = upto;
    __syncthreads();
    const double total = T.scan[VTHR - 1], goal = u * total;
    if (!(total > 0.0)) {
        if (tid == 0) P.next[seq] = -1;
        return;
    }
    // the lowest thread that has passed the goal with `a`, or, if none has, the last one that has `b` at all (all of 256 threads on one address in LDS took 3 us)
    auto first_or_last = [&](bool pass, int a, int b) {
        const unsigned long long ps = __ballot(pass), as = __ballot(b >= 0);
        const int f = __builtin_amdgcn_readlane(a, ps ? __builtin_ctzll(ps) : 0), z = __builtin_amdgcn_readlane(b, as ? 63 - __builtin_clzll(as) : 0);
        if (lane == 0) { T.first[wave] = ps ? f : -1; T.last[wave] = as ? z : -1; }
        __syncthreads();
        int r = -1;
#pragma unroll
        for (int w = 0; w < VTHR / 64; ++w) r = r < 0 ? T.first[w] : r;
#pragma unroll
        for (int w = VTHR / 64 - 1; w >= 0; --w) r = r < 0 ? T.last[w] : r;
        return r;
    };
    const int zf = first_or_last(mine > 0.0 && upto > goal, tid, mine > 0.0 ? tid : -1);   // (u of 1 and above: the last that weighs anything)
    const double before = zf ? T.scan[zf - 1] : 0.0;
    // ---- the value: 16 on end a thread ----
    const bool draft = some && P.draft && a > 0.0;
    float x[PER], y[PER];
    load_run(x, P.target + (size_t) t * P.ld_target * (P.target_bf16 ? 2 : 4), P.target_bf16, zf * STRETCH + tid * PER, P.V, MINUS_INF);
    if (draft) load_run(y, P.draft + (size_t) t * P.ld_draft * (P.draft_bf16 ? 2 : 4), P.draft_bf16, zf * STRETCH + tid * PER, P.V, 0.f);
    take_out(P, v, t - v.first, zf * STRETCH, T);
    double p[PER], sum = 0.0;
    with_row(P, seq, t, pw, [&](auto weight) {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int i = tid * PER + e;
            p[e] = weight(x[e], zf * STRETCH + i);
            if (draft) p[e] = fmax(p[e] - a * probability(y[e]), 0.0);
            else if (some && (T.out[i >> 5] >> (i & 31) & 1)) p[e] = 0.0;
            sum += p[e];
        }
    });
    double at = before + running(sum) - sum;
    int pass = -1, any = -1;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        at += p[e];
        if (p[e] > 0.0) {
            any = zf * STRETCH + tid * PER + e;
            if (at > goal && pass < 0) pass = any;
        }
    }
    const int token = first_or_last(pass >= 0, pass, any);    // (none has passed: the stretch's own sum was rounded above this one)
    if (tid == 0) P.next[seq] = token;
}
__global__ void __launch_bounds__(VTHR) pick_k(const verify_params P) {
    __shared__ powers pw;
    __shared__ last_lds T;
    const int seq = blockIdx.x, t = P.last_row[seq];
    // (asked for together with t)
    const double mine = (int) threadIdx.x < P.stretches ? P.sums[0][(size_t) seq * P.stretches + threadIdx.x] : 0.0, a = P.last_a[seq], u = (double) P.u_next[seq];
    if (t < 0) return;
    if (P.logits) fill(pw);
    pick(P, seq, seq_of<true>(P.R, seq), t, a, true, mine, u, pw, T);
}

// round: -1 at first; or the round whose sums are to be taken. walk: the path is known behind this one; and_pick: and so are the sums of all rows
__global__ void __launch_bounds__(VTHR) decide_k(const verify_params P, int round, bool walk, bool and_pick) {
    __shared__ tree_lds T;
    __shared__ last_lds U;
    __shared__ powers pw;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const seq_view v = seq_of<true>(P.R, seq);
    const int n = min(v.count, NODES);
    const double u_next = and_pick ? (double) P.u_next[seq] : 0.0;
    if (n < 1) {
        if (tid == 0) { P.n_accept[seq] = 0; P.next[seq] = -1; P.last_row[seq] = -1; P.n_waiting[seq] = 0; }
        for (int k = tid; k < P.ld_path; k += VTHR) P.path[(size_t) seq * P.ld_path + k] = -1;
        return;
    }
    if (P.logits) fill(pw);
    if (round < 0) {
        const double by = P.logits ? by_of(P, seq) : 0.0;
        for (int i = tid; i < n; i += VTHR) {
            const int x = P.token[v.first + i], p = P.parent ? P.parent[v.first + i] : i - 1;
            const bool is = i > 0 && p >= 0 && p < i && x >= 0 && x < P.V;
            T.token[i] = x;
            T.up[i] = (int16_t) (is ? p : -1);
            T.first[i] = NODES;
            T.sibling[i] = -1;
            T.again[i] = false;
            T.u[i] = P.u[v.first + i];
            if (is) {
                T.value[i] = value_at(P.target, (size_t) (v.first + p) * P.ld_target + x, P.target_bf16);
                if (P.draft) T.q[i] = value_at(P.draft, (size_t) (v.first + p) * P.ld_draft + x, P.draft_bf16);
            }
        }
        if (tid == 0) T.waiting = 0;
        // ---- logits: a wave a row: the sum of its stretches ----
        if (P.logits)
            for (int i = wave; i < n; i += VTHR / 64) {
                const size_t at = (size_t) (v.first + i) * P.stretches;
                float m = MINUS_INF;
                for (int z = lane; z < P.stretches; z += 64) m = fmaxf(m, P.st_max[at + z]);
                m = wave_max(m);
                int arg = INT32_MAX;
                double s = 0.0;
                if (by < 0.0) {
                    for (int z = lane; z < P.stretches; z += 64) arg = P.st_max[at + z] == m ? min(arg, P.st_arg[at + z]) : arg;
#pragma unroll
                    for (int d = 1; d < 64; d <<= 1) arg = min(arg, __shfl_xor(arg, d));
                } else if (m > MINUS_INF) {
                    softmax(by, m, 0, 1.0).with(pw, [&](auto weight) {
                        for (int z = lane; z < P.stretches; z += 64) s += P.st_sum[at + z] * weight(P.st_max[at + z], 0);
                    });
                    s = wave_sum(s);
                }
                if (lane == 0) {
                    T.most[i] = P.row_max[v.first + i] = m;
                    T.arg[i] = P.row_arg[v.first + i] = m > MINUS_INF ? arg : -1;
                    T.z[i] = P.row_z[v.first + i] = s > 0.0 ? 1.0 / s : 0.0;
                }
            }
        __syncthreads();
        // ---- children of a node in their order: each looks for the nearest elder one, but for the first ----
        if (P.parent) {
            for (int i = tid; i < n; i += VTHR) if (T.up[i] >= 0) atomicMin(&T.first[T.up[i]], i);
            __syncthreads();
            for (int i = tid; i < n; i += VTHR) {
                const int p = T.up[i];
                if (p < 0 || T.first[p] == i) continue;
                int j = i - 1;
                while (T.up[j] != p) --j;
                T.sibling[j] = i;
            }
            __syncthreads();
            if (!P.draft) {
                for (int i = tid; i < n; i += VTHR)
                    if (T.up[i] >= 0) for (int j = T.first[T.up[i]]; j != i && !T.again[i]; j = T.sibling[j]) T.again[i] = T.token[j] == T.token[i];
            } else
                for (int i = tid; i < n; i += VTHR) {         // (what no round is left for is not looked at: the list ends)
                    int j = T.first[i];
                    for (int k = 1; k < P.max_children && j >= 0 && j < NODES; ++k) j = T.sibling[j];
                    if (j >= 0 && j < NODES) T.sibling[j] = -1;
                }
            __syncthreads();
        } else
            for (int i = tid; i < n; i += VTHR) T.first[i] = i + 1 < n && T.up[i + 1] == i ? i + 1 : NODES;
        for (int i = tid; i < n; i += VTHR) P.sibling[v.first + i] = (int16_t) T.sibling[i];
        // ---- every node tests ----
        for (int i = tid; i < n; i += VTHR) {
            const int row = v.first + i;
            int c = T.first[i] < NODES ? T.first[i] : -1, state = NONE;
            double a = 0.0, gone = 0.0, mass = 1.0;
            while (c >= 0) {
                const double u = (double) T.u[c];
                double p = probability(T.value[c]);
                if (P.logits) softmax(by, T.most[i], T.arg[i], T.z[i]).with(pw, [&](auto weight) { p = weight(T.value[c], T.token[c]); });
                if (P.draft) {
                    const double q = probability(T.q[c]);
                    if (accept(u, 1.0, p, q, 0.0, 0.0)) { state = c; break; }
                    c = T.sibling[c];
                    if (reject(P, 1.0, q, a, gone) && c >= 0) state = WAITS;
                    break;
                }
                const double left = T.again[c] ? 0.0 : p;     // (a token that was taken out already)
                if (u * mass < left) { state = c; break; }
                mass -= left;
                c = T.sibling[c];
            }
            T.state[i] = state;
            P.node_a[row] = a;
            P.node_state[row] = state;
            T.gone[i] = gone;
            T.first[i] = c;
        }
        __syncthreads();
        // ---- nodes that wait and can still be reached: every one above lets the walk through, or waits itself and has not tested the child yet ----
        for (int i = tid; i < n; i += VTHR) {
            if (T.state[i] != WAITS) continue;
            bool reach = true;
            int j = i;
            for (int p = T.up[j]; p >= 0 && reach; j = p, p = T.up[j]) {
                const int sp = T.state[p];
                reach = sp == j || (sp == WAITS && j >= T.first[p]);
            }
            if (reach && j == 0) {                            // (in any order: each has its own sums; a behind one rejection is 1)
                const int c = T.first[i];
                P.wait[0][v.first + atomicAdd(&T.waiting, 1)] = pending{1.0, T.gone[i], i, c, WAITS, T.token[c], T.u[c], T.sibling[c], {0, 0}};
            }
        }
        __syncthreads();
        if (tid == 0) P.n_waiting[seq] = T.waiting;
    } else {
        const int in = round & 1;
        for (int i = tid; i < n; i += VTHR) T.state[i] = P.node_state[v.first + i];
        __syncthreads();
        // ---- nodes that waited: a wave each, with the last round's sum ----
        const int m = P.n_waiting[seq];
        for (int w = wave; w < m; w += VTHR / 64) {
            const pending o = P.wait[in][row_in(P, v.first + w)];
            const int i = min(max(o.node, 0), n - 1), row = v.first + i;
            int state = o.state;
            double a = o.a;
            if (state == WAITS) {
                double mass = 0.0;
                for (int z = lane; z < P.stretches; z += 64) mass += P.sums[in][(size_t) row * P.stretches + z];
                const int x = min(max(o.token, 0), P.V - 1);
                const float l = value_at(P.target, (size_t) row * P.ld_target + x, P.target_bf16);
                const double q = probability(value_at(P.draft, (size_t) row * P.ld_draft + x, P.draft_bf16));
                mass = wave_sum(mass);
                double gone = o.gone, p = 0.0;
                with_row(P, seq, row, pw, [&](auto weight) { p = weight(l, x); });
                if (accept((double) o.u, mass, p, q, a, gone)) state = o.child;
                else {
                    reject(P, mass, q, a, gone);
                    state = NONE;
                }
            }
            if (lane == 0) {
                T.state[i] = state;
                P.node_a[row] = a;
            }
        }
        __threadfence_block();
        __syncthreads();
    }
    if (!walk) return;
    // ---- the walk ----
    if (tid == 0) {
        int at = 0, k = 0;
        for (int c = T.state[0]; c > at && c < n; c = T.state[at]) {
            if (k < P.ld_path) P.path[(size_t) seq * P.ld_path + k] = c;
            ++k;
            at = c;
        }
        P.n_accept[seq] = k;
        P.last_row[seq] = v.first + at;
        P.last_a[seq] = P.node_a[v.first + at];
        T.length = k;
        T.waiting = at;
    }
    __syncthreads();
    for (int k = T.length + tid; k < P.ld_path; k += VTHR) P.path[(size_t) seq * P.ld_path + k] = -1;
    if (and_pick) pick(P, seq, v, v.first + T.waiting, 0.0, false, 0.0, u_next, pw, U);
}

// Round k: a node that waits takes the sum of round k - 1 and tests its child with it (every workgroup of the node does, the first writes it down); if that is rejected and there is
// another one, the sum of what is left now. SLOTS nodes of a sequence at a time.
constexpr int SLOTS = 4;
__global__ void __launch_bounds__(VTHR) sums_k(const verify_params P, int k) {
    __shared__ double ws[VTHR / 64];
    __shared__ powers pw;
    const int z = blockIdx.x % P.stretches, b = blockIdx.x / P.stretches, slot = b % SLOTS, seq = b / SLOTS, tid = threadIdx.x, lane = tid & 63;
    const int m = P.n_waiting[seq];
    if (slot >= m) return;
    const int in = k & 1, first = seq_of<true>(P.R, seq).first;
    if (P.logits) fill(pw);
    for (int w = slot; w < m; w += SLOTS) {
        pending o = P.wait[in][row_in(P, first + w)];
        const int t = row_in(P, first + o.node);
        float x[PER], y[PER];
        const places at{z * STRETCH, tid, P.target_bf16 != 0};
        if (o.state == WAITS) {
            load16(x, P.target + (size_t) t * P.ld_target * (P.target_bf16 ? 2 : 4), P.target_bf16, at, P.V, MINUS_INF);
            load16(y, P.draft + (size_t) t * P.ld_draft * (P.draft_bf16 ? 2 : 4), P.draft_bf16, at, P.V, 0.f);
            if (k) {
                const int token = min(max(o.token, 0), P.V - 1), behind = row_in(P, first + o.next);
                const float l = value_at(P.target, (size_t) t * P.ld_target + token, P.target_bf16), u = P.u[behind];
                const double q = probability(value_at(P.draft, (size_t) t * P.ld_draft + token, P.draft_bf16));
                const int then = P.token[behind], next = P.sibling[behind];
                double mass = 0.0;                            // (every wave for itself, all alike)
                for (int i = lane; i < P.stretches; i += 64) mass += P.sums[in][(size_t) t * P.stretches + i];
                mass = wave_sum(mass);
                double p = 0.0;
                with_row(P, seq, t, pw, [&](auto weight) { p = weight(l, token); });
                if (accept((double) o.u, mass, p, q, o.a, o.gone)) o.state = o.child;
                else {
                    if (!reject(P, mass, q, o.a, o.gone) || o.next < 0) o.state = NONE;
                    o.child = o.next;
                    o.token = then;
                    o.u = u;
                    o.next = next;
                }
            }
        }
        if (z == 0 && tid == 0) P.wait[in ^ 1][row_in(P, first + w)] = o;
        if (o.state != WAITS) continue;
        const double a = o.a;
        double s = 0.0;
        with_row(P, seq, t, pw, [&](auto weight) {
#pragma unroll
            for (int e = 0; e < PER; ++e) s += fmax(weight(x[e], at.of(e)) - a * probability(y[e]), 0.0);
        });
        s = group_sum(s, ws);
        if (tid == 0) P.sums[in ^ 1][(size_t) t * P.stretches + z] = s;
    }
}

}   // namespace

verify_plan plan_verify(const rows_view & R, int V, bool logits, bool draft) {
    verify_plan pl{};
    pl.stretches = std::max((V + STRETCH - 1) / STRETCH, 1);
    const size_t T = R.T, S = R.n_seq, z = pl.stretches;
    size_t at = 0;
    auto put = [&](int i, size_t bytes) { pl.at[i] = at; at += (bytes + 255) & ~(size_t) 255; };
    put(0, logits ? T * z * 8 : 0);
    put(1, logits ? T * z * 4 : 0);
    put(2, logits ? T * z * 4 : 0);
    put(3, T * 8);
    put(4, T * 4);
    put(5, T * 4);
    put(6, T * 8);                                            // node_a, node_state
    put(7, T * 4);
    put(8, draft ? T * sizeof(pending) : 0);
    put(9, draft ? T * sizeof(pending) : 0);
    put(10, std::max(draft ? T : 0, S) * z * 8);              // sums
    put(11, draft ? T * z * 8 : 0);
    put(12, T * 2);
    put(13, S * 4);
    put(14, S * 4);
    put(15, S * 8);
    pl.bytes = at;
    return pl;
}

int launch_verify(const verify_args & a, hipStream_t s) {
    const verify_plan pl = plan_verify(a.R, a.V, a.logits, a.draft != nullptr);
    // rounds: children behind the first that a node may have
    const int rounds = a.draft ? std::max(std::min(a.parent ? a.max_children : 1, a.R.max_rows - 1) - 1, 0) : 0;
    const long long most = std::max(a.logits ? (long long) a.R.T * pl.stretches : 0, (long long) a.R.n_seq * pl.stretches * (rounds ? SLOTS : 1));
    if (most > MOST_GROUPS) { set_error("p1a_tree_verify: unsupported shape (T=%d n_seq=%d V=%d: %lld workgroups)", a.R.T, a.R.n_seq, a.V, most); return P1A_E_SHAPE; }
    char * at = (char *) a.scratch;
    if (!at || ((uintptr_t) at & 255) || a.scratch_bytes < pl.bytes) {
        float * big, * small;
        if (!split_scratch(s, kept_bytes(pl.bytes), kept_bytes(1), big, small)) return P1A_E_SCRATCH;
        at = (char *) big;
    }
    verify_params P;
    P.target = (const char *) a.target; P.draft = (const char *) a.draft; P.ld_target = a.ld_target; P.ld_draft = a.ld_draft;
    P.token = a.token; P.parent = a.parent; P.temp = a.logits ? a.temp : nullptr; P.u = a.u; P.u_next = a.u_next;
    P.n_accept = a.n_accept; P.path = a.path; P.next = a.next; P.R = a.R; P.V = a.V; P.stretches = pl.stretches; P.ld_path = a.ld_path;
    P.max_children = a.parent ? a.max_children : 1;
    P.target_bf16 = a.target_bf16; P.draft_bf16 = a.draft_bf16; P.logits = a.logits; P.distinct = a.distinct;
    P.st_sum = (double *) (at + pl.at[0]); P.st_max = (float *) (at + pl.at[1]); P.st_arg = (int *) (at + pl.at[2]);
    P.row_z = (double *) (at + pl.at[3]); P.row_max = (float *) (at + pl.at[4]); P.row_arg = (int *) (at + pl.at[5]);
    P.node_a = (double *) (at + pl.at[6]); P.node_state = (int *) (at + pl.at[7]);
    for (int i = 0; i < 2; ++i) { P.wait[i] = (pending *) (at + pl.at[8 + i]); P.sums[i] = (double *) (at + pl.at[10 + i]); }
    P.sibling = (int16_t *) (at + pl.at[12]); P.n_waiting = (int *) (at + pl.at[13]); P.last_row = (int *) (at + pl.at[14]); P.last_a = (double *) (at + pl.at[15]);
    if (a.logits && a.R.T) stats_k<<<(unsigned) a.R.T * (unsigned) pl.stretches, VTHR, 0, s>>>(P);
    const bool at_once = a.logits && !a.draft;                // (stats_k has summed every row, and a rejection takes one value out)
    decide_k<<<a.R.n_seq, VTHR, 0, s>>>(P, -1, rounds == 0, at_once);
    for (int k = 0; k < rounds; ++k) sums_k<<<(unsigned) a.R.n_seq * SLOTS * pl.stretches, VTHR, 0, s>>>(P, k);
    if (rounds) decide_k<<<a.R.n_seq, VTHR, 0, s>>>(P, rounds, true, false);
    if (a.R.T && !at_once) {
        left_k<<<(unsigned) a.R.n_seq * pl.stretches, VTHR, 0, s>>>(P);
        pick_k<<<a.R.n_seq, VTHR, 0, s>>>(P);
    }
    return launched();
}

}   // namespace p1a
