// Which drafted tokens stand, and the token behind them (p1a_tree_verify).
//
// The decision at a node needs its row's distribution at the children's tokens and, after a rejection, the sum of what is left over the whole vocabulary. With
// left = max(p - a q, 0) throughout (a: the sum of mass / (1 - gone) over the rejections so far) a rejection only moves the number a, and a node's
// outcome does not depend on how the walk came there: all nodes decide at once, in as many rounds as a node has children, and the walk follows what they decided.
//   stats_k   logits: every row in stretches of 4096 values, a workgroup each: the largest, where it is, the sum of exp((l - largest) / temp)
//   decide_k  a workgroup per sequence: every node tests its first child (without a draft: all of them, as a rejection takes one known weight out); the walk
//   sums_k    further children of nodes that the walk can still reach: the sum of max(p - a q, 0) a stretch; the last workgroup of a sequence decides on
//   pick_k    the last node's row: sums a stretch; the last workgroup of a sequence finds the stretch where the running sum passes u, and the value in it
// Sums, exponentials and comparisons are made in 64 bits: with 32 one draw in some hundreds would take the neighbouring token. exp2 is a Taylor polynomial (11
// terms on |x ln 2| <= 0.347: 7e-15 of the value), 19 64-bit instructions a value: 24 M logits 12 us on the vector units, 20 from memory - both at once.
// A sum's order is fixed by its place, so the same call gives the same tokens.
#include "p1a_tiles.hpp"

#include <algorithm>

namespace p1a {
namespace {

constexpr int VTHR = 256, PER = 16, STRETCH = VTHR * PER;     // values of a thread, of a workgroup
constexpr int NODES = P1A_TREE_NODES;

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
    double * node_a, * node_gone;                             // [T]
    int * node_child;      // [T] the child under test
    int * node_state;      // [T] accepted child, NONE, or WAITS for its sum
    double * sums;         // [T][stretches] of a round, then [n_seq][stretches][2] of the last row
    int * due, * here;     // [n_seq] workgroups that a round has for the sequence; that have come
    int * last_row;        // [n_seq] the row that the token is drawn from (-1: none)
    double * last_a;       // [n_seq]
};
enum { NONE = -1, WAITS = -2 };

// 2^x for x <= 0
__device__ __forceinline__ double exp2_64(double x) {
    x = fmax(x, -1100.0);                                     // (below 2^-1074: 0)
    const double n = __builtin_rint(x), f = (x - n) * 0.6931471805599453094;
    double p = 2.50521083854417188e-8;                        // 1 / 11!, 1 / 10! ...
    p = fma(p, f, 2.75573192239858907e-7);
    p = fma(p, f, 2.75573192239858907e-6);
    p = fma(p, f, 2.48015873015873016e-5);
    p = fma(p, f, 1.98412698412698413e-4);
    p = fma(p, f, 1.38888888888888889e-3);
    p = fma(p, f, 8.33333333333333333e-3);
    p = fma(p, f, 4.16666666666666667e-2);
    p = fma(p, f, 1.66666666666666667e-1);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, (int) n);
}
constexpr double LOG2E_64 = 1.4426950408889634074;

// weight of a logit beside the largest one: by = log2 e / temp
__device__ __forceinline__ double logit_weight(float l, float most, double by) {
    return l == most ? 1.0 : l > MINUS_INF ? exp2_64(((double) l - (double) most) * by) : 0.0;   // (a NaN: 0; finite beside an infinite one: 2^-inf)
}
// the scale of a sequence's logits; below 0: the largest one, with certainty
__device__ __forceinline__ double by_of(const verify_params & P, int seq) {
    if (!P.temp) return LOG2E_64;
    const float t = P.temp[seq];
    return t > 0.f ? LOG2E_64 / (double) t : -1.0;
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
// Both types leave the values in the order of `at` (that of the target's type)
__device__ __forceinline__ void load16(float (&x)[PER], const char * row, bool bf16, const places & at, int V, float none) {
    if (at.j0 + STRETCH <= V && bf16 == at.bf16) {
        if (bf16) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const u4 w = gload<u4_a2>((gbytes) row + 2 * (size_t) at.of(8 * k));
#pragma unroll
                for (int e = 0; e < 8; ++e) x[8 * k + e] = __builtin_bit_cast(float, e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u4 w = gload<u4_a4>((gbytes) row + 4 * (size_t) at.of(4 * k));
#pragma unroll
                for (int e = 0; e < 4; ++e) { const uint32_t v = w[e]; x[4 * k + e] = __builtin_bit_cast(float, v); }   // (of an element itself the compiler casts the first)
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int j = at.of(e);
        x[e] = j < V ? value_at(row, j, bf16) : none;
    }
}

// sums over the workgroup, the same in every thread (lanes by an xor butterfly, waves in order)
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    return x;
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
    const int t = blockIdx.x / P.stretches, z = blockIdx.x - t * P.stretches, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float x[PER];
    const places at{z * STRETCH, tid, P.target_bf16 != 0};
    load16(x, P.target + (size_t) t * P.ld_target * (P.target_bf16 ? 2 : 4), P.target_bf16, at, P.V, MINUS_INF);
    const int seq = seq_of_row(P.R, t);
    if (seq < 0) return;
    const double by = by_of(P, seq);
    float m = MINUS_INF;
    int arg = INT32_MAX;
#pragma unroll
    for (int e = 0; e < PER; ++e) if (x[e] > m) { m = x[e]; arg = at.of(e); }      // (a thread's places ascend)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float om = __shfl_xor(m, d);
        const int oi = __shfl_xor(arg, d);
        if (om > m || (om == m && oi < arg)) { m = om; arg = oi; }
    }
    if (lane == 0) { wm[wave] = m; wi[wave] = arg; }
    __syncthreads();
    m = wm[0]; arg = wi[0];
#pragma unroll
    for (int w = 1; w < VTHR / 64; ++w) if (wm[w] > m || (wm[w] == m && wi[w] < arg)) { m = wm[w]; arg = wi[w]; }
    double s = 0.0;
    if (by >= 0.0) {
#pragma unroll
        for (int e = 0; e < PER; ++e) s += logit_weight(x[e], m, by);
        s = group_sum(s, ws);
    }
    if (tid == 0) {
        const size_t i = (size_t) t * P.stretches + z;
        P.st_sum[i] = m > MINUS_INF ? s : 0.0;
        P.st_max[i] = m;
        P.st_arg[i] = arg;
    }
}

// ---- what a workgroup knows about its sequence while it decides ----
struct tree_lds {
    int16_t up[NODES], first[NODES], sibling[NODES];          // parent, first child, next child of the same parent: of nodes whose token there is
    int token[NODES];
    int state[NODES];
    bool again[NODES];                                        // an elder sibling has the same token
    int waiting;
};

// p at token x of a row
__device__ __forceinline__ double target_at(const verify_params & P, int seq, int row, int x) {
    const float l = value_at(P.target, (size_t) row * P.ld_target + x, P.target_bf16);
    if (!P.logits) return l > 0.f ? (double) l : 0.0;
    const double by = by_of(P, seq);
    if (by < 0.0) return x == P.row_arg[row] ? 1.0 : 0.0;
    const float most = P.row_max[row];
    return most > MINUS_INF ? logit_weight(l, most, by) * P.row_z[row] : 0.0;
}
__device__ __forceinline__ double draft_at(const verify_params & P, int row, int x) {
    const float q = value_at(P.draft, (size_t) row * P.ld_draft + x, P.draft_bf16);
    return q > 0.f ? (double) q : 0.0;
}

// One round for sequence `seq`: nodes that wait have their sums. All threads of the workgroup call.
__device__ void decide(const verify_params & P, int seq, bool begin, tree_lds & T) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const seq_view v = seq_of<true>(P.R, seq);
    const int n = min(v.count, NODES);
    if (n < 1) {
        if (tid == 0) { P.n_accept[seq] = 0; P.next[seq] = -1; P.last_row[seq] = -1; P.due[seq] = 0; P.here[seq] = 0; }
        for (int k = tid; k < P.ld_path; k += VTHR) P.path[(size_t) seq * P.ld_path + k] = -1;
        return;
    }
    for (int i = tid; i < n; i += VTHR) {
        const int x = P.token[v.first + i], p = P.parent ? P.parent[v.first + i] : i - 1;
        T.token[i] = x;
        T.up[i] = (int16_t) (i > 0 && p >= 0 && p < i && x >= 0 && x < P.V ? p : -1);
        T.first[i] = -1;
        T.state[i] = begin ? NONE : P.node_state[v.first + i];
    }
    if (tid == 0) T.waiting = 0;
    __syncthreads();
    // (a child's elder siblings: the nearest one's `sibling` it is; how many there are, against max_children)
    for (int i = tid; i < n; i += VTHR) {
        const int p = T.up[i];
        const int x = T.token[i];
        int elder = -1, k = 0;
        bool again = false;
        if (p >= 0)
            for (int j = p + 1; j < i; ++j) if (T.up[j] == p) { elder = j; ++k; again |= T.token[j] == x; }
        T.again[i] = again;
        if (p >= 0 && (!P.draft || k < P.max_children)) {
            if (elder < 0) T.first[p] = (int16_t) i;
            else T.sibling[elder] = (int16_t) i;
        }
        int younger = -1;                                     // (the last one, or the last that is looked at, has none)
        if (p >= 0 && (!P.draft || k + 1 < P.max_children))
            for (int j = i + 1; j < n; ++j) if (T.up[j] == p) { younger = j; break; }
        if (younger < 0) T.sibling[i] = -1;
    }
    __syncthreads();
    // ---- rows' sums (logits), or sums of what is left at nodes that wait: a wave a row ----
    for (int i = wave; i < n; i += VTHR / 64) {
        const int row = v.first + i;
        if (begin) {
            if (!P.logits) continue;
            const size_t at = (size_t) row * P.stretches;
            float m = MINUS_INF;
            int arg = INT32_MAX;
            for (int z = lane; z < P.stretches; z += 64) { const float x = P.st_max[at + z]; if (x > m) { m = x; arg = P.st_arg[at + z]; } }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const float om = __shfl_xor(m, d);
                const int oi = __shfl_xor(arg, d);
                if (om > m || (om == m && oi < arg)) { m = om; arg = oi; }
            }
            const double by = by_of(P, seq);
            double s = 0.0;
            if (by >= 0.0 && m > MINUS_INF)
                for (int z = lane; z < P.stretches; z += 64) s += P.st_sum[at + z] * logit_weight(P.st_max[at + z], m, by);
            s = wave_sum(s);
            if (lane == 0) {
                P.row_max[row] = m;
                P.row_arg[row] = m > MINUS_INF ? arg : -1;
                P.row_z[row] = s > 0.0 ? 1.0 / s : 0.0;
            }
        } else if (T.state[i] == WAITS) {
            double s = 0.0;
            for (int z = lane; z < P.stretches; z += 64) s += P.sums[(size_t) row * P.stretches + z];
            s = wave_sum(s);
            if (lane == 0) P.sums[(size_t) row * P.stretches] = s;
        }
    }
    __threadfence_block();
    __syncthreads();
    // ---- every node tests ----
    for (int i = tid; i < n; i += VTHR) {
        const int row = v.first + i;
        if (!begin && T.state[i] != WAITS) continue;
        int c = begin ? T.first[i] : P.node_child[row], state = NONE;
        double a = begin ? 0.0 : P.node_a[row], gone = begin ? 0.0 : P.node_gone[row], mass = begin ? 1.0 : P.sums[(size_t) row * P.stretches];
        while (c >= 0) {
            const int x = T.token[c];
            const double u = (double) P.u[v.first + c], p = target_at(P, seq, row, x);
            if (P.draft) {
                const double q = draft_at(P, row, x), rest = 1.0 - gone;
                const bool any = rest > 0.0;                  // (nothing left to draw from: passed over)
                if (any && u * (q / rest) * mass < fmax(p - a * q, 0.0)) { state = c; break; }
                c = T.sibling[c];
                if (!any) continue;
                a += mass / rest;
                if (P.distinct) gone += q;
                if (c < 0) break;
                if (mass > 0.0) { state = WAITS; break; }     // (mass 0: nothing changes from here on, nobody is accepted)
            } else {
                const double left = T.again[c] ? 0.0 : p;     // (a token that was taken out already)
                if (u * mass < left) { state = c; break; }
                mass -= left;
                c = T.sibling[c];
            }
        }
        T.state[i] = state;
        P.node_a[row] = a;
        P.node_gone[row] = gone;
        P.node_child[row] = c;
    }
    __syncthreads();
    // ---- nodes that wait and can still be reached: every one above lets the walk through, or waits itself and has not tested the child yet ----
    for (int i = tid; i < n; i += VTHR) {
        int state = T.state[i];
        if (state == WAITS) {
            bool reach = true;
            int j = i;
            for (int p = T.up[j]; p >= 0 && reach; j = p, p = T.up[j]) {
                const int sp = T.state[p];
                reach = sp == j || (sp == WAITS && j >= P.node_child[v.first + p]);
            }
            if (reach && j == 0) atomicAdd(&T.waiting, 1);
            else state = NONE;                                // (never asked again)
        }
        P.node_state[v.first + i] = state;
    }
    __syncthreads();
    const int waiting = T.waiting;
    __syncthreads();
    if (tid == 0) {
        P.due[seq] = waiting * P.stretches;
        P.here[seq] = 0;
    }
    // ---- the walk ----
    if (waiting == 0) {
        if (tid == 0) {
            int at = 0, k = 0;
            for (int c = T.state[0]; c >= 0; c = T.state[at]) {
                if (k < P.ld_path) P.path[(size_t) seq * P.ld_path + k] = c;
                ++k;
                at = c;
            }
            P.n_accept[seq] = k;
            P.last_row[seq] = v.first + at;
            P.last_a[seq] = P.node_a[v.first + at];
            T.waiting = k;
        }
        __syncthreads();
        for (int k = T.waiting + tid; k < P.ld_path; k += VTHR) P.path[(size_t) seq * P.ld_path + k] = -1;
    }
}

__global__ void __launch_bounds__(VTHR) decide_k(const verify_params P) {
    __shared__ tree_lds T;
    decide(P, blockIdx.x, true, T);
}

// what the values of a row weigh
struct row_of {
    bool logits, certain;
    float most;
    int arg;
    double by, z;
    __device__ __forceinline__ row_of(const verify_params & P, int seq, int row) {
        logits = P.logits;
        by = logits ? by_of(P, seq) : 0.0;
        certain = logits && by < 0.0;
        most = logits ? P.row_max[row] : 0.f;
        arg = logits ? P.row_arg[row] : -1;
        z = logits ? P.row_z[row] : 1.0;
    }
    __device__ __forceinline__ double weight(float l, int j) const {
        if (!logits) return l > 0.f ? (double) l : 0.0;
        if (certain) return j == arg ? 1.0 : 0.0;
        return most > MINUS_INF ? logit_weight(l, most, by) * z : 0.0;
    }
};

// true in the workgroup that comes last of `due` for the sequence; what the others wrote is there for it
__device__ __forceinline__ bool comes_last(int * here, int due, int * lds) {
    if (threadIdx.x == 0) {
        __threadfence();
        const int was = atomicAdd(here, 1);
        __threadfence();
        *lds = was == due - 1;
    }
    __syncthreads();
    return *lds != 0;
}

__global__ void __launch_bounds__(VTHR) sums_k(const verify_params P) {
    __shared__ tree_lds T;
    __shared__ double ws[VTHR / 64];
    __shared__ int last;
    const int t = blockIdx.x / P.stretches, z = blockIdx.x - t * P.stretches, tid = threadIdx.x;
    const int seq = seq_of_row(P.R, t);
    if (seq < 0 || P.node_state[t] != WAITS) return;
    const double a = P.node_a[t];
    const row_of row(P, seq, t);
    float x[PER], y[PER];
    const places at{z * STRETCH, tid, P.target_bf16 != 0};
    load16(x, P.target + (size_t) t * P.ld_target * (P.target_bf16 ? 2 : 4), P.target_bf16, at, P.V, MINUS_INF);
    load16(y, P.draft + (size_t) t * P.ld_draft * (P.draft_bf16 ? 2 : 4), P.draft_bf16, at, P.V, 0.f);
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < PER; ++e) s += fmax(row.weight(x[e], at.of(e)) - a * (y[e] > 0.f ? (double) y[e] : 0.0), 0.0);
    s = group_sum(s, ws);
    if (tid == 0) P.sums[(size_t) t * P.stretches + z] = s;
    if (comes_last(P.here + seq, P.due[seq], &last)) decide(P, seq, false, T);
}

__global__ void __launch_bounds__(VTHR) pick_k(const verify_params P) {
    __shared__ double ws[VTHR / 64];
    __shared__ double scan[VTHR];
    __shared__ uint32_t out[STRETCH / 32];                    // values of a stretch that are taken out
    __shared__ int last, found;
    const int seq = blockIdx.x / P.stretches, z = blockIdx.x - seq * P.stretches, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int t = P.last_row[seq];
    if (t < 0) return;
    const double a = P.last_a[seq];
    const seq_view v = seq_of<true>(P.R, seq);
    const int n = min(v.count, NODES), me = t - v.first;
    const row_of row(P, seq, t);
    const bool draft = P.draft && a > 0.0;
    // (without a draft every child of the last node was rejected)
    auto take_out = [&](int j0) {
        for (int i = tid; i < STRETCH / 32; i += VTHR) out[i] = 0;
        __syncthreads();
        if (!P.draft)
            for (int i = me + 1 + tid; i < n; i += VTHR) {
                const int x = P.token[v.first + i] - j0;
                if (x >= 0 && x < STRETCH && (P.parent ? P.parent[v.first + i] : i - 1) == me) atomicOr(&out[x >> 5], 1u << (x & 31));
            }
        __syncthreads();
    };
    take_out(z * STRETCH);
    const char * const tr = P.target + (size_t) t * P.ld_target * (P.target_bf16 ? 2 : 4), * const dr = P.draft + (size_t) t * P.ld_draft * (P.draft_bf16 ? 2 : 4);
    {
        float x[PER], y[PER];
        const places at{z * STRETCH, tid, P.target_bf16 != 0};
        load16(x, tr, P.target_bf16, at, P.V, MINUS_INF);
        if (draft) load16(y, dr, P.draft_bf16, at, P.V, 0.f);
        double left = 0.0, all = 0.0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int j = at.of(e), i = j - z * STRETCH;
            const double p = row.weight(x[e], j);
            all += p;
            left += draft ? fmax(p - a * (y[e] > 0.f ? (double) y[e] : 0.0), 0.0) : out[i >> 5] >> (i & 31) & 1 ? 0.0 : p;
        }
        left = group_sum(left, ws);
        all = group_sum(all, ws);
        if (tid == 0) {
            double * const to = P.sums + 2 * ((size_t) seq * P.stretches + z);
            to[0] = left;
            to[1] = all;
        }
    }
    if (!comes_last(P.here + seq, P.stretches, &last)) return;
    // ---- the stretch: one a thread (there are 256 at most) ----
    const double * const from = P.sums + 2 * (size_t) seq * P.stretches;
    const double mine = tid < P.stretches ? from[2 * tid] : 0.0, whole = tid < P.stretches ? from[2 * tid + 1] : 0.0;
    const bool some = group_sum(mine, ws) > 0.0;              // (nothing left: from p)
    auto running = [&](double x) {                            // sums over the threads up to this one
        __syncthreads();
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const double y = __shfl_up(x, d); if (lane >= d) x += y; }
        if (lane == 63) ws[wave] = x;
        __syncthreads();
        for (int w = 0; w < wave; ++w) x += ws[w];
        return x;
    };
    const double w = some ? mine : whole, upto = running(w);
    scan[tid] = upto;
    if (tid == 0) found = INT32_MAX;
    __syncthreads();
    const double total = scan[VTHR - 1];
    if (!(total > 0.0)) {
        if (tid == 0) P.next[seq] = -1;
        return;
    }
    const double goal = (double) P.u_next[seq] * total;
    if (upto > goal && w > 0.0) atomicMin(&found, tid);
    __syncthreads();
    if (found == INT32_MAX) {                                 // (u of 1 and above: the last that weighs anything)
        __syncthreads();
        if (tid == 0) found = -1;
        __syncthreads();
        if (w > 0.0) atomicMax(&found, tid);
        __syncthreads();
    }
    const int zf = found;
    const double before = zf ? scan[zf - 1] : 0.0;
    __syncthreads();
    take_out(zf * STRETCH);
    // ---- the value: 16 on end a thread ----
    double p[PER], sum = 0.0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int i = tid * PER + e, j = zf * STRETCH + i;
        p[e] = 0.0;
        if (j < P.V) {
            p[e] = row.weight(value_at(tr, j, P.target_bf16), j);
            if (some && draft) { const float q = value_at(dr, j, P.draft_bf16); p[e] = fmax(p[e] - a * (q > 0.f ? (double) q : 0.0), 0.0); }
            else if (some && (out[i >> 5] >> (i & 31) & 1)) p[e] = 0.0;
        }
        sum += p[e];
    }
    double at = before + running(sum) - sum;
    if (tid == 0) { found = INT32_MAX; last = -1; }
    __syncthreads();
    int pass = INT32_MAX, any = -1;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        at += p[e];
        if (p[e] > 0.0) {
            any = zf * STRETCH + tid * PER + e;
            if (at > goal) pass = min(pass, any);
        }
    }
    if (pass != INT32_MAX) atomicMin(&found, pass);
    if (any >= 0) atomicMax(&last, any);
    __syncthreads();
    if (tid == 0) P.next[seq] = found != INT32_MAX ? found : last;   // (the stretch's own sum rounded above this one: its last)
}

}   // namespace

verify_plan plan_verify(const rows_view & R, int V, bool logits) {
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
    put(6, T * 8);
    put(7, T * 8);
    put(8, T * 4);
    put(9, T * 4);
    put(10, std::max(T, 2 * S) * z * 8);
    put(11, S * 4);
    put(12, S * 4);
    put(13, S * 4);
    put(14, S * 8);
    pl.bytes = at;
    return pl;
}

int launch_verify(const verify_args & a, hipStream_t s) {
    const verify_plan pl = plan_verify(a.R, a.V, a.logits);
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
    P.node_a = (double *) (at + pl.at[6]); P.node_gone = (double *) (at + pl.at[7]); P.node_child = (int *) (at + pl.at[8]); P.node_state = (int *) (at + pl.at[9]);
    P.sums = (double *) (at + pl.at[10]); P.due = (int *) (at + pl.at[11]); P.here = (int *) (at + pl.at[12]); P.last_row = (int *) (at + pl.at[13]); P.last_a = (double *) (at + pl.at[14]);
    const unsigned rows = (unsigned) a.R.T * (unsigned) pl.stretches;
    if (a.logits && a.R.T) stats_k<<<rows, VTHR, 0, s>>>(P);
    decide_k<<<a.R.n_seq, VTHR, 0, s>>>(P);
    if (a.draft && a.R.T)
        for (int k = 1; k < std::min(P.max_children, a.R.max_rows - 1); ++k) sums_k<<<rows, VTHR, 0, s>>>(P);
    if (a.R.T) pick_k<<<(unsigned) a.R.n_seq * pl.stretches, VTHR, 0, s>>>(P);
    return launched();
}

}   // namespace p1a
