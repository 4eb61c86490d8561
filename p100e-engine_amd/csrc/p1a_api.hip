// extern "C" layer of the paged-KV attention library: argument validation (refusals launch nothing), split-K
// scratch ownership per (device, stream), split-count bookkeeping. All device work lives in the other .hip files.
#include "p1a_common.hpp"
#include "p1a_tiles.hpp"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

// Split scratch of the allocation-free decode entry point (p1a_attn_decode_noalloc): a fixed array in device memory,
// one copy per GPU, held until the process ends. In host code the array's NAME is only a handle: its device address is
// asked for once per device with hipGetSymbolAddress and only that address is ever handed to kernels.
static __device__ __align__(256) unsigned char scratch[P1A_NOALLOC_SCRATCH_BYTES];

namespace p1a {

static thread_local char g_err[256] = "";

void set_error(const char * fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    fprintf(stderr, "p1a_attn: %s\n", g_err);
}

namespace {

// Split partials per (device, stream): calls on different streams of one device may overlap. A captured graph holds the
// pointers it was recorded with, so a buffer is NEVER freed while the library lives: the decode buffers are allocated on
// the first call at the footprint of P1A_MAX_ROWS rows of that call's head shape (every KV type and row grouping), and
// in the rare case that a later call needs more (another head shape, a larger split count) the new buffer replaces the
// old one only for later calls - the old one stays allocated (g_retired) until p1a_release(). Nothing is allocated
// while the stream is being captured. The partials of a key-split prefill have a pair of their own.
struct bufpair { float * o = nullptr; float * ml = nullptr; size_t cap_o = 0, cap_ml = 0; };
struct stream_bufs { int dev = -1; hipStream_t s = nullptr; bufpair dec, pf; void * stage = nullptr; size_t cap_stage = 0; bool stage_captured = false; };
constexpr int MAX_SCR = 64;
constexpr int MAX_RETIRED = 1024;
stream_bufs g_scr[MAX_SCR];
int g_nscr = 0;
struct retired { int dev; void * p; };
retired g_retired[MAX_RETIRED];
int g_nretired = 0;
std::mutex g_mu;
int g_nsplit_override = 0;
int g_env_split = -1;   // P1A_DEC_SPLIT as last read (-1 = not read yet)
size_t g_stage_limit = (size_t) 1 << 30;   // largest f16 staging copy the library keeps per (device, stream); 0 = none
int g_cus[16] = {0};
constexpr int MAX_DEV = 64;
void * g_static_scratch[MAX_DEV] = {nullptr};   // device address of `scratch` on each device (nullptr = not asked for yet)

}   // namespace

// the device address of the static split scratch on the CURRENT device (resolved on the first call per device), or
// nullptr with the error set
void * static_scratch() {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEV) { set_error("p1a_attn_decode_noalloc: no current device"); return nullptr; }
    std::lock_guard<std::mutex> lk(g_mu);
    if (!g_static_scratch[dev]) {
        void * ptr = nullptr;
        const hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(::scratch));
        if (e != hipSuccess || !ptr) {
            (void) hipGetLastError();
            set_error("p1a_attn_decode_noalloc: hipGetSymbolAddress failed (%s)", hipGetErrorString(e));
            return nullptr;
        }
        g_static_scratch[dev] = ptr;
    }
    return g_static_scratch[dev];
}

int cu_count() {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 256;
    int & n = g_cus[dev & 15];
    if (!n && hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) n = 256;
    return n;
}

namespace {

enum which_buf { BUF_DECODE, BUF_PREFILL };

// the buffer pair `w` of (current device, s) with at least these capacities, or nullptr (error set unless quiet)
bufpair * scratch_for(hipStream_t s, which_buf w, size_t need_o, size_t need_ml, bool quiet = false) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return nullptr;
    std::lock_guard<std::mutex> lk(g_mu);
    stream_bufs * e = nullptr;
    for (int i = 0; i < g_nscr; ++i) if (g_scr[i].dev == dev && g_scr[i].s == s) e = &g_scr[i];
    if (!e) {
        if (g_nscr == MAX_SCR) { if (!quiet) set_error("too many (device, stream) pairs"); return nullptr; }
        e = &g_scr[g_nscr++];
        e->dev = dev; e->s = s;
    }
    bufpair & b = w == BUF_DECODE ? e->dec : e->pf;
    if (need_o > b.cap_o || need_ml > b.cap_ml) {
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        if (s && hipStreamIsCapturing(s, &st) == hipSuccess && st != hipStreamCaptureStatusNone) {
            if (!quiet) set_error("split scratch would have to be allocated during stream capture: call p1a_warmup%s first", w == BUF_PREFILL ? "_prefill" : "");
            return nullptr;
        }
        if (b.o && g_nretired + 2 > MAX_RETIRED) { if (!quiet) set_error("split scratch replaced too often"); return nullptr; }
        if (need_o < b.cap_o) need_o = b.cap_o;
        if (need_ml < b.cap_ml) need_ml = b.cap_ml;
        float * no = nullptr, * nm = nullptr;
        if (hipMalloc(&no, need_o) != hipSuccess || hipMalloc(&nm, need_ml) != hipSuccess) {
            (void) hipGetLastError();
            if (no) (void) hipFree(no);
            if (!quiet) set_error("split scratch allocation failed (%zu bytes)", need_o + need_ml);
            return nullptr;
        }
        // the replaced buffers stay allocated: a graph captured earlier on this stream may still write and read them
        if (b.o) { g_retired[g_nretired++] = retired{dev, b.o}; g_retired[g_nretired++] = retired{dev, b.ml}; }
        b.o = no; b.ml = nm; b.cap_o = need_o; b.cap_ml = need_ml;
    }
    return &b;
}

bool kv_ok(const p1a_kv * c, const char * who) {
    if (!c || !c->k || !c->v) { set_error("%s: null cache", who); return false; }
    if (c->type != P1A_KV_F16 && c->type != P1A_KV_Q8_0 && c->type != P1A_KV_Q4_0) { set_error("%s: unknown KV type %u", who, c->type); return false; }
    if (c->Hkv < 1 || c->D < 32 || c->D % 32 || c->D > 512) { set_error("%s: unsupported shape (Hkv=%d D=%d)", who, c->Hkv, c->D); return false; }
    if (c->pt && (c->psh < 0 || c->psh > 24 || c->pstride == 0)) { set_error("%s: bad page geometry (psh=%d pstride=%zu)", who, c->psh, c->pstride); return false; }
    return true;
}

// requested split-stream count: the setter, then the environment, else 0 = the plan's default for the device
int read_env_split() {
    const char * e = getenv("P1A_DEC_SPLIT");
    const int v = e && *e ? atoi(e) : 0;
    return v > 0 ? v : 0;
}
int nsplit_req() {
    if (g_env_split < 0) g_env_split = read_env_split();
    return g_nsplit_override > 0 ? g_nsplit_override : g_env_split;
}

// the decode split buffers of a head shape: P1A_MAX_ROWS rows, the largest need over the KV types and row groupings
void decode_footprint(int Hq, int Hkv, int D, size_t & need_o, size_t & need_ml) {
    // (two dozen plans, about 1 us: the last answer of a thread is kept with all that it depends on)
    struct memo { int Hq, Hkv, D, req, cus; size_t o, ml; };
    static thread_local memo last = {0, 0, 0, 0, 0, 0, 0};
    const int req = nsplit_req(), cus = cu_count();
    if (last.Hq == Hq && last.Hkv == Hkv && last.D == D && last.req == req && last.cus == cus) { need_o = last.o; need_ml = last.ml; return; }
    p1a_kv c;
    memset(&c, 0, sizeof c);
    c.Hkv = Hkv; c.D = D;
    need_o = need_ml = 0;
    const uint32_t types[3] = {P1A_KV_F16, P1A_KV_Q8_0, P1A_KV_Q4_0};
    // (a cache the MFMA kernel cannot take - a misaligned base, short pages - goes to the kernel for any shape, which has a plan of
    // its own: both count, so that a warm-up also covers such caches)
    for (uintptr_t base : {(uintptr_t) 16, (uintptr_t) 2})
        for (uint32_t ty : types)
            for (int rg = 1; rg <= 4; ++rg) {
                size_t o, m;
                c.type = ty;
                c.k = c.v = (void *) base;
                decode_scratch_need(c, Hq, P1A_MAX_ROWS, rg, req, cus, o, m);
                if (o > need_o) need_o = o;
                if (m > need_ml) need_ml = m;
            }
    last = memo{Hq, Hkv, D, req, cus, need_o, need_ml};
}

// ext / ext_bytes: split scratch brought by the caller of this function (the allocation-free entry point); nullptr = the
// library's own per-stream buffers
int decode_call(const float * q, const p1a_kv * c, float * out, const float * gate, void * qbuf, int T, int p0,
                const int32_t * p0_dev, const int32_t * pos_rows, int rows_per_seq, int Hq, float scale, bool split_only,
                hipStream_t s, void * ext = nullptr, size_t ext_bytes = 0) {
    if (!kv_ok(c, "p1a_attn_decode")) return P1A_E_ARG;
    if (qbuf && (((uintptr_t) qbuf & 15) || (Hq * c->D) % 32)) { set_error("p1a_attn_decode: qbuf must be 16-byte aligned and Hq*D %% 32 == 0"); return P1A_E_SHAPE; }
    if (!q || !out) { set_error("p1a_attn_decode: null q/out"); return P1A_E_ARG; }
    if (T < 1 || T > P1A_MAX_ROWS || Hq < c->Hkv || Hq % c->Hkv) {
        set_error("p1a_attn_decode: unsupported shape (D=%d Hq=%d Hkv=%d T=%d)", c->D, Hq, c->Hkv, T);
        return P1A_E_SHAPE;
    }
    if ((((uintptr_t) q | (uintptr_t) out | (uintptr_t) gate) & 15)) { set_error("p1a_attn_decode: q/out/gate must be 16-byte aligned"); return P1A_E_SHAPE; }
    if (!pos_rows && !p0_dev && p0 < 0) { set_error("p1a_attn_decode: negative p0"); return P1A_E_ARG; }
    decode_args a;
    a.q = q; a.out = out; a.gate = gate; a.T = T; a.p0 = p0; a.p0_dev = p0_dev; a.pos_rows = pos_rows;
    a.host_n = pos_rows || p0_dev ? 0 : (long long) p0 + T;
    a.Hq = Hq; a.scale = scale;
    a.rows_per_group = decode_rows_per_group(*c, Hq, pos_rows ? (rows_per_seq < 1 ? 1 : rows_per_seq) : T);
    // a sequence's rows must split into whole groups, or a group would mix two sequences
    while (pos_rows && rows_per_seq > 1 && rows_per_seq % a.rows_per_group) --a.rows_per_group;
    a.rows_per_seq = pos_rows ? (rows_per_seq < 1 ? 1 : rows_per_seq) : 1 << 30;
    a.nsplit = nsplit_req();
    a.cus = cu_count();
    a.skip_merge = split_only;
    a.qbuf = qbuf;
    size_t need_o, need_ml;
    if (ext) {
        decode_scratch_need(*c, Hq, T, a.rows_per_group, a.nsplit, a.cus, need_o, need_ml);
        need_o = (need_o + 255) & ~(size_t) 255;
        if (need_o + need_ml > ext_bytes) {
            set_error("p1a_attn_decode_noalloc: this call needs %zu bytes of split scratch, the static buffer holds %zu", need_o + need_ml, ext_bytes);
            return P1A_E_SCRATCH;
        }
        a.part_o = reinterpret_cast<float *>(ext);
        a.part_ml = reinterpret_cast<float *>(reinterpret_cast<char *>(ext) + need_o);
        a.cap_o = need_o; a.cap_ml = ext_bytes - need_o;
        return launch_decode(*c, a, s);
    }
    // the footprint of the head shape (so that the pointer never changes again), and never less than THIS call needs
    size_t real_o, real_ml;
    decode_scratch_need(*c, Hq, T, a.rows_per_group, a.nsplit, a.cus, real_o, real_ml);
    decode_footprint(Hq, c->Hkv, c->D, need_o, need_ml);
    if (real_o > need_o) need_o = real_o;
    if (real_ml > need_ml) need_ml = real_ml;
    bufpair * sc = scratch_for(s, BUF_DECODE, need_o, need_ml);
    if (!sc) return P1A_E_SCRATCH;
    a.part_o = sc->o; a.part_ml = sc->ml;
    a.cap_o = sc->cap_o; a.cap_ml = sc->cap_ml;
    return launch_decode(*c, a, s);
}


// the rows of a call over bounded caches, checked: what the kernels take (`max_n`: the most positions a sequence may hold)
int rows_ok(const p1a_kv * c, const p1a_rows * r, int Hq, const char * who, rows_view & R, int & max_n) {
    if (!kv_ok(c, who)) return P1A_E_ARG;
    if (!r || r->T < 0 || r->n_seq < 0 || r->max_rows < 0 || r->max_n < 0 || r->window < 0 || r->n_sink < 0 || c->n_ctx < 0) { set_error("%s: no rows, or a negative count among them", who); return P1A_E_ARG; }
    if (!r->pos0 && r->n_seq > 1) { set_error("%s: %d sequences need positions in device memory", who, r->n_seq); return P1A_E_ARG; }
    if (r->n_seq > 1 && (!c->pt || !c->rtab)) { set_error("%s: %d sequences need a page table and a row table", who, r->n_seq); return P1A_E_ARG; }
    if (!r->row0 && r->n_seq > 0 && r->T % r->n_seq) { set_error("%s: %d rows do not divide among %d sequences", who, r->T, r->n_seq); return P1A_E_ARG; }
    if ((c->D != 64 && c->D != 128 && c->D != 256) || Hq < c->Hkv || Hq % c->Hkv || Hq / c->Hkv > 64 || r->n_seq > 65535 || c->Hkv > 4096 || (long long) r->n_seq * c->Hkv > 1 << 22 || (long long) r->T * Hq > 1 << 30 || c->n_ctx > 1 << 30) {
        set_error("%s: unsupported shape (D=%d Hq=%d Hkv=%d T=%d n_seq=%d n_ctx=%d)", who, c->D, Hq, c->Hkv, r->T, r->n_seq, c->n_ctx);
        return P1A_E_SHAPE;
    }
    const uintptr_t al = c->type == P1A_KV_F16 ? 15 : c->type == P1A_KV_Q8_0 ? 3 : 1;
    if ((((uintptr_t) c->k | (uintptr_t) c->v) & al) || (c->pt && (c->pstride & al))) { set_error("%s: cache base / page stride must be %d-byte aligned", who, (int) al + 1); return P1A_E_SHAPE; }
    R.row0 = r->row0; R.pos0 = r->pos0; R.T = r->T; R.n_seq = r->n_seq; R.p0 = r->p0;
    R.per = r->row0 || !r->n_seq ? 0 : r->T / r->n_seq;
    R.max_rows = r->max_rows && r->max_rows < r->T ? r->max_rows : r->T;
    if (!r->row0 && R.per < R.max_rows) R.max_rows = R.per;
    R.window = r->window ? r->window : INT32_MAX;
    R.n_sink = r->window ? r->n_sink : 0;
    R.n_ctx = c->n_ctx;
    max_n = r->max_n && r->max_n < c->n_ctx ? r->max_n : c->n_ctx;
    if (!r->pos0) max_n = (int) std::max(1LL, std::min<long long>(max_n, (long long) r->p0 + r->T));
    return P1A_OK;
}
// the rows of a call on drafted trees that has no cache
int tree_rows_ok(const p1a_rows * r, const char * who, bool with_pos, rows_view & R) {
    if (!r || r->T < 0 || r->n_seq < 0 || r->max_rows < 0) { set_error("%s: no rows, or a negative count among them", who); return P1A_E_ARG; }
    if (with_pos && !r->pos0 && r->n_seq > 1) { set_error("%s: %d sequences need positions in device memory", who, r->n_seq); return P1A_E_ARG; }
    if (!r->row0 && r->n_seq > 0 && r->T % r->n_seq) { set_error("%s: %d rows do not divide among %d sequences", who, r->T, r->n_seq); return P1A_E_ARG; }
    R.row0 = r->row0; R.pos0 = r->pos0; R.T = r->T; R.n_seq = r->n_seq; R.p0 = r->p0;
    R.per = r->row0 || !r->n_seq ? 0 : r->T / r->n_seq;
    R.max_rows = r->max_rows && r->max_rows < r->T ? r->max_rows : r->T;
    if (!r->row0 && R.per < R.max_rows) R.max_rows = R.per;
    R.window = INT32_MAX; R.n_sink = 0; R.n_ctx = 1 << 30;
    if (r->T > 1 << 20 || r->n_seq > 65535 || R.max_rows > P1A_TREE_NODES) {
        set_error("%s: unsupported shape (T=%d n_seq=%d, %d nodes of a sequence): up to 2^20, 65535, %d", who, r->T, r->n_seq, R.max_rows, P1A_TREE_NODES);
        return P1A_E_SHAPE;
    }
    return P1A_OK;
}
bool rows_type_ok(int type, const char * who) {
    if (type == P1A_ROWS_F32 || type == P1A_ROWS_BF16) return true;
    set_error("%s: unknown type of rows %d", who, type);
    return false;
}

}   // namespace

bool split_scratch(hipStream_t s, size_t bytes_o, size_t bytes_ml, float *& o, float *& ml) {
    bufpair * e = scratch_for(s, BUF_PREFILL, bytes_o, bytes_ml);
    if (!e) return false;
    o = e->o; ml = e->ml;
    return true;
}

// The library's own f16 staging copy for a prefill over a quantized cache without caller scratch: a buffer of at least
// `bytes` bytes of (current device, s), or nullptr when there is none to be had now - over the limit, allocation failed, or
// the stream is being captured and the buffer would have to be allocated or grown. Never an error: the caller then
// converts inside the kernel, with the same result bits. Grown in steps (64 MiB granules, at least half as much again).
// A replaced buffer is freed on the spot (hipFree waits for the work that still reads it) unless a call under stream
// capture has been handed it - a captured graph holds its address - in which case it stays allocated until
// p1a_release(): what the library keeps per (device, stream) is at most the limit, plus what graphs pin.
void * stage_scratch(hipStream_t s, size_t bytes) {
    int dev = 0;
    if (!bytes || bytes > g_stage_limit || hipGetDevice(&dev) != hipSuccess) return nullptr;
    std::lock_guard<std::mutex> lk(g_mu);
    stream_bufs * e = nullptr;
    for (int i = 0; i < g_nscr; ++i) if (g_scr[i].dev == dev && g_scr[i].s == s) e = &g_scr[i];
    if (!e) {
        if (g_nscr == MAX_SCR) return nullptr;
        e = &g_scr[g_nscr++];
        e->dev = dev; e->s = s;
    }
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    const bool capturing = s && hipStreamIsCapturing(s, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
    if (bytes <= e->cap_stage) { if (capturing) e->stage_captured = true; return e->stage; }
    if (capturing) return nullptr;
    if (e->stage && e->stage_captured && g_nretired + 1 > MAX_RETIRED) return nullptr;
    const size_t gran = (size_t) 64 << 20;
    size_t want = (bytes + gran - 1) / gran * gran;
    if (want < e->cap_stage + e->cap_stage / 2) want = e->cap_stage + e->cap_stage / 2;
    if (want > g_stage_limit) want = g_stage_limit;
    if (want < bytes) want = bytes;
    void * p = nullptr;
    if (hipMalloc(&p, want) != hipSuccess) { (void) hipGetLastError(); return nullptr; }
    if (e->stage) {
        if (e->stage_captured) g_retired[g_nretired++] = retired{dev, e->stage};
        else (void) hipFree(e->stage);
    }
    e->stage = p; e->cap_stage = want; e->stage_captured = false;
    return p;
}

}   // namespace p1a

using namespace p1a;

extern "C" {

size_t p1a_kv_row_bytes(uint32_t type, int Hkv, int D) {
    return type == P1A_KV_F16 ? (size_t) Hkv * D * 2 : type == P1A_KV_Q8_0 ? (size_t) Hkv * (D / 32) * 34 : (size_t) Hkv * (D / 32) * 18;
}

int p1a_kv_append(const p1a_kv * c, const float * k, const float * v, int p0, const int32_t * p0_dev,
                  const int32_t * pos_rows, int T, void * stream) {
    if (!kv_ok(c, "p1a_kv_append")) return P1A_E_ARG;
    if (!k || !v || T < 0) { set_error("p1a_kv_append: null input or negative T"); return P1A_E_ARG; }
    if (T == 0) return P1A_OK;
    if ((((uintptr_t) k | (uintptr_t) v) & 15) || (c->Hkv * c->D) % 32) { set_error("p1a_kv_append: k/v must be 16-byte aligned, Hkv*D %% 32 == 0"); return P1A_E_SHAPE; }
    if (T > 65535) { set_error("p1a_kv_append: T=%d exceeds 65535 rows per call", T); return P1A_E_SHAPE; }
    if (!pos_rows && !p0_dev && p0 < 0) { set_error("p1a_kv_append: negative p0"); return P1A_E_ARG; }
    return launch_append(*c, k, v, p0, p0_dev, pos_rows, T, (hipStream_t) stream);
}

int p1a_kv_fill_random(const p1a_kv * c, int p0, int p1, uint32_t seed, void * stream) {
    if (!kv_ok(c, "p1a_kv_fill_random")) return P1A_E_ARG;
    if (p0 < 0) { set_error("p1a_kv_fill_random: negative p0"); return P1A_E_ARG; }
    if (p1 <= p0) return P1A_OK;
    if (c->type != P1A_KV_F16 && c->D % 32) { set_error("p1a_kv_fill_random: D %% 32 != 0"); return P1A_E_SHAPE; }
    if (!c->pt && p1 > c->n_ctx) { set_error("p1a_kv_fill_random: positions up to %d in a cache of %d", p1, c->n_ctx); return P1A_E_ARG; }
    return launch_fill_random(*c, p0, p1, seed, (hipStream_t) stream);
}

int p1a_attn_prep(const float * qg, const float * k, const float * v, const float * q_norm, const float * k_norm,
                  const int32_t * pos, float * q, float * gate, const p1a_kv * c, int p0, int T, int Hq, int n_rot,
                  float freq_base, float eps, int ldq, int ldk, int ldv, void * stream) {
    return p1a_attn_prep_mrope(qg, k, v, q_norm, k_norm, pos, q, gate, c, p0, T, Hq, n_rot, freq_base, eps, ldq, ldk, ldv,
                               nullptr, 0, 0, 0, 0, 0, stream);
}

int p1a_attn_prep_mrope(const float * qg, const float * k, const float * v, const float * q_norm, const float * k_norm,
                        const int32_t * pos, float * q, float * gate, const p1a_kv * c, int p0, int T, int Hq, int n_rot,
                        float freq_base, float eps, int ldq, int ldk, int ldv, const int32_t * mr_pos, int mr_stride,
                        int s0, int s1, int s2, int sect, void * stream) {
    if (!kv_ok(c, "p1a_attn_prep")) return P1A_E_ARG;
    if (mr_pos && (sect <= 0 || mr_stride < T || s0 < 0 || s1 < 0 || s2 < 0)) {
        set_error("p1a_attn_prep: M-RoPE needs sect > 0, sections >= 0 and a stream stride of at least T (sect=%d stride=%d)", sect, mr_stride);
        return P1A_E_ARG;
    }
    if (!qg || !k || !v || !pos || !q || !gate || T < 0 || Hq < 1) { set_error("p1a_attn_prep: null argument or bad T / Hq"); return P1A_E_ARG; }
    if (T == 0) return P1A_OK;
    const int D = c->D, Hkv = c->Hkv;
    if (D > 256 || n_rot < 0 || n_rot % 8 || n_rot > D || T > 65535) {
        set_error("p1a_attn_prep: unsupported shape (D=%d n_rot=%d T=%d): D <= 256, n_rot %% 8 == 0, n_rot <= D", D, n_rot, T);
        return P1A_E_SHAPE;
    }
    if (!(freq_base > 0.0f) || !(freq_base < 3.0e38f)) { set_error("p1a_attn_prep: freq_base must be a positive finite number"); return P1A_E_ARG; }
    if (!ldq) ldq = Hq * 2 * D;
    if (!ldk) ldk = Hkv * D;
    if (!ldv) ldv = Hkv * D;
    const uintptr_t al = (uintptr_t) qg | (uintptr_t) k | (uintptr_t) v | (uintptr_t) q | (uintptr_t) gate | (uintptr_t) q_norm | (uintptr_t) k_norm;
    if ((al & 15) || ((ldq | ldk | ldv) & 3) || ldq < Hq * 2 * D || ldk < Hkv * D || ldv < Hkv * D) {
        set_error("p1a_attn_prep: pointers must be 16-byte aligned, row strides multiples of 4 floats and at least one row");
        return P1A_E_SHAPE;
    }
    const mrope_view mr{mr_pos, mr_stride, s0, s1, s2, sect};
    return launch_prep(*c, qg, k, v, q_norm, k_norm, pos, q, gate, p0, T, Hq, n_rot, freq_base, eps, ldq, ldk, ldv, mr, (hipStream_t) stream);
}

size_t p1a_a16_bytes(int T, int n) { return T < 0 || n < 0 ? 0 : (size_t) T * (size_t) (n / 32) * 17 * 4; }

int p1a_ew_quant(int op, const float * a, const float * b, float * y, void * qbuf, int T, int n, int lda, int ldb, void * stream) {
    if (!a || !b || !y || !qbuf || T < 0 || (op != 0 && op != 1)) { set_error("p1a_ew_quant: null argument, negative T or unknown op"); return P1A_E_ARG; }
    if (T == 0) return P1A_OK;
    if (!lda) lda = n;
    if (!ldb) ldb = n;
    const uintptr_t al = (uintptr_t) a | (uintptr_t) b | (uintptr_t) y | (uintptr_t) qbuf;
    if (n < 32 || n % 32 || (al & 15) || ((lda | ldb) & 3) || lda < n || ldb < n || T > 65535 || (y == a && lda != n)) {
        set_error("p1a_ew_quant: n %% 32 == 0, 16-byte aligned pointers, row strides multiples of 4 and >= n (y may alias a only when dense)");
        return P1A_E_SHAPE;
    }
    return launch_ew_quant(op, a, b, y, qbuf, T, n, lda, ldb, (hipStream_t) stream);
}

int p1a_attn_decode(const float * q, const p1a_kv * c, float * out, const float * gate, int T, int p0,
                    const int32_t * p0_dev, const int32_t * pos_rows, int rows_per_seq, int Hq, float scale,
                    void * stream) {
    return p1a_attn_decode_a16(q, c, out, gate, nullptr, T, p0, p0_dev, pos_rows, rows_per_seq, Hq, scale, stream);
}

int p1a_attn_decode_a16(const float * q, const p1a_kv * c, float * out, const float * gate, void * qbuf, int T, int p0,
                        const int32_t * p0_dev, const int32_t * pos_rows, int rows_per_seq, int Hq, float scale,
                        void * stream) {
    return decode_call(q, c, out, gate, qbuf, T, p0, p0_dev, pos_rows, rows_per_seq, Hq, scale, false, (hipStream_t) stream);
}

int p1a_attn_decode_noalloc(const float * q, const p1a_kv * c, float * out, const float * gate, void * qbuf, int T, int p0,
                            const int32_t * p0_dev, const int32_t * pos_rows, int rows_per_seq, int Hq, float scale,
                            void * stream) {
    void * ptr = static_scratch();
    if (!ptr) return P1A_E_SCRATCH;
    return decode_call(q, c, out, gate, qbuf, T, p0, p0_dev, pos_rows, rows_per_seq, Hq, scale, false, (hipStream_t) stream,
                       ptr, P1A_NOALLOC_SCRATCH_BYTES);
}

int p1a_bench_decode_split_only(const float * q, const p1a_kv * c, float * out, int T, int p0, const int32_t * p0_dev,
                                const int32_t * pos_rows, int rows_per_seq, int Hq, float scale, void * stream) {
    return decode_call(q, c, out, nullptr, nullptr, T, p0, p0_dev, pos_rows, rows_per_seq, Hq, scale, true, (hipStream_t) stream);
}

int p1a_warmup(int rows, int Hq, int Hkv, int D, void * stream) {
    if (rows < 1 || rows > P1A_MAX_ROWS || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 32) { set_error("p1a_warmup: bad shape"); return P1A_E_ARG; }
    size_t need_o, need_ml;
    decode_footprint(Hq, Hkv, D, need_o, need_ml);
    (void) static_scratch();   // set-up time: the allocation-free entry point then has nothing left to resolve on this device
    return scratch_for((hipStream_t) stream, BUF_DECODE, need_o, need_ml) ? P1A_OK : P1A_E_SCRATCH;
}

int p1a_warmup_prefill(int T, int p0, int Hq, int Hkv, int D, void * stream) {
    if (T < 1 || p0 < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || D < 32) { set_error("p1a_warmup_prefill: bad shape"); return P1A_E_ARG; }
    size_t bo, bm;
    prefill_part_need(T, p0, Hq, Hkv, D, bo, bm);
    // (the f16 staging copy of a quantized cache, when it is within the limit: optional, a call without it converts in the kernel)
    (void) stage_scratch((hipStream_t) stream, prefill_stage_bytes(p0 + T, Hkv, D));
    if (!bo) return P1A_OK;
    return scratch_for((hipStream_t) stream, BUF_PREFILL, bo, bm) ? P1A_OK : P1A_E_SCRATCH;
}

void p1a_set_prefill_staging_limit(size_t bytes) { g_stage_limit = bytes; }

int p1a_attn_prefill(const float * q, const p1a_kv * c, float * out, const float * gate, int T, int p0, int Hq,
                     float scale, void * scratch, size_t scratch_bytes, void * stream) {
    if (!kv_ok(c, "p1a_attn_prefill")) return P1A_E_ARG;
    if (!q || !out || T < 1 || p0 < 0) { set_error("p1a_attn_prefill: bad argument"); return P1A_E_ARG; }
    if (Hq < c->Hkv || Hq % c->Hkv) { set_error("p1a_attn_prefill: unsupported shape (Hq=%d Hkv=%d)", Hq, c->Hkv); return P1A_E_SHAPE; }
    if ((((uintptr_t) q | (uintptr_t) out | (uintptr_t) gate) & 15)) { set_error("p1a_attn_prefill: q/out/gate must be 16-byte aligned"); return P1A_E_SHAPE; }
    return launch_prefill(*c, q, out, gate, T, p0, Hq, scale, scratch, scratch_bytes, (hipStream_t) stream);
}

int p1a_attn_chunk(const void * q, int q_type, const p1a_kv * c, void * out, int out_type, const float * gate, float * lse, const p1a_rows * rows,
                   int Hq, float scale, void * scratch, size_t scratch_bytes, void * stream) {
    static const char * const who = "p1a_attn_chunk";
    chunk_args a;
    const int rc = rows_ok(c, rows, Hq, who, a.R, a.max_n);
    if (rc != P1A_OK) return rc;
    if (!q || !out || !rows_type_ok(q_type, who) || !rows_type_ok(out_type, who)) { if (!q || !out) set_error("%s: null q/out", who); return P1A_E_ARG; }
    if (((uintptr_t) q | (uintptr_t) out | (uintptr_t) gate) & 15 || (uintptr_t) lse & 3) { set_error("%s: q/out/gate must be 16-byte aligned, lse 4-byte", who); return P1A_E_SHAPE; }
    if (!rows->T || !rows->n_seq) return P1A_OK;
    a.q = q; a.out = out; a.gate = gate; a.lse = lse; a.q_bf16 = q_type == P1A_ROWS_BF16; a.out_bf16 = out_type == P1A_ROWS_BF16;
    a.Hq = Hq; a.scale = scale; a.scratch = scratch; a.scratch_bytes = scratch_bytes;
    return launch_chunk(*c, a, (hipStream_t) stream);
}

size_t p1a_attn_chunk_scratch_bytes(const p1a_kv * c, const p1a_rows * rows, int Hq) {
    rows_view R;
    int max_n;
    if (rows_ok(c, rows, Hq, "p1a_attn_chunk_scratch_bytes", R, max_n) != P1A_OK || !rows->T || !rows->n_seq) return 0;
    const chunk_plan pl = plan_chunk(*c, R, Hq, max_n, cu_count());
    return pl.bytes_n + pl.bytes_ml + pl.bytes_o;
}

int p1a_attn_mass(const void * q, int q_type, const p1a_kv * c, const float * lse, float * mass, int ld, const p1a_rows * rows, int Hq, float scale,
                  void * scratch, size_t scratch_bytes, void * stream) {
    static const char * const who = "p1a_attn_mass";
    mass_args a;
    const int rc = rows_ok(c, rows, Hq, who, a.R, a.max_n);
    if (rc != P1A_OK) return rc;
    if (!q || !lse || !mass || ld < 0) { set_error("%s: null q / lse / mass or negative ld", who); return P1A_E_ARG; }
    if (!rows_type_ok(q_type, who)) return P1A_E_ARG;
    if (ld > 1 << 30) { set_error("%s: unsupported shape (ld=%d)", who, ld); return P1A_E_SHAPE; }
    if (((uintptr_t) q & 15) || (((uintptr_t) lse | (uintptr_t) mass) & 3)) { set_error("%s: q must be 16-byte aligned, lse and mass 4-byte", who); return P1A_E_SHAPE; }
    if (!rows->T || !rows->n_seq || !ld) return P1A_OK;
    a.q = q; a.q_bf16 = q_type == P1A_ROWS_BF16; a.lse = lse; a.mass = mass; a.ld = ld; a.Hq = Hq; a.scale = scale; a.scratch = scratch; a.scratch_bytes = scratch_bytes;
    return launch_mass(*c, a, (hipStream_t) stream);
}

size_t p1a_attn_mass_scratch_bytes(const p1a_kv * c, int ld, const p1a_rows * rows, int Hq) {
    rows_view R;
    int max_n;
    if (rows_ok(c, rows, Hq, "p1a_attn_mass_scratch_bytes", R, max_n) != P1A_OK || !rows->T || !rows->n_seq || ld < 1 || ld > 1 << 30) return 0;
    return plan_mass(*c, R, Hq, max_n, ld, cu_count()).bytes;
}

int p1a_evict_select(const float * mass, int ld, int n_seq, int Hkv, const int32_t * n_dev, int n, int budget, int n_sink, int n_recent,
                     int32_t * keep, void * stream) {
    static const char * const who = "p1a_evict_select";
    if (!mass || !keep || ld < 0 || n_seq < 0 || Hkv < 1 || n_sink < 0 || n_recent < 0 || (!n_dev && n < 0)) { set_error("%s: null argument or a negative count", who); return P1A_E_ARG; }
    if (budget < 0 || budget > 1 << 20 || (long long) n_sink + n_recent > budget || n_seq > 65535 || Hkv > 4096 || ld > 1 << 30) {
        set_error("%s: budget=%d must hold n_sink=%d and n_recent=%d and be at most 2^20, n_seq=%d, Hkv=%d, ld=%d at most 65535, 4096, 2^30", who, budget, n_sink, n_recent, n_seq, Hkv, ld);
        return P1A_E_SHAPE;
    }
    if (((uintptr_t) mass | (uintptr_t) keep) & 3) { set_error("%s: mass and keep must be 4-byte aligned", who); return P1A_E_SHAPE; }
    if (!n_seq || !budget) return P1A_OK;
    return launch_evict_select(mass, ld, n_seq, Hkv, n_dev, n, budget, n_sink, n_recent, keep, (hipStream_t) stream);
}

int p1a_kv_compact(const p1a_kv * c, const int32_t * keep, int n_seq, int budget, const float * mass, float * mass_out, int ld, void * stream) {
    static const char * const who = "p1a_kv_compact";
    if (!kv_ok(c, who)) return P1A_E_ARG;
    if (!keep || n_seq < 0 || budget < 0 || !mass != !mass_out || (mass && ld < 0) || c->n_ctx < 0) { set_error("%s: null keep, a negative count, or one of mass and mass_out alone", who); return P1A_E_ARG; }
    if (n_seq > 1 && (!c->pt || !c->rtab)) { set_error("%s: %d sequences need a page table and a row table", who, n_seq); return P1A_E_ARG; }
    if (budget > 1 << 20 || n_seq > 65535 || (long long) n_seq * c->Hkv * ((head_bytes(c->type, c->D) + 15) / 16) > 1 << 20 || (mass && ld > 1 << 30)) {
        set_error("%s: unsupported shape (budget=%d n_seq=%d Hkv=%d D=%d ld=%d)", who, budget, n_seq, c->Hkv, c->D, ld);
        return P1A_E_SHAPE;
    }
    if ((((uintptr_t) c->k | (uintptr_t) c->v) & 1) || (c->pt && (c->pstride & 1)) || (((uintptr_t) keep | (uintptr_t) mass | (uintptr_t) mass_out) & 3)) {
        set_error("%s: cache base and page stride must be 2-byte aligned, keep and mass 4-byte", who);
        return P1A_E_SHAPE;
    }
    if (mass && mass != mass_out && mass < mass_out + (size_t) n_seq * c->Hkv * ld && mass_out < mass + (size_t) n_seq * c->Hkv * ld) { set_error("%s: mass and mass_out overlap in part", who); return P1A_E_ARG; }
    if (!n_seq || (!budget && !mass)) return P1A_OK;
    return launch_kv_compact(*c, keep, n_seq, budget, mass, mass_out, ld, (hipStream_t) stream);
}

int p1a_tree_rows(const int32_t * parent, const p1a_rows * rows, uint32_t * mask, int words, int32_t * pos, int32_t * slot, void * stream) {
    static const char * const who = "p1a_tree_rows";
    rows_view R;
    const int rc = tree_rows_ok(rows, who, true, R);
    if (rc != P1A_OK) return rc;
    if ((rows->T && (!parent || !mask)) || words < 0) { set_error("%s: null parent / mask or negative words", who); return P1A_E_ARG; }   // (no rows: tensors without memory)
    if ((long long) words * 32 < R.max_rows || words > P1A_TREE_NODES / 32) { set_error("%s: %d words for trees of %d nodes", who, words, R.max_rows); return P1A_E_SHAPE; }
    if (((uintptr_t) parent | (uintptr_t) mask | (uintptr_t) pos | (uintptr_t) slot) & 3) { set_error("%s: pointers must be 4-byte aligned", who); return P1A_E_SHAPE; }
    if (!rows->T || !rows->n_seq) return P1A_OK;
    return launch_tree_rows(parent, R, mask, words, pos, slot, (hipStream_t) stream);
}

int p1a_attn_tree(const void * q, int q_type, const p1a_kv * c, void * out, int out_type, const float * gate, float * lse, const p1a_rows * rows,
                  const uint32_t * mask, int words, int Hq, float scale, void * scratch, size_t scratch_bytes, void * stream) {
    static const char * const who = "p1a_attn_tree";
    chunk_args a;
    const int rc = rows_ok(c, rows, Hq, who, a.R, a.max_n);
    if (rc != P1A_OK) return rc;
    if ((rows->T && (!q || !out || !mask)) || words < 0) { set_error("%s: null q / out / mask or negative words", who); return P1A_E_ARG; }
    if (!rows_type_ok(q_type, who) || !rows_type_ok(out_type, who)) return P1A_E_ARG;
    if (((uintptr_t) q | (uintptr_t) out | (uintptr_t) gate) & 15 || ((uintptr_t) lse | (uintptr_t) mask) & 3) { set_error("%s: q/out/gate must be 16-byte aligned, lse and mask 4-byte", who); return P1A_E_SHAPE; }
    if (a.R.max_rows > P1A_TREE_NODES || (long long) words * 32 < a.R.max_rows || words > P1A_TREE_NODES / 32) { set_error("%s: %d words for trees of %d nodes (up to %d)", who, words, a.R.max_rows, P1A_TREE_NODES); return P1A_E_SHAPE; }
    if (!rows->T || !rows->n_seq) return P1A_OK;
    a.q = q; a.out = out; a.gate = gate; a.lse = lse; a.q_bf16 = q_type == P1A_ROWS_BF16; a.out_bf16 = out_type == P1A_ROWS_BF16;
    a.Hq = Hq; a.scale = scale; a.scratch = scratch; a.scratch_bytes = scratch_bytes;
    return launch_tree(*c, a, mask, words, (hipStream_t) stream);
}

size_t p1a_attn_tree_scratch_bytes(const p1a_kv * c, const p1a_rows * rows, int Hq, int f32) {
    static const char * const who = "p1a_attn_tree_scratch_bytes";
    rows_view R;
    int max_n;
    if (rows_ok(c, rows, Hq, who, R, max_n) != P1A_OK || !rows->T || !rows->n_seq || R.max_rows > P1A_TREE_NODES) return 0;
    const tree_plan pl = plan_tree(*c, R, Hq, max_n, f32 != 0, cu_count());
    return pl.bytes_n + pl.bytes_ml + pl.bytes_o;
}

int p1a_tree_verify(const void * target, int target_type, size_t ld_target, const void * draft, int draft_type, size_t ld_draft, int V, const int32_t * token,
                    const int32_t * parent, const float * temp, const float * u, const float * u_next, int32_t * n_accept, int32_t * path, int ld_path, int32_t * next,
                    const p1a_rows * rows, int max_children, int flags, void * scratch, size_t scratch_bytes, void * stream) {
    static const char * const who = "p1a_tree_verify";
    verify_args a;
    const int rc = tree_rows_ok(rows, who, false, a.R);
    if (rc != P1A_OK) return rc;
    if ((rows->T && (!target || !token || !u)) || !u_next || !n_accept || !path || !next || ld_path < 1 || V < 1 || flags & ~(P1A_VERIFY_PROBS | P1A_VERIFY_DISTINCT) || (draft && parent && max_children < 1)) {
        set_error("%s: null argument, unknown flag, or a count below 1 (ld_path=%d V=%d max_children=%d)", who, ld_path, V, max_children);
        return P1A_E_ARG;
    }
    if (!rows_type_ok(target_type, who) || (draft && !rows_type_ok(draft_type, who))) return P1A_E_ARG;
    if (!ld_target) ld_target = V;
    if (!ld_draft) ld_draft = V;
    if (V > 1 << 20 || ld_target < (size_t) V || ld_draft < (size_t) V || ld_target > (size_t) 1 << 40 || ld_draft > (size_t) 1 << 40) { set_error("%s: unsupported shape (V=%d, rows %zu and %zu apart)", who, V, ld_target, ld_draft); return P1A_E_SHAPE; }
    const uintptr_t words = (uintptr_t) token | (uintptr_t) parent | (uintptr_t) temp | (uintptr_t) u | (uintptr_t) u_next | (uintptr_t) n_accept | (uintptr_t) path | (uintptr_t) next;
    if (words & 3 || (uintptr_t) target & (target_type == P1A_ROWS_BF16 ? 1 : 3) || (draft && (uintptr_t) draft & (draft_type == P1A_ROWS_BF16 ? 1 : 3))) { set_error("%s: tensors must be aligned to their types", who); return P1A_E_SHAPE; }
    if (!rows->n_seq) return P1A_OK;
    a.target = target; a.draft = draft; a.ld_target = ld_target; a.ld_draft = ld_draft; a.token = token; a.parent = parent; a.temp = temp; a.u = u; a.u_next = u_next;
    a.n_accept = n_accept; a.path = path; a.next = next; a.V = V; a.ld_path = ld_path; a.max_children = max_children;
    a.target_bf16 = target_type == P1A_ROWS_BF16; a.draft_bf16 = draft && draft_type == P1A_ROWS_BF16; a.logits = !(flags & P1A_VERIFY_PROBS); a.distinct = flags & P1A_VERIFY_DISTINCT;
    a.scratch = scratch; a.scratch_bytes = scratch_bytes;
    return launch_verify(a, (hipStream_t) stream);
}

size_t p1a_tree_verify_scratch_bytes(const p1a_rows * rows, int V, int flags) {
    rows_view R;
    if (tree_rows_ok(rows, "p1a_tree_verify_scratch_bytes", false, R) != P1A_OK || !rows->n_seq || V < 1 || V > 1 << 20) return 0;
    return plan_verify(R, V, !(flags & P1A_VERIFY_PROBS), true).bytes;
}

int p1a_tree_commit(const p1a_kv * layers, int n_layers, const p1a_rows * rows, const int32_t * n_accept, const int32_t * path, int ld_path, void * stream) {
    static const char * const who = "p1a_tree_commit";
    rows_view R;
    const int rc = tree_rows_ok(rows, who, true, R);
    if (rc != P1A_OK) return rc;
    if (!layers || n_layers < 0 || !n_accept || !path || ld_path < 1) { set_error("%s: null argument or a bad count (n_layers=%d ld_path=%d)", who, n_layers, ld_path); return P1A_E_ARG; }
    if (n_layers > P1A_TREE_LAYERS) { set_error("%s: %d layers, up to %d a call", who, n_layers, P1A_TREE_LAYERS); return P1A_E_SHAPE; }
    for (int i = 0; i < n_layers; ++i) {
        const p1a_kv & c = layers[i], & f = layers[0];
        if (!kv_ok(&c, who)) return P1A_E_ARG;
        if (c.type != f.type || c.n_ctx != f.n_ctx || c.Hkv != f.Hkv || c.D != f.D || c.pt != f.pt || c.rtab != f.rtab || c.psh != f.psh || c.pstride != f.pstride || c.n_ctx < 0) {
            set_error("%s: layer %d has another shape or page table than the first, or a negative n_ctx", who, i);
            return P1A_E_ARG;
        }
        if (R.n_seq > 1 && (!c.pt || !c.rtab)) { set_error("%s: %d sequences need a page table and a row table", who, R.n_seq); return P1A_E_ARG; }
        if ((((uintptr_t) c.k | (uintptr_t) c.v) & 1) || (c.pt && (c.pstride & 1))) { set_error("%s: cache base and page stride must be 2-byte aligned", who); return P1A_E_SHAPE; }
    }
    if (((uintptr_t) n_accept | (uintptr_t) path) & 3) { set_error("%s: n_accept and path must be 4-byte aligned", who); return P1A_E_SHAPE; }
    if (!rows->T || !rows->n_seq || !n_layers) return P1A_OK;
    R.n_ctx = layers[0].n_ctx;
    return launch_tree_commit(layers, n_layers, R, n_accept, path, ld_path, (hipStream_t) stream);
}

int p1a_sigmoid_mul(float * x, const float * g, size_t n, void * stream) {
    if (!x || !g) { set_error("p1a_sigmoid_mul: null argument"); return P1A_E_ARG; }
    if (!n) return P1A_OK;
    return launch_sigmoid_mul(x, g, n, (hipStream_t) stream);
}

int p1a_get_nsplit(int Hkv) {
    p1a_kv c;
    memset(&c, 0, sizeof c);
    c.type = P1A_KV_Q8_0; c.Hkv = Hkv < 1 ? 1 : Hkv; c.D = 256; c.k = c.v = (void *) 16;
    return decode_nsplit(c, 6 * c.Hkv, nsplit_req(), cu_count());
}

void p1a_set_nsplit(int n) { g_nsplit_override = n > 0 ? n : 0; }

size_t p1a_decode_scratch_bytes(const p1a_kv * c, int Hq, int T, int rows_per_seq) {
    if (!c || c->Hkv < 1 || Hq < c->Hkv || Hq % c->Hkv || T < 1) return 0;
    int rg = decode_rows_per_group(*c, Hq, rows_per_seq < 1 ? 1 : rows_per_seq);
    while (rows_per_seq > 1 && rows_per_seq % rg) --rg;
    size_t o, m;
    decode_scratch_need(*c, Hq, T, rg, nsplit_req(), cu_count(), o, m);
    return ((o + 255) & ~(size_t) 255) + m;
}

size_t p1a_decode_footprint_bytes(int Hq, int Hkv, int D) {
    if (Hkv < 1 || Hq < Hkv || Hq % Hkv || D < 32) return 0;
    size_t o, m;
    decode_footprint(Hq, Hkv, D, o, m);
    return ((o + 255) & ~(size_t) 255) + m;
}

uint64_t p1a_numerics_id(int Hq, int Hkv) {
    // FNV-1a over what fixes the summation order of the results on this device
    uint64_t h = 1469598103934665603ull;
    auto mix = [&](uint64_t v) { for (int i = 0; i < 8; ++i) { h ^= (v >> (8 * i)) & 0xff; h *= 1099511628211ull; } };
    for (const char * p = p1a_version(); *p; ++p) { h ^= (unsigned char) *p; h *= 1099511628211ull; }
    mix((uint64_t) P1A_NUMERICS_REV);
    mix((uint64_t) cu_count());
    mix((uint64_t) p1a_get_nsplit(Hkv < 1 ? 1 : Hkv));
    mix((uint64_t) (Hq > 0 ? Hq : 0));
    mix((uint64_t) (Hkv > 0 ? Hkv : 0));
    return h;
}

int p1a_reload_env(void) {
    const int v = read_env_split();
    // (the first read counts as a change, as in the reference, whose switch starts out unread: src/fast/attn_dec2.cu reload)
    const bool changed = v != g_env_split;
    g_env_split = v;
    return changed ? 1 : 0;
}

int p1a_bench_stream_read(const void * src, size_t bytes, void * stream) {
    if (!src || bytes < 16 || ((uintptr_t) src & 15)) { set_error("p1a_bench_stream_read: null, short or misaligned source"); return P1A_E_ARG; }
    return launch_stream_read(src, bytes, (hipStream_t) stream);
}

void p1a_release(void) {
    std::lock_guard<std::mutex> lk(g_mu);
    int cur = 0;
    (void) hipGetDevice(&cur);
    for (int i = 0; i < g_nscr; ++i) {
        (void) hipSetDevice(g_scr[i].dev);
        (void) hipDeviceSynchronize();
        for (bufpair * b : {&g_scr[i].dec, &g_scr[i].pf})
            if (b->o) { (void) hipFree(b->o); (void) hipFree(b->ml); }
        if (g_scr[i].stage) (void) hipFree(g_scr[i].stage);
        g_scr[i] = stream_bufs{};
    }
    g_nscr = 0;
    for (int i = 0; i < g_nretired; ++i) {
        (void) hipSetDevice(g_retired[i].dev);
        (void) hipFree(g_retired[i].p);
    }
    g_nretired = 0;
    (void) hipSetDevice(cur);
}

const char * p1a_last_error(void) { return g_err; }
const char * p1a_version(void) { return "p1a_attn 0.1 (gfx950)"; }

}   // extern "C"
