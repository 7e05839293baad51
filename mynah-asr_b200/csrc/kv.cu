// The paged key/value cache at the C boundary (include/mynah_b200.h): checks of arguments, the handle and its memory.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <mutex>
#include <new>

#include "../../include/mynah_b200.h"
#include "kv.h"

using namespace mb;

// Device memory of a handle: the two pools, and a block [status, what a sync took of it, 256 B | turns of the rotation | norm weights].
struct mynah_b200_kv {
    mynah_b200_kv_config cfg;
    int fmt = KV_BF16, device = 0;
    cudaStream_t stream = nullptr;
    uint16_t *k = nullptr, *v = nullptr;
    uint8_t *block = nullptr;
    double *turns = nullptr;
    float *q_norm = nullptr, *k_norm = nullptr;
    CUtensorMap map_k, map_v, chunk_k, chunk_v;                // for single tokens, for prompts
    int chunk_box = 0;
    std::mutex syncing;
    bool owed = false;                                         // what was taken has not reached the host
    int *status() const { return reinterpret_cast<int *>(block); }
    int *taken() const { return reinterpret_cast<int *>(block + 128); }
    ~mynah_b200_kv() {
        cudaFree(k); cudaFree(v); cudaFree(block);              // (waits for the handle's work)
        if (stream) cudaStreamDestroy(stream);
    }
};

namespace {
// The handle's device is the current one while a call runs, and its context the calling thread's: a thread that has made no CUDA call yet has a
// device, but no context, which the encoding of tensor maps asks for.
struct OnDevice {
    static thread_local int bound;                             // the device that the thread has been set to
    int before = -1;
    explicit OnDevice(int dev) {
        if (cudaGetDevice(&before) != cudaSuccess) { cudaGetLastError(); before = -1; }
        if (before != dev || bound != dev) cudaSetDevice(dev);
        bound = dev;
        if (before == dev) before = -1;
    }
    ~OnDevice() {
        if (before < 0) return;
        cudaSetDevice(before);
        bound = before;
    }
};
thread_local int OnDevice::bound = -1;

int row_bytes(int fmt) { return fmt == KV_F32 ? 4 : 2; }

bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }

const char *refuse_config(const mynah_b200_kv_config &c, int *fmt) {
    if (c.fmt == MYNAH_B200_F32) *fmt = KV_F32;
    else if (c.fmt == MYNAH_B200_F16) *fmt = KV_F16;
    else if (c.fmt == MYNAH_B200_BF16) *fmt = KV_BF16;
    else return "rows are F32, F16 or BF16";
    if (c.n_kv_heads < 1 || c.n_heads < 1 || c.n_heads % c.n_kv_heads || c.n_heads / c.n_kv_heads > 64 || c.n_heads > 1024)
        return "n_heads is 1 to 64 times n_kv_heads, at most 1024";
    if (c.head_dim < 16 || c.head_dim > 128 || c.head_dim % 16) return "head_dim is a multiple of 16 up to 128";
    if (!power_of_two(c.page_size) || c.page_size < 8 || c.page_size > 256) return "page_size is a power of two from 8 to 256";
    if (c.n_pages < 1 || (int64_t)c.n_pages * c.page_size * c.n_kv_heads > 0x7fffffffll) return "n_pages x page_size x n_kv_heads is from 1 page to 2^31 - 1 rows";
    if (c.rotary_dim < 0 || c.rotary_dim > c.head_dim || c.rotary_dim % 8) return "rotary_dim is a multiple of 8 up to head_dim";
    if (c.rotary_dim && !c.inv_freq && !(c.rope_theta > 0 && isfinite(c.rope_theta))) return "rope_theta is positive";
    if (c.window < 0 || c.n_sinks < 0 || (c.n_sinks && !c.window)) return "window and n_sinks are not negative, and sinks need a window";
    if (!(c.scale == 0 || (c.scale >= 1e-20f && c.scale <= 1e20f))) return "scale is 0 or from 1e-20 to 1e20";
    if ((c.q_norm || c.k_norm) && !(c.norm_eps >= 0 && isfinite(c.norm_eps))) return "norm_eps is not negative";
    return nullptr;
}

// Memory that a kernel on `dev` can reach. An address of the host or of another GPU would be a fault there.
bool reachable(const void *p, int dev) {
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) { cudaGetLastError(); return false; }
    return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev) ||
           (at.type == cudaMemoryTypeHost && at.devicePointer == p);
}

}  // namespace

namespace mb {
typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);

static bool encode(CUtensorMap *m, bool bf, int rank, const void *base, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<EncodeFn>(p);
        cudaGetLastError();
        return EncodeFn(nullptr);
    }();
    const cuuint32_t one[3] = {1, 1, 1};
    return fn && fn(m, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, one,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// A pool as [rows][D]: boxes of 64 columns (zeros beyond D) and box_rows slots of one page and head, 128-byte swizzle
static bool pool_map(CUtensorMap *m, const uint16_t *pool, const mynah_b200_kv_config &c, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.n_pages * c.page_size * c.n_kv_heads}, strides[1] = {(cuuint64_t)c.head_dim * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    return encode(m, c.fmt == MYNAH_B200_BF16, 2, pool, dims, strides, box);
}
bool kv_rows_map(CUtensorMap *m, const KvArgs &a, bool bf) {
    const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.H, (cuuint64_t)a.n_rows}, strides[2] = {(cuuint64_t)a.D * 2, (cuuint64_t)a.ldq * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)(128 / a.G)};
    return encode(m, bf, 3, a.q, dims, strides, box);
}
}  // namespace mb

namespace {

// Rows of `width` values with stride ld, of which the last one ends where the buffer does
const char *refuse_rows(const mynah_b200_kv *h, const void *p, long long ld, int width) {
    if (!p) return "a null pointer";
    if (ld < width) return "a row stride below the row's width";
    if (ld > (1ll << 36)) return "a row stride out of range";
    if (((uintptr_t)p & 15) || (ld * row_bytes(h->fmt)) % 16) return "rows start on 16-byte boundaries";
    if (!reachable(p, h->device)) return "a pointer that is not of the handle's device";
    return nullptr;
}

// Whether rows that are written share values with rows that are read, other than by being the same ones: one row's result would be read as
// another's input. `n` rows of `width` values, `size` bytes each.
bool clash(const void *out, long long ldo, int wo, const void *in, long long ldi, int wi, int n, int size) {
    if (out == in && (ldo == ldi || n == 1)) return false;
    const uintptr_t o = (uintptr_t)out, i = (uintptr_t)in;
    if (o + ((uintptr_t)(n - 1) * ldo + wo) * size <= i || i + ((uintptr_t)(n - 1) * ldi + wi) * size <= o) return false;
    if (ldo != ldi) return true;
    // side by side in wider rows: the columns where those behind begin
    const uintptr_t ld = (uintptr_t)ldo * size, ahead = (o > i ? o - i : i - o) % ld, first = (uintptr_t)(o > i ? wi : wo) * size, second = (uintptr_t)(o > i ? wo : wi) * size;
    return ahead < first || ahead + second > ld;
}

// 1: nothing to do, 0: go on, -1: refused
int take_batch(const char *what, const mynah_b200_kv *h, const mynah_b200_kv_batch *b, KvArgs *a) {
    const mynah_b200_kv_config &c = h->cfg;
    const char *no = nullptr;
    if (b->n_seq < 0 || b->n_rows < 0) no = "a negative count";
    else if (b->n_seq > KV_MOST_SEQ || b->n_rows > 1 << 30) no = "at most 2^16 sequences and 2^30 rows";
    else if (b->n_seq == 0 || b->n_rows == 0) return 1;
    else if (!b->kv_len || !b->page_table) no = "a null table";
    else if (b->max_pages < 1 || (int64_t)b->max_pages * c.page_size > KV_MOST) no = "max_pages x page_size is from 1 page to 2^26 positions";
    else if (!b->row_off && b->n_rows < b->n_seq) no = "fewer rows than sequences";
    else if (((uintptr_t)b->kv_len | (uintptr_t)b->page_table | (uintptr_t)b->row_off) & 3) no = "a misaligned table";
    else if (!reachable(b->kv_len, h->device) || !reachable(b->page_table, h->device) || (b->row_off && !reachable(b->row_off, h->device)))
        no = "a table that is not of the handle's device";
    if (no) { set_error("%s: %s", what, no); return -1; }
    a->H = c.n_heads; a->Hkv = c.n_kv_heads; a->G = c.n_heads / c.n_kv_heads; a->D = c.head_dim;
    a->page_shift = __builtin_ctz((unsigned)c.page_size); a->n_pages = c.n_pages;
    a->window = c.window < KV_MOST ? c.window : KV_MOST; a->sinks = c.n_sinks < KV_MOST ? c.n_sinks : KV_MOST;
    const double scale = c.scale > 0 ? (double)c.scale : 1 / sqrt((double)c.head_dim);
    a->scale2 = (float)(scale * 1.4426950408889634);
    a->k = h->k; a->v = h->v; a->status = h->status();
    a->n_seq = b->n_seq; a->n_rows = b->n_rows; a->max_pages = b->max_pages;
    a->row_off = b->row_off; a->kv_len = b->kv_len; a->table = b->page_table;
    return 0;
}

__global__ void kv_take_kernel(int *status, int *taken, int keep) {
    const int found = atomicExch(status, 0);
    *taken = keep ? *taken | found : found;
}
}  // namespace

extern "C" {

void mynah_b200_kv_config_default(mynah_b200_kv_config *c) {
    if (!c) return;
    memset(c, 0, sizeof(*c));
    c->page_size = 16;
    c->fmt = MYNAH_B200_F32;
    c->rope_theta = 10000.0;
    c->norm_eps = 1e-6f;
}

mynah_b200_kv *mynah_b200_kv_create(const mynah_b200_kv_config *cfg) {
    if (!mynah_b200_available()) { set_error("no sm_100 CUDA device available"); return nullptr; }
    if (!cfg) { set_error("kv_create: null config"); return nullptr; }
    int fmt = 0;
    if (const char *no = refuse_config(*cfg, &fmt)) { set_error("kv_create: %s", no); return nullptr; }
    const int rot = cfg->rotary_dim, D = cfg->head_dim;
    double turns[64];
    for (int i = 0; i < rot / 2; i++) {
        const double f = cfg->inv_freq ? cfg->inv_freq[i] : pow(cfg->rope_theta, -2.0 * i / rot);
        if (!isfinite(f)) { set_error("kv_create: a rotation frequency is not finite"); return nullptr; }
        turns[i] = f / 6.283185307179586476925;
    }
    for (int i = 0; i < 2 * D; i++) {
        const float *w = i < D ? cfg->q_norm : cfg->k_norm;
        if (w && !isfinite(w[i % D])) { set_error("kv_create: a norm weight is not finite"); return nullptr; }
    }
    RelaxedCapture relaxed;
    mynah_b200_kv *h = new (std::nothrow) mynah_b200_kv();
    if (!h) { set_error("kv_create: host allocation failed"); return nullptr; }
    h->cfg = *cfg; h->fmt = fmt;
    h->cfg.inv_freq = nullptr; h->cfg.q_norm = h->cfg.k_norm = nullptr;              // borrowed for this call only
    const size_t pool = (size_t)cfg->n_pages * cfg->page_size * cfg->n_kv_heads * D * sizeof(uint16_t);
    const size_t block = 256 + sizeof(turns) + 2 * 128 * sizeof(float);
    bool ok = cudaGetDevice(&h->device) == cudaSuccess && cudaStreamCreateWithFlags(&h->stream, cudaStreamNonBlocking) == cudaSuccess &&
              cudaMalloc((void **)&h->block, block) == cudaSuccess && cudaMalloc((void **)&h->k, pool) == cudaSuccess &&
              cudaMalloc((void **)&h->v, pool) == cudaSuccess;
    if (ok) {
        h->turns = reinterpret_cast<double *>(h->block + 256);
        float *norms = reinterpret_cast<float *>(h->block + 256 + sizeof(turns));
        if (cfg->q_norm) h->q_norm = norms;
        if (cfg->k_norm) h->k_norm = norms + 128;
        // every slot is finite from the start: what a mask hides is multiplied by a probability of 0
        ok = cudaMemsetAsync(h->block, 0, block, h->stream) == cudaSuccess && cudaMemsetAsync(h->k, 0, pool, h->stream) == cudaSuccess &&
             cudaMemsetAsync(h->v, 0, pool, h->stream) == cudaSuccess;
        // (not by the legacy default stream, which may not wait for a stream that another thread records)
        auto put = [&](void *to, const void *from, size_t n) { return cudaMemcpyAsync(to, from, n, cudaMemcpyHostToDevice, h->stream) == cudaSuccess; };
        ok = ok && (!rot || put(h->turns, turns, (size_t)(rot / 2) * sizeof(double))) && (!cfg->q_norm || put(h->q_norm, cfg->q_norm, (size_t)D * sizeof(float))) &&
             (!cfg->k_norm || put(h->k_norm, cfg->k_norm, (size_t)D * sizeof(float)));
        ok = cudaStreamSynchronize(h->stream) == cudaSuccess && ok;
    }
    if (!ok) {
        const cudaError_t e = cudaGetLastError();
        set_error("kv_create: device memory for 2 x %zu bytes: %s", pool, cudaGetErrorString(e));
        delete h;
        return nullptr;
    }
    const int box = kv_box(D, cfg->page_size);
    h->chunk_box = cfg->page_size < 32 ? cfg->page_size : 32;
    if (!pool_map(&h->map_k, h->k, *cfg, box) || !pool_map(&h->map_v, h->v, *cfg, box) || !pool_map(&h->chunk_k, h->k, *cfg, h->chunk_box) ||
        !pool_map(&h->chunk_v, h->v, *cfg, h->chunk_box)) {
        set_error("kv_create: no tensor map of the pools");
        delete h;
        return nullptr;
    }
    return h;
}

void mynah_b200_kv_free(mynah_b200_kv *h) {
    if (!h) return;
    OnDevice on(h->device);
    RelaxedCapture relaxed;
    delete h;
}

int mynah_b200_kv_pages(const mynah_b200_kv *h, void **k, void **v) {
    if (!h || !k || !v) { set_error("kv_pages: bad argument"); return -1; }
    *k = h->k; *v = h->v;
    return 0;
}

int mynah_b200_kv_append(mynah_b200_kv *h, const mynah_b200_kv_batch *b, const void *q, long long ldq, const void *k, long long ldk,
                         const void *v, long long ldv, void *q_out, long long ldqo, void *stream) {
    if (!h || !b) { set_error("kv_append: bad argument"); return -1; }
    OnDevice on(h->device);
    KvAppendArgs p = {};
    const int go = take_batch("kv_append", h, b, &p.a);
    if (go) return go < 0 ? -1 : 0;
    const int D = p.a.D;
    const char *no = refuse_rows(h, q, ldq, p.a.H * D);
    if (!no) no = refuse_rows(h, k, ldk, p.a.Hkv * D);
    if (!no) no = refuse_rows(h, v, ldv, p.a.Hkv * D);
    if (!no) no = refuse_rows(h, q_out, ldqo, p.a.H * D);
    const int n = p.a.n_rows, size = row_bytes(h->fmt);
    if (!no && (clash(q_out, ldqo, p.a.H * D, q, ldq, p.a.H * D, n, size) || clash(q_out, ldqo, p.a.H * D, k, ldk, p.a.Hkv * D, n, size) ||
                clash(q_out, ldqo, p.a.H * D, v, ldv, p.a.Hkv * D, n, size)))
        no = "q_out overlaps rows that are read";
    if (no) { set_error("kv_append: %s", no); return -1; }
    p.a.q = q; p.a.ldq = ldq; p.a.out = q_out; p.a.ldo = ldqo;
    p.k_rows = k; p.ldk = ldk; p.v_rows = v; p.ldv = ldv;
    p.q_norm = h->q_norm; p.k_norm = h->k_norm; p.eps = h->cfg.norm_eps;
    p.turns = h->turns; p.rot = h->cfg.rotary_dim; p.interleaved = h->cfg.rotary_interleaved != 0;
    return kv_append(p, h->fmt, stream ? (cudaStream_t)stream : h->stream);
}

int mynah_b200_kv_attend(mynah_b200_kv *h, const mynah_b200_kv_batch *b, const void *q, long long ldq, void *out, long long ldo,
                         void *stream) {
    if (!h || !b) { set_error("kv_attend: bad argument"); return -1; }
    OnDevice on(h->device);
    KvArgs a = {};
    const int go = take_batch("kv_attend", h, b, &a);
    if (go) return go < 0 ? -1 : 0;
    const char *no = refuse_rows(h, q, ldq, a.H * a.D);
    if (!no) no = refuse_rows(h, out, ldo, a.H * a.D);
    if (!no && clash(out, ldo, a.H * a.D, q, ldq, a.H * a.D, a.n_rows, row_bytes(h->fmt))) no = "out overlaps rows that are read";
    if (no) { set_error("kv_attend: %s", no); return -1; }
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo;
    const cudaStream_t st = stream ? (cudaStream_t)stream : h->stream;
    return a.row_off ? kv_chunk(h->chunk_k, h->chunk_v, a, h->chunk_box, h->fmt, st) : kv_step(h->map_k, h->map_v, a, h->fmt, st);
}

int mynah_b200_kv_sync(mynah_b200_kv *h, void *stream) {
    if (!h) { set_error("kv_sync: null handle"); return -1; }
    OnDevice on(h->device);
    RelaxedCapture relaxed;                                    // (waits and copies)
    const cudaStream_t st = stream ? (cudaStream_t)stream : h->stream;
    MB_CUDA(cudaStreamSynchronize(st));
    // Read and cleared in one step: calls on other streams may be reporting at the same time
    std::lock_guard<std::mutex> one(h->syncing);
    int found = 0;
    MB_CUDA(launch_kernel(kv_take_kernel, dim3(1), dim3(1), 0, h->stream, false, 1, h->status(), h->taken(), h->owed ? 1 : 0));
    h->owed = true;
    MB_CUDA(cudaMemcpyAsync(&found, h->taken(), sizeof(int), cudaMemcpyDeviceToHost, h->stream));
    MB_CUDA(cudaStreamSynchronize(h->stream));
    h->owed = false;
    if (found == 0) return 0;
    const int waits = found & (1 << ST_TIMEOUT_PRODUCER | 1 << ST_TIMEOUT_MMA | 1 << ST_TIMEOUT_EPILOGUE);
    char text[3][160] = {"", "", ""};
    if (waits) snprintf(text[0], sizeof(text[0]), " a bounded wait inside an attention kernel ran out (code %d);", __builtin_ctz((unsigned)waits));
    if (found & 1 << ST_PAGE) snprintf(text[1], sizeof(text[1]), " a table names a page, a length or a row that does not exist;");
    if (found & 1 << ST_RANGE)
        snprintf(text[2], sizeof(text[2]), " a value did not fit its 16 bits (f16: 65504), or a value or a score was not finite;");
    char all[480];
    const int n = snprintf(all, sizeof(all), "%s%s%s", text[0], text[1], text[2]);
    set_error("kv:%.*s", n - 1, all);
    return -1;
}

}  // extern "C"
