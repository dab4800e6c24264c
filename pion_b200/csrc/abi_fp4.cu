// C-ABI entry points of microscaled 4-bit rows: a store written, read back, multiplied with
// query batches and searched (fp4_rows.cu, flat_fp4.cu).  No counterpart in the reference.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdlib>

#include "fp4.cuh"
#include "internal.h"

using namespace pion;

namespace {

constexpr int64_t kMaxRows = (int64_t)INT32_MAX - 256;  // slots are 32-bit TMA coordinates
constexpr int64_t kMaxK = 256;
constexpr int64_t kMaxQueries = 1 << 24;
constexpr int64_t kQueryChunk = 4096;  // queries searched at once: bounds the scratch (64 KB each)
int elem_bytes(int type) { return type == PION_B200_F32 ? 4 : 2; }
bool type_ok(int type) { return type >= PION_B200_F32 && type <= PION_B200_F16; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int sizes(int format, int64_t n_rows, int64_t dim, int64_t* codes, int64_t* scales) {
    if (format != PION_B200_FP4_MX && format != PION_B200_FP4_NV) return PION_B200_EINVAL;
    if (n_rows < 0) return PION_B200_EINVAL;
    if (n_rows > kMaxRows || dim < 1 || dim > fp4_max_dim()) return PION_B200_ESHAPE;
    const int dp = fp4::pad_dim((int)dim);
    *codes = n_rows * (dp / 2);
    *scales = (n_rows + 127) / 128 * fp4::atoms_of(format, dp) * 512;
    return 0;
}

int check_rows(pion_b200_ctx* ctx, const pion_b200_fp4_rows* r, const char* who) {
    if (!r) return set_error(ctx, PION_B200_EINVAL, "%s: null store", who);
    int64_t c, s;
    if (int rc = sizes(r->format, r->n_rows, r->dim, &c, &s))
        return set_error(ctx, rc, "%s: unsupported store (format %d, %lld rows, dim %lld; dim <= %d)",
                         who, r->format, (long long)r->n_rows, (long long)r->dim, fp4_max_dim());
    if (r->n_rows > 0 && (!r->codes || !r->scales || !r->row_scale || !r->norm_max))
        return set_error(ctx, PION_B200_EINVAL, "%s: null buffer in the store", who);
    if (!aligned(r->codes, 16) || !aligned(r->scales, 16) || !aligned(r->row_scale, 4) ||
        !aligned(r->norm_max, 4) || !aligned(r->claim, 4))
        return set_error(ctx, PION_B200_EINVAL, "%s: misaligned buffer in the store", who);
    return 0;
}

// Rows [0, n) of `dim` elements `stride` apart: the elements they span.
int64_t span(int64_t n, int64_t stride, int64_t dim) { return n > 0 ? (n - 1) * stride + dim : 0; }

int check_matrix(pion_b200_ctx* ctx, const char* who, const char* what, const void* p, int type,
                 int64_t n, int64_t stride, int64_t dim) {
    if (!type_ok(type)) return set_error(ctx, PION_B200_EINVAL, "%s: %s of unknown type %d", who, what, type);
    if (n < 0) return set_error(ctx, PION_B200_EINVAL, "%s: negative number of rows", who);
    if (n > 0 && !p) return set_error(ctx, PION_B200_EINVAL, "%s: null %s", who, what);
    if (n > 0 && stride < dim)
        return set_error(ctx, PION_B200_EINVAL, "%s: %s rows overlap (stride %lld, %lld elements)", who,
                         what, (long long)stride, (long long)dim);
    if (n > 1 && stride > INT64_MAX / 8 / n)
        return set_error(ctx, PION_B200_EINVAL, "%s: %s rows past 64 bits (stride %lld)", who, what,
                         (long long)stride);
    if (!aligned(p, elem_bytes(type)))
        return set_error(ctx, PION_B200_EINVAL, "%s: misaligned %s", who, what);
    return 0;
}

int check_mem(pion_b200_ctx* ctx, const char* who, int mem) {
    if (mem != PION_B200_MEM_HOST && mem != PION_B200_MEM_DEVICE)
        return set_error(ctx, PION_B200_EINVAL, "%s: mem %d", who, mem);
    return 0;
}

// The scratch of a scores or knn call of at most `nq` queries at once.
struct Scratch {
    size_t q_codes, q_scales, q_scale, q_norm, theta, cand_n, n_flagged, flagged, done, parts, sample,
        cand, total;
    Fp4Plan plan;
};

bool plan_scratch(int format, int dim, int64_t n_rows, int64_t nq, int64_t k, Scratch* out) {
    const int dp = fp4::pad_dim(dim);
    Scratch s;
    if (!fp4_plan(format, dp, (int)nq, n_rows, &s.plan)) return false;
    const size_t slots = (size_t)s.plan.n_qt * s.plan.nt_pad;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t o = off;
        off += align_up(bytes, 256);
        return o;
    };
    s.q_codes = take(slots * (dp / 2));
    s.q_scales = take(slots / 128 * fp4::atoms_of(format, dp) * 512);
    s.q_scale = take(slots * 4);
    s.q_norm = take((size_t)nq * 4);
    s.theta = s.cand_n = s.n_flagged = s.flagged = s.done = s.parts = s.sample = s.cand = 0;
    if (k > 0) {
        const bool split = fp4_splits(nq, n_rows, k);
        const int64_t most = split ? (n_rows + 3) / 4 * 4
                                   : (int64_t)fp4_sample_tiles((int)nq) * fp4_tile_rows();
        s.theta = take((size_t)nq * 4);
        s.n_flagged = take((size_t)(nq + 1) * 4);
        s.cand_n = s.n_flagged + 4;
        s.flagged = take((size_t)nq * 4);
        s.done = take((size_t)nq * 4);
        s.parts = take((size_t)fp4_rescue_items(nq) * k * 8);
        s.sample = take((size_t)nq * (n_rows < most && !split ? n_rows : most) * 4);
        if (split || n_rows > most) s.cand = take((size_t)nq * fp4_cap() * 8);
    }
    s.total = off;
    *out = s;
    return true;
}

int64_t workspace(const pion_b200_fp4_rows* r, int64_t n_rows, int64_t nq, int64_t k) {
    if (!r || n_rows < 0 || nq < 0 || k < 0) return PION_B200_EINVAL;
    int64_t c, b;
    if (int rc = sizes(r->format, r->n_rows, r->dim, &c, &b)) return rc;
    if (n_rows > r->n_rows || nq > kMaxQueries || k > kMaxK) return PION_B200_ESHAPE;
    if (nq == 0 || n_rows == 0) return 0;
    // The last chunk of queries may be smaller, with another plan.
    int64_t most = 0;
    const int64_t first = k > 0 && nq > kQueryChunk ? kQueryChunk : nq;
    for (int64_t n : {first, k > 0 ? nq % kQueryChunk : 0}) {
        Scratch s;
        if (n == 0) continue;
        if (!plan_scratch(r->format, (int)r->dim, n_rows, n, k, &s)) return PION_B200_ESHAPE;
        most = (int64_t)s.total > most ? (int64_t)s.total : most;
    }
    return most;
}

// Runs a device-memory call on the caller's stream.
struct StreamScope {
    pion_b200_ctx* ctx;
    cudaStream_t before;
    StreamScope(pion_b200_ctx* c, void* stream, int mem) : ctx(c), before(c->stream) {
        if (stream && mem == PION_B200_MEM_DEVICE) c->stream = static_cast<cudaStream_t>(stream);
    }
    ~StreamScope() { ctx->stream = before; }
    bool own() const { return ctx->stream != before; }
};

// The caller's workspace, or on the context's own stream its scratch.
int take_workspace(pion_b200_ctx* ctx, const char* who, int64_t need, void* ws, int64_t bytes,
                   bool own_stream, char** out) {
    if (need == 0) return 0;
    if (ws) {
        if (bytes < need || !aligned(ws, 16))
            return set_error(ctx, PION_B200_EINVAL, "%s: workspace of %lld bytes, need %lld (16-byte aligned)",
                             who, (long long)bytes, (long long)need);
        *out = static_cast<char*>(ws);
        return 0;
    }
    if (own_stream || stream_capturing(ctx->stream))
        return set_error(ctx, PION_B200_EINVAL,
                         "%s: a call on a stream of its own, or captured, needs a workspace", who);
    if (ensure(ctx->scratch, (size_t)need) != 0)
        return set_error(ctx, PION_B200_ENOMEM, "%s: %lld bytes of scratch", who, (long long)need);
    *out = static_cast<char*>(ctx->scratch.ptr);
    return 0;
}

int no_host_capture(pion_b200_ctx* ctx, const char* who, int mem) {
    if (mem == PION_B200_MEM_HOST && stream_capturing(ctx->stream))
        return set_error(ctx, PION_B200_EINVAL, "%s: host memory cannot be captured", who);
    return 0;
}

// Host rows into the context's staging buffer, `extra` bytes of room behind them.
int stage_rows(pion_b200_ctx* ctx, const char* who, const void* src, size_t bytes, size_t extra,
               char** out) {
    if (ensure(ctx->stage_in, align_up(bytes, 256) + extra) != 0)
        return set_error(ctx, PION_B200_ENOMEM, "%s: staging", who);
    *out = static_cast<char*>(ctx->stage_in.ptr);
    if (cudaMemcpyAsync(*out, src, bytes, cudaMemcpyHostToDevice, ctx->stream) != cudaSuccess)
        return set_error(ctx, PION_B200_ECUDA, "%s: input copy failed", who);
    return 0;
}

// The call's queries, quantised into its scratch.
int quantise_queries(pion_b200_ctx* ctx, const pion_b200_fp4_rows* r, const void* q, int type,
                     int64_t stride, int64_t nq, const Scratch& s, char* base, int64_t k) {
    Fp4Write w;
    w.format = r->format;
    w.dim = (int)r->dim;
    w.src = q;
    w.type = type;
    w.stride = stride;
    w.n = nq;
    w.tile = s.plan.nt;
    w.tile_pad = s.plan.nt_pad;
    w.codes = reinterpret_cast<uint8_t*>(base + s.q_codes);
    w.scales = reinterpret_cast<uint8_t*>(base + s.q_scales);
    w.row_scale = reinterpret_cast<float*>(base + s.q_scale);
    w.norm = reinterpret_cast<float*>(base + s.q_norm);
    if (k > 0) w.zero = reinterpret_cast<int*>(base + s.n_flagged);
    ctx->launches++;
    return launch_fp4_write(w, ctx->stream);
}

Fp4Product product_of(pion_b200_ctx* ctx, const pion_b200_fp4_rows* r, int64_t n_rows, int64_t nq,
                      const Scratch& s, char* base, int mem) {
    Fp4Product L;
    L.format = r->format;
    L.dim = (int)r->dim;
    L.codes = r->codes;
    L.scales = r->scales;
    L.row_scale = r->row_scale;
    L.store_rows = r->n_rows;
    L.n_rows = n_rows;
    L.q_codes = reinterpret_cast<uint8_t*>(base + s.q_codes);
    L.q_scales = reinterpret_cast<uint8_t*>(base + s.q_scales);
    L.q_scale = reinterpret_cast<float*>(base + s.q_scale);
    L.nq = (int)nq;
    L.status = call_status(ctx, mem);
    L.wait_ns = ctx->wait_ns;
    L.test_stall = test_stall();
    L.num_sms = ctx->num_sms;
    return L;
}

// One chunk of queries: the candidates of each -- from the scores of every row where those are
// few, else the rows that reach a threshold taken from a sample of them and tightened over
// growing parts -- then the k best of those exactly.
int knn_chunk(pion_b200_ctx* ctx, const pion_b200_fp4_rows* r, int64_t n_rows, int64_t id_base,
              const void* q, int q_type, int64_t q_stride, int64_t nq, int64_t k, int32_t* ids,
              float* scores, const Scratch& s, char* base, int mem) {
    cudaStream_t st = ctx->stream;
    float* theta = reinterpret_cast<float*>(base + s.theta);
    int* cand_n = reinterpret_cast<int*>(base + s.cand_n);
    float* sample = reinterpret_cast<float*>(base + s.sample);
    uint64_t* cand = reinterpret_cast<uint64_t*>(base + s.cand);
    const float* q_scale = reinterpret_cast<const float*>(base + s.q_scale);
    const float* q_norm = reinterpret_cast<const float*>(base + s.q_norm);
    int rc = quantise_queries(ctx, r, q, q_type, q_stride, nq, s, base, k);
    if (rc != 0) return rc;

    const int64_t n_tiles = (n_rows + fp4_tile_rows() - 1) / fp4_tile_rows();
    const int samples = fp4_sample_tiles((int)nq);
    const bool split = fp4_splits(nq, n_rows, k);
    const bool dense = !split && n_tiles <= samples;
    const int64_t m = split   ? (n_rows + 3) / 4 * 4
                      : dense ? n_rows
                              : (int64_t)samples * fp4_tile_rows();
    timing_begin(ctx);
    Fp4Product L = product_of(ctx, r, n_rows, nq, s, base, mem);
    L.n_tiles = (int)(split || dense ? n_tiles : samples);
    L.tile_step = split || dense ? 1 : (int)(n_tiles / samples);
    L.out = sample;
    L.out_type = PION_B200_F32;
    L.ld = m;
    rc = launch_fp4_product(L, st);
    ctx->launches++;
    if (split && rc == 0) {
        rc = launch_fp4_split(sample, m, n_rows, (int)k, (int)r->dim, q_scale, s.plan.nt,
                              s.plan.nt_pad, q_norm, r->norm_max, (int)nq, cand, cand_n, st);
        ctx->launches++;
    } else if (!dense && rc == 0) {
        rc = launch_fp4_theta(sample, nullptr, (int)k, (int)r->dim, q_scale, s.plan.nt,
                              s.plan.nt_pad, q_norm, r->norm_max, (int)nq, theta, cand_n, st);
        ctx->launches++;
        L.theta = theta;
        L.cand_n = cand_n;
        L.cand = cand;
        // Stages over growing parts of the rows, each with the threshold of the rows before it:
        // every R^(L-1)-th tile, then those of every R^(L-2)-th that are new, and so on.  About
        // k R rows of the first stage and k (R - 1) of each later one reach their threshold,
        // with a deviation of 1 / sqrt(k) of that: the lists have room for 13 deviations.  A
        // batch takes more stages, since its candidates cost the product's epilogue more than
        // a stage costs.
        const double ratio = (double)n_tiles / (double)samples;
        const double room = fp4_cap() / ((double)k + 13.0 * sqrt((double)k));
        int stages = 1;
        int64_t grow = 0;
        for (;; ++stages) {
            grow = (int64_t)ceil(pow(ratio, 1.0 / stages));
            if (grow < 2) grow = 2;
            if ((double)(grow + (stages - 1) * (grow - 1)) <= room && (nq <= 64 || grow <= 12)) break;
            if (grow == 2) break;
        }
        int64_t step = 1;
        for (int i = 1; i < stages; ++i) step *= grow;
        for (int i = 0; i < stages && rc == 0; ++i) {
            if (i > 0) {
                rc = launch_fp4_theta(nullptr, cand, (int)k, (int)r->dim, q_scale, s.plan.nt,
                                      s.plan.nt_pad, q_norm, r->norm_max, (int)nq, theta, cand_n,
                                      st);
                ctx->launches++;
                if (rc != 0) break;
                step /= grow;
            }
            const int64_t tiles = (n_tiles + step - 1) / step;
            const int64_t before = i > 0 ? (n_tiles + step * grow - 1) / (step * grow) : 0;
            if (tiles == before) continue;
            L.tile_step = (int)step;
            L.tile_skip = i > 0 ? (int)grow : 0;
            L.n_tiles = (int)(tiles - before);
            rc = launch_fp4_product(L, st);
            ctx->launches++;
        }
    }
    timing_end(ctx);
    if (rc != 0) return rc;
    Fp4Finish f;
    f.format = r->format;
    f.dim = (int)r->dim;
    f.codes = r->codes;
    f.scales = r->scales;
    f.row_scale = r->row_scale;
    f.norm_max = r->norm_max;
    f.n_rows = n_rows;
    f.id_base = id_base;
    f.q_codes = L.q_codes;
    f.q_scales = L.q_scales;
    f.q_scale = q_scale;
    f.q_norm = q_norm;
    f.nt = s.plan.nt;
    f.nt_pad = s.plan.nt_pad;
    f.nq = (int)nq;
    f.k = (int)k;
    f.dense = dense ? sample : nullptr;
    f.ld = m;
    f.cand_n = cand_n;
    f.cand = cand;
    f.n_flagged = reinterpret_cast<int*>(base + s.n_flagged);
    f.flagged = reinterpret_cast<int*>(base + s.flagged);
    f.done = reinterpret_cast<int*>(base + s.done);
    f.parts = reinterpret_cast<uint64_t*>(base + s.parts);
    f.out_ids = ids;
    f.out_scores = scores;
    ctx->launches += dense ? 1 : 2;
    return launch_fp4_finish(f, st);
}

}  // namespace

extern "C" {

int pion_v_b200_fp4_sizes(int format, int64_t n_rows, int64_t dim, int64_t* codes_bytes,
                          int64_t* scales_bytes) {
    if (!codes_bytes || !scales_bytes) return PION_B200_EINVAL;
    return sizes(format, n_rows, dim, codes_bytes, scales_bytes);
}

int pion_v_b200_fp4_clear(pion_b200_ctx* ctx, const pion_b200_fp4_rows* rows,
                          void* cuda_stream) {
    if (!valid_ctx(ctx)) return PION_B200_EINVAL;
    if (int rc = check_rows(ctx, rows, "fp4_clear")) return rc;
    if (rows->n_rows == 0) return 0;
    StreamScope scope(ctx, cuda_stream, PION_B200_MEM_DEVICE);
    if (int rc = use_device(ctx)) return rc;
    int64_t c, s;
    sizes(rows->format, rows->n_rows, rows->dim, &c, &s);
    cudaStream_t st = ctx->stream;
    const size_t n = (size_t)rows->n_rows;
    // 0xffffffff is a NaN
    if (cudaMemsetAsync(rows->codes, 0, (size_t)c, st) != cudaSuccess ||
        cudaMemsetAsync(rows->scales, 0, (size_t)s, st) != cudaSuccess ||
        cudaMemsetAsync(rows->row_scale, 0xff, n * 4, st) != cudaSuccess ||
        cudaMemsetAsync(rows->norm_max, 0, 4, st) != cudaSuccess ||
        (rows->claim && cudaMemsetAsync(rows->claim, 0, n * 4, st) != cudaSuccess))
        return set_error(ctx, PION_B200_ECUDA, "fp4_clear: %s", cudaGetErrorString(cudaGetLastError()));
    return 0;
}

int pion_v_b200_fp4_write(pion_b200_ctx* ctx, const pion_b200_fp4_rows* rows, const void* src,
                          int type, int64_t stride, int64_t n, const int64_t* slots,
                          int64_t start, int mem, void* cuda_stream) {
    const char* who = "fp4_write";
    if (!valid_ctx(ctx)) return PION_B200_EINVAL;
    if (int rc = check_rows(ctx, rows, who)) return rc;
    if (int rc = check_mem(ctx, who, mem)) return rc;
    if (int rc = check_matrix(ctx, who, "rows", src, type, n, stride, rows->dim)) return rc;
    if (n > kMaxRows) return set_error(ctx, PION_B200_ESHAPE, "%s: %lld rows", who, (long long)n);
    if (n == 0) return 0;
    if (slots && !rows->claim)
        return set_error(ctx, PION_B200_EINVAL, "%s: slots need the store's claim buffer", who);
    if (!slots && (start < 0 || start > rows->n_rows - n))
        return set_error(ctx, PION_B200_EINVAL, "%s: rows [%lld, %lld) of a store of %lld", who,
                         (long long)start, (long long)(start + n), (long long)rows->n_rows);
    if (slots && mem == PION_B200_MEM_HOST)
        for (int64_t i = 0; i < n; ++i)
            if (slots[i] >= rows->n_rows)
                return set_error(ctx, PION_B200_EINVAL, "%s: slot %lld of a store of %lld", who,
                                 (long long)slots[i], (long long)rows->n_rows);
    if (slots && !aligned(slots, 8)) return set_error(ctx, PION_B200_EINVAL, "%s: misaligned slots", who);
    if (int rc = use_device(ctx)) return rc;
    StreamScope scope(ctx, cuda_stream, mem);
    if (int rc = no_host_capture(ctx, who, mem)) return rc;
    Fp4Write w;
    w.format = rows->format;
    w.dim = (int)rows->dim;
    w.src = src;
    w.type = type;
    w.stride = stride;
    w.n = n;
    w.slots = slots;
    w.start = start;
    w.n_slots = rows->n_rows;
    w.claim = rows->claim;
    w.codes = rows->codes;
    w.scales = rows->scales;
    w.row_scale = rows->row_scale;
    w.norm_max = rows->norm_max;
    w.status = call_status(ctx, mem);
    if (mem == PION_B200_MEM_HOST) {
        const size_t bytes = (size_t)span(n, stride, rows->dim) * elem_bytes(type);
        char* dev;
        if (int rc = stage_rows(ctx, who, src, bytes, slots ? (size_t)n * 8 : 0, &dev)) return rc;
        w.src = dev;
        if (slots) {
            int64_t* ds = reinterpret_cast<int64_t*>(dev + align_up(bytes, 256));
            if (cudaMemcpyAsync(ds, slots, (size_t)n * 8, cudaMemcpyHostToDevice, ctx->stream) !=
                cudaSuccess)
                return set_error(ctx, PION_B200_ECUDA, "%s: slots copy failed", who);
            w.slots = ds;
        }
    }
    ctx->launches += fp4_write_launches(slots != nullptr, n);
    if (int rc = launch_fp4_write(w, ctx->stream))
        return set_error(ctx, rc, "%s: launch failed: %s", who, cudaGetErrorString(cudaGetLastError()));
    return mem == PION_B200_MEM_HOST ? finish_sync(ctx) : 0;
}

int pion_v_b200_fp4_read(pion_b200_ctx* ctx, const pion_b200_fp4_rows* rows, const int64_t* slots,
                         int64_t start, int64_t n, void* dst, int type, int64_t stride, int mem,
                         void* cuda_stream) {
    const char* who = "fp4_read";
    if (!valid_ctx(ctx)) return PION_B200_EINVAL;
    if (int rc = check_rows(ctx, rows, who)) return rc;
    if (int rc = check_mem(ctx, who, mem)) return rc;
    if (int rc = check_matrix(ctx, who, "output", dst, type, n, stride, rows->dim)) return rc;
    if (n > kMaxRows) return set_error(ctx, PION_B200_ESHAPE, "%s: %lld rows", who, (long long)n);
    if (n == 0) return 0;
    if (!slots && (start < 0 || start > rows->n_rows - n))
        return set_error(ctx, PION_B200_EINVAL, "%s: rows [%lld, %lld) of a store of %lld", who,
                         (long long)start, (long long)(start + n), (long long)rows->n_rows);
    if (slots && !aligned(slots, 8)) return set_error(ctx, PION_B200_EINVAL, "%s: misaligned slots", who);
    if (slots && mem == PION_B200_MEM_HOST)
        for (int64_t i = 0; i < n; ++i)
            if (slots[i] < 0 || slots[i] >= rows->n_rows)
                return set_error(ctx, PION_B200_EINVAL, "%s: slot %lld of a store of %lld", who,
                                 (long long)slots[i], (long long)rows->n_rows);
    if (int rc = use_device(ctx)) return rc;
    StreamScope scope(ctx, cuda_stream, mem);
    if (int rc = no_host_capture(ctx, who, mem)) return rc;
    Fp4Read r;
    r.format = rows->format;
    r.dim = (int)rows->dim;
    r.codes = rows->codes;
    r.scales = rows->scales;
    r.row_scale = rows->row_scale;
    r.n_slots = rows->n_rows;
    r.slots = slots;
    r.start = start;
    r.n = n;
    r.dst = dst;
    r.type = type;
    r.stride = stride;
    r.status = call_status(ctx, mem);
    const int es = elem_bytes(type);
    if (mem == PION_B200_MEM_HOST) {
        if (ensure(ctx->stage_out, (size_t)n * rows->dim * es) != 0)
            return set_error(ctx, PION_B200_ENOMEM, "%s: staging", who);
        r.dst = ctx->stage_out.ptr;
        r.stride = rows->dim;
        if (slots) {
            char* ds;
            if (int rc = stage_rows(ctx, who, slots, (size_t)n * 8, 0, &ds)) return rc;
            r.slots = reinterpret_cast<int64_t*>(ds);
        }
    }
    ctx->launches++;
    if (int rc = launch_fp4_read(r, ctx->stream))
        return set_error(ctx, rc, "%s: launch failed: %s", who, cudaGetErrorString(cudaGetLastError()));
    if (mem != PION_B200_MEM_HOST) return 0;
    if (cudaMemcpy2DAsync(dst, (size_t)stride * es, r.dst, (size_t)rows->dim * es,
                          (size_t)rows->dim * es, (size_t)n, cudaMemcpyDeviceToHost,
                          ctx->stream) != cudaSuccess)
        return set_error(ctx, PION_B200_ECUDA, "%s: output copy failed", who);
    return finish_sync(ctx);
}

int64_t pion_v_b200_fp4_workspace(const pion_b200_fp4_rows* rows, int64_t n_rows, int64_t nq,
                                  int64_t k) {
    return workspace(rows, n_rows, nq, k);
}

int pion_v_b200_fp4_scores(pion_b200_ctx* ctx, const pion_b200_fp4_rows* rows, int64_t n_rows,
                           const void* q, int q_type, int64_t q_stride, int64_t nq, void* out,
                           int out_type, int64_t out_stride, void* workspace_ptr,
                           int64_t workspace_bytes, int mem, void* cuda_stream) {
    const char* who = "fp4_scores";
    if (!valid_ctx(ctx)) return PION_B200_EINVAL;
    if (int rc = check_rows(ctx, rows, who)) return rc;
    if (int rc = check_mem(ctx, who, mem)) return rc;
    if (n_rows < 0 || n_rows > rows->n_rows)
        return set_error(ctx, PION_B200_EINVAL, "%s: %lld rows of a store of %lld", who,
                         (long long)n_rows, (long long)rows->n_rows);
    if (int rc = check_matrix(ctx, who, "queries", q, q_type, nq, q_stride, rows->dim)) return rc;
    if (nq > kMaxQueries) return set_error(ctx, PION_B200_ESHAPE, "%s: %lld queries", who, (long long)nq);
    if (nq == 0 || n_rows == 0) return 0;
    if (int rc = check_matrix(ctx, who, "output", out, out_type, nq, out_stride, n_rows)) return rc;
    const int64_t need = workspace(rows, n_rows, nq, 0);
    if (need < 0) return set_error(ctx, (int)need, "%s: unsupported shape", who);
    if (int rc = use_device(ctx)) return rc;
    StreamScope scope(ctx, cuda_stream, mem);
    if (int rc = no_host_capture(ctx, who, mem)) return rc;
    const bool host = mem == PION_B200_MEM_HOST;
    char* base = nullptr;
    if (int rc = take_workspace(ctx, who, need, host ? nullptr : workspace_ptr, workspace_bytes,
                                scope.own(), &base))
        return rc;
    Scratch s;
    plan_scratch(rows->format, (int)rows->dim, n_rows, nq, 0, &s);
    const void* dq = q;
    if (host) {
        char* dev;
        if (int rc = stage_rows(ctx, who, q, (size_t)span(nq, q_stride, rows->dim) * elem_bytes(q_type),
                                0, &dev))
            return rc;
        dq = dev;
        if (ensure(ctx->stage_out, (size_t)nq * n_rows * elem_bytes(out_type)) != 0)
            return set_error(ctx, PION_B200_ENOMEM, "%s: staging", who);
    }
    int rc = quantise_queries(ctx, rows, dq, q_type, q_stride, nq, s, base, 0);
    if (rc == 0) {
        Fp4Product L = product_of(ctx, rows, n_rows, nq, s, base, mem);
        L.out = host ? ctx->stage_out.ptr : out;
        L.out_type = out_type;
        L.ld = host ? n_rows : out_stride;
        timing_begin(ctx);
        rc = launch_fp4_product(L, ctx->stream);
        timing_end(ctx);
        ctx->launches++;
    }
    if (rc != 0)
        return set_error(ctx, rc, "%s: launch failed: %s", who, cudaGetErrorString(cudaGetLastError()));
    if (!host) return 0;
    const size_t es = elem_bytes(out_type);
    if (cudaMemcpy2DAsync(out, (size_t)out_stride * es, ctx->stage_out.ptr, (size_t)n_rows * es,
                          (size_t)n_rows * es, (size_t)nq, cudaMemcpyDeviceToHost,
                          ctx->stream) != cudaSuccess)
        return set_error(ctx, PION_B200_ECUDA, "%s: output copy failed", who);
    return finish_sync(ctx);
}

int pion_v_b200_flat_fp4_knn(pion_b200_ctx* ctx, const pion_b200_fp4_rows* rows, int64_t n_rows,
                             int64_t id_base, const void* q, int q_type, int64_t q_stride,
                             int64_t nq, int64_t k, int32_t* out_ids, float* out_scores,
                             void* workspace_ptr, int64_t workspace_bytes, int mem, void* cuda_stream) {
    const char* who = "flat_fp4_knn";
    if (!valid_ctx(ctx)) return PION_B200_EINVAL;
    if (int rc = check_rows(ctx, rows, who)) return rc;
    if (int rc = check_mem(ctx, who, mem)) return rc;
    if (n_rows < 0 || n_rows > rows->n_rows)
        return set_error(ctx, PION_B200_EINVAL, "%s: %lld rows of a store of %lld", who,
                         (long long)n_rows, (long long)rows->n_rows);
    if (int rc = check_matrix(ctx, who, "queries", q, q_type, nq, q_stride, rows->dim)) return rc;
    if (k < 1 || k > kMaxK || nq > kMaxQueries)
        return set_error(ctx, PION_B200_ESHAPE, "%s: k %lld (1 to %lld), %lld queries", who,
                         (long long)k, (long long)kMaxK, (long long)nq);
    if (id_base < 0 || id_base > INT32_MAX - n_rows)
        return set_error(ctx, PION_B200_EINVAL, "%s: ids past 32 bits (id_base %lld)", who,
                         (long long)id_base);
    if (nq == 0) return 0;
    if (!out_ids || !out_scores || !aligned(out_ids, 4) || !aligned(out_scores, 4))
        return set_error(ctx, PION_B200_EINVAL, "%s: null or misaligned output", who);
    const int64_t need = workspace(rows, n_rows, nq, k);
    if (need < 0) return set_error(ctx, (int)need, "%s: unsupported shape", who);
    if (int rc = use_device(ctx)) return rc;
    StreamScope scope(ctx, cuda_stream, mem);
    if (int rc = no_host_capture(ctx, who, mem)) return rc;
    const bool host = mem == PION_B200_MEM_HOST;
    char* base = nullptr;
    if (int rc = take_workspace(ctx, who, need, host ? nullptr : workspace_ptr, workspace_bytes,
                                scope.own(), &base))
        return rc;
    cudaStream_t st = ctx->stream;
    const size_t out_bytes = (size_t)nq * k * 4;
    const char* dq = static_cast<const char*>(q);
    int32_t* di = out_ids;
    float* dv = out_scores;
    if (host) {
        char* dev;
        if (int rc = stage_rows(ctx, who, q, (size_t)span(nq, q_stride, rows->dim) * elem_bytes(q_type),
                                0, &dev))
            return rc;
        dq = dev;
        if (ensure(ctx->stage_out, 2 * align_up(out_bytes, 256)) != 0)
            return set_error(ctx, PION_B200_ENOMEM, "%s: staging", who);
        di = static_cast<int32_t*>(ctx->stage_out.ptr);
        dv = reinterpret_cast<float*>(static_cast<char*>(ctx->stage_out.ptr) + align_up(out_bytes, 256));
    }
    int rc = 0;
    if (n_rows == 0) {
        rc = launch_fill_results(dv, di, (size_t)nq * k, -INFINITY, st);
        ctx->launches++;
    }
    for (int64_t t = 0; t < nq && rc == 0 && n_rows > 0; t += kQueryChunk) {
        const int64_t n = nq - t < kQueryChunk ? nq - t : kQueryChunk;
        Scratch s;
        plan_scratch(rows->format, (int)rows->dim, n_rows, n, k, &s);
        rc = knn_chunk(ctx, rows, n_rows, id_base, dq + t * q_stride * elem_bytes(q_type), q_type,
                       q_stride, n, k, di + t * k, dv + t * k, s, base, mem);
    }
    if (rc != 0)
        return set_error(ctx, rc, "%s: launch failed: %s", who, cudaGetErrorString(cudaGetLastError()));
    if (!host) return 0;
    if (cudaMemcpyAsync(out_ids, di, out_bytes, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaMemcpyAsync(out_scores, dv, out_bytes, cudaMemcpyDeviceToHost, st) != cudaSuccess)
        return set_error(ctx, PION_B200_ECUDA, "%s: result copy failed", who);
    return finish_sync(ctx);
}

}  // extern "C"
