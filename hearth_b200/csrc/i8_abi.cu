// Entry points of the 8-bit linear path (include/hb200.h, section "8-bit linear path"): resident int8 weights with a scale
// per row, activation planes with a scale per token, their producers and the product.  Kernels in i8_quant.cu and
// i8_gemm.cu.  Errors never cross the boundary as exceptions.
#include <cuda.h>

#include <cfloat>
#include <new>
#include <vector>

#include "../../include/hb200.h"
#include "common.cuh"

using namespace hb200;

struct hb200_weight_i8 {
    int slot = 0, device = 0;
    size_t n_rows = 0, n_cols = 0;
    int kb = 0;
    I8Plane plane = {};
    float* scales = nullptr;
    size_t resident_bytes = 0;
    CUtensorMap map;  // one 128-row tile of one block
};
struct hb200_act_i8 {
    int slot = 0, device = 0;
    size_t max_seq = 0, n_cols = 0;
    int kb = 0;
    I8Plane plane = {};
    float* scales = nullptr;
    CUtensorMap map64, map128;  // 64 and 128 tokens of one block
};

namespace {

// Inside a call the object's slot is the current one and the calling thread is on its device; afterwards both are what
// they were (one without the other would have the next object created on a device that is not its slot's).
struct DeviceScope {
    int prev = -1, prev_slot;
    int rc = 0;
    explicit DeviceScope(int slot) : prev_slot(current_slot()) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        rc = use_slot_of(slot);
        if (rc) return;
        if (prev == bound_device()) return;  // (use_slot_of may have switched, never away from the slot's device)
        const cudaError_t e = cudaSetDevice(bound_device());
        if (e != cudaSuccess) {
            set_error("cudaSetDevice(%d) failed: %s", bound_device(), cudaGetErrorString(e));
            rc = HB200_ERR_CUDA;
        }
    }
    ~DeviceScope() {
        if (prev >= 0 && prev != bound_device()) cudaSetDevice(prev);
        restore_slot(prev_slot);
    }
};

#define I8_BEGIN try {
#define I8_END                                    \
    }                                             \
    catch (const std::bad_alloc&) {               \
        set_error("host allocation failed");      \
        return HB200_ERR_TOO_LARGE;               \
    }                                             \
    catch (...) {                                 \
        set_error("unexpected C++ exception");    \
        return HB200_ERR_CUDA;                    \
    }
#define I8_USE(slot)              \
    DeviceScope _scope(slot);     \
    if (_scope.rc) return _scope.rc
// For a call whose kernels read an object: the object outlives hb200_shutdown, and its slot may be bound to another device since.
#define I8_USE_OF(obj)            \
    I8_USE((obj)->slot);          \
    if (const int _rc = check_device((obj)->device)) return _rc

// Host-buffer product: staging kept per slot and grown on demand.
struct Staging {
    float* x = nullptr;
    float* out = nullptr;
    size_t x_bytes = 0, out_bytes = 0;
    hb200_act_i8_t act = nullptr;
};
Staging g_staging[MAX_PEERS];

int need_init() {
    if (bound_device() < 0) {
        set_error("hb200_init has not succeeded in this process");
        return HB200_ERR_NOT_INITIALIZED;
    }
    return 0;
}

int check_device(int device) {
    if (device == bound_device()) return 0;
    set_error("the object lives on device %d, its slot is bound to device %d now", device, bound_device());
    return HB200_ERR_NOT_INITIALIZED;
}

int grow_floats(float** p, size_t* have, size_t want) {
    if (*have >= want) return 0;
    if (*p) HB_CUDA(cudaFree(*p));
    *p = nullptr;
    *have = 0;
    HB_CUDA(cudaMalloc(p, want + want / 4 + 4096));
    *have = want + want / 4 + 4096;
    return 0;
}

int check_cols(size_t n_cols) {
    if (n_cols == 0) { set_error("0 columns"); return HB200_ERR_BAD_SHAPE; }
    if (n_cols > HB200_I8_MAX_COLS) { set_error("%zu columns (limit %d)", n_cols, HB200_I8_MAX_COLS); return HB200_ERR_TOO_LARGE; }
    return 0;
}
int check_rows(size_t n_rows, size_t n_cols) {
    const int rc = check_cols(n_cols);
    if (rc) return rc;
    if (n_rows > HB200_I8_MAX_ROWS) { set_error("%zu rows (limit %d)", n_rows, HB200_I8_MAX_ROWS); return HB200_ERR_TOO_LARGE; }
    return 0;
}
int check_seq(hb200_act_i8_t a, size_t seq_len) {
    if (seq_len > a->max_seq) { set_error("seq_len %zu exceeds the activation's capacity %zu", seq_len, a->max_seq); return HB200_ERR_BAD_SHAPE; }
    return 0;
}
int check_ld(const char* what, size_t ld, size_t least) {
    if (ld < least) { set_error("%s %zu is smaller than a row of %zu", what, ld, least); return HB200_ERR_BAD_SHAPE; }
    return 0;
}

// Device inputs of the calls that take no handle: memory a kernel on the current slot's device can read (nothing else ties
// them to that device, and reading memory of another one, or of the host, would be a fault).
int check_memory(const char* what, const void* p) {
    cudaPointerAttributes at = {};
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess || at.type == cudaMemoryTypeUnregistered) {
        cudaGetLastError();
        set_error("%s: not device memory", what);
        return HB200_ERR_BAD_SHAPE;
    }
    if (at.type == cudaMemoryTypeDevice && at.device != bound_device()) {
        set_error("%s: on device %d, the current slot is on device %d", what, at.device, bound_device());
        return HB200_ERR_BAD_SHAPE;
    }
    return 0;
}

int weight_new(size_t n_rows, size_t n_cols, hb200_weight_i8** out) {
    hb200_weight_i8* w = new hb200_weight_i8();
    w->slot = current_slot();
    w->device = bound_device();
    w->n_rows = n_rows;
    w->n_cols = n_cols;
    w->kb = (int)((n_cols + 127) / 128);
    w->plane.kb_stride = 16384;
    w->plane.tile_stride = (size_t)w->kb * 16384;
    w->plane.row_shift = 7;
    const size_t tiles = (n_rows + 127) / 128, bytes = tiles * w->plane.tile_stride, sbytes = tiles * 128 * sizeof(float);
    w->resident_bytes = bytes + sbytes;
    if (tiles > 0) {
        cudaError_t e = cudaMalloc(&w->plane.q, bytes + sbytes);  // the scales behind the plane
        // rows past the last one take part in the product of their tile (and are not stored)
        const size_t keep = (tiles - 1) * w->plane.tile_stride;
        if (e == cudaSuccess) e = cudaMemset(w->plane.q + keep, 0, bytes - keep + sbytes);
        if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
        if (e != cudaSuccess) {
            set_error("weight of %zu x %zu: %s", n_rows, n_cols, cudaGetErrorString(e));
            cudaGetLastError();
            if (w->plane.q) cudaFree(w->plane.q);
            delete w;
            return HB200_ERR_CUDA;
        }
        w->scales = reinterpret_cast<float*>(w->plane.q + bytes);
        const int rc = encode_i8_plane(&w->map, w->plane.q, 128, tiles * w->kb, 16384, 128);
        if (rc) {
            cudaFree(w->plane.q);
            delete w;
            return rc;
        }
    }
    *out = w;
    return 0;
}
void weight_delete(hb200_weight_i8* w) {
    if (w->plane.q) cudaFree(w->plane.q);
    delete w;
}
// The weight is complete when the call returns: the product reads it ahead of its stream's order.
int weight_finish(hb200_weight_i8* w, int rc, cudaStream_t st, hb200_weight_i8_t* out) {
    if (!rc) {
        const cudaError_t e = cudaStreamSynchronize(st);
        if (e != cudaSuccess) { set_error("weight re-tiling failed: %s", cudaGetErrorString(e)); rc = HB200_ERR_CUDA; }
    }
    if (rc) { weight_delete(w); return rc; }
    *out = w;
    return HB200_OK;
}

int weight_upload(size_t n_rows, size_t n_cols, const int8_t* q, const float* scales, hb200_weight_i8_t* out) {
    hb200_weight_i8* w = nullptr;
    int rc = weight_new(n_rows, n_cols, &w);
    if (rc) return rc;
    cudaStream_t st = slot_stream();
    int8_t* q_dev = nullptr;
    float* s_dev = nullptr;
    if (n_rows > 0) {
        cudaError_t e = cudaMalloc(&q_dev, n_rows * n_cols);
        if (e == cudaSuccess) e = cudaMalloc(&s_dev, n_rows * sizeof(float));
        if (e == cudaSuccess) e = cudaMemcpyAsync(q_dev, q, n_rows * n_cols, cudaMemcpyHostToDevice, st);
        if (e == cudaSuccess) e = cudaMemcpyAsync(s_dev, scales, n_rows * sizeof(float), cudaMemcpyHostToDevice, st);
        if (e != cudaSuccess) { set_error("weight copy failed: %s", cudaGetErrorString(e)); cudaGetLastError(); rc = HB200_ERR_CUDA; }
        if (!rc) rc = launch_i8_load(q_dev, n_cols, s_dev, (int)n_rows, (int)n_cols, w->plane, w->scales, st);
    }
    rc = weight_finish(w, rc, st, out);
    if (q_dev) cudaFree(q_dev);
    if (s_dev) cudaFree(s_dev);
    return rc;
}

I8Rows rows_of(hb200_act_i8_t a) {
    I8Rows p = {};
    p.n_cols = (int)a->n_cols;
    p.plane = a->plane;
    p.scales = a->scales;
    return p;
}

int check_product(hb200_weight_i8_t w, hb200_act_i8_t a, size_t seq_len, size_t ld_out) {
    if (!w || !a) { set_error("null weight or activation handle"); return HB200_ERR_NULL; }
    if (a->slot != w->slot) { set_error("the weight lives in device slot %d, the activation in slot %d", w->slot, a->slot); return HB200_ERR_BAD_SHAPE; }
    if (a->device != w->device) { set_error("the weight lives on device %d, the activation on device %d", w->device, a->device); return HB200_ERR_BAD_SHAPE; }
    if (a->n_cols != w->n_cols) { set_error("dim mismatch: weight has %zu columns, activation %zu", w->n_cols, a->n_cols); return HB200_ERR_BAD_SHAPE; }
    int rc = check_seq(a, seq_len);
    if (rc) return rc;
    return check_ld("ld_out", ld_out, w->n_rows);
}

int product(hb200_weight_i8_t w, hb200_act_i8_t a, size_t seq_len, float* out, size_t ld_out, int accumulate, cudaStream_t st, int report_rank = 0) {
    I8Product p = {};
#ifdef HB200_BOUNDS
    p.report_rank = report_rank;
#endif
    p.w = w->plane.q;
    p.sw = w->scales;
    p.a = a->plane.q;
    p.sx = a->scales;
    p.out = out;
    p.ld_out = ld_out;
    p.a_kb_stride = a->plane.kb_stride;
    p.n_rows = (int)w->n_rows;
    p.n_tok = (int)seq_len;
    p.kb = w->kb;
    p.accumulate = accumulate != 0;
    p.status = slot_status();
    p.w_map = &w->map;
    p.x_map_n128 = &a->map64;
    p.x_map_n256 = &a->map128;
    return launch_i8_gemm(p, st);
}

}  // namespace

// ----------------------------------------------------------------- weights --

extern "C" int hb200_weight_i8_upload(size_t n_rows, size_t n_cols, const int8_t* q, const float* scales, hb200_weight_i8_t* out) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!out) { set_error("null output handle"); return HB200_ERR_NULL; }
    if ((rc = check_rows(n_rows, n_cols))) return rc;
    if (n_rows > 0 && (!q || !scales)) { set_error("null weight values or scales"); return HB200_ERR_NULL; }
    I8_USE(current_slot());
    return weight_upload(n_rows, n_cols, q, scales, out);
    I8_END
}

extern "C" int hb200_weight_i8_upload_rows(size_t n_rows, size_t n_cols, const int8_t* q, const float* scales, size_t row_begin, size_t row_end,
                                           hb200_weight_i8_t* out) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!out) { set_error("null output handle"); return HB200_ERR_NULL; }
    if (row_begin > row_end || row_end > n_rows) { set_error("row range [%zu, %zu) outside 0..%zu", row_begin, row_end, n_rows); return HB200_ERR_BAD_SHAPE; }
    if ((rc = check_rows(row_end - row_begin, n_cols))) return rc;
    if (row_end > row_begin && (!q || !scales)) { set_error("null weight values or scales"); return HB200_ERR_NULL; }
    I8_USE(current_slot());
    return row_end > row_begin ? weight_upload(row_end - row_begin, n_cols, q + row_begin * n_cols, scales + row_begin, out)
                               : weight_upload(0, n_cols, nullptr, nullptr, out);
    I8_END
}

extern "C" int hb200_weight_i8_upload_dev(size_t n_rows, size_t n_cols, const int8_t* q_dev, size_t ld_q, const float* scales_dev, void* stream,
                                          hb200_weight_i8_t* out) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!out) { set_error("null output handle"); return HB200_ERR_NULL; }
    if ((rc = check_rows(n_rows, n_cols))) return rc;
    if ((rc = check_ld("ld_q", ld_q, n_cols))) return rc;
    if (n_rows > 0 && (!q_dev || !scales_dev)) { set_error("null weight values or scales"); return HB200_ERR_NULL; }
    I8_USE(current_slot());
    if (n_rows > 0 && ((rc = check_memory("weight values", q_dev)) || (rc = check_memory("weight scales", scales_dev)))) return rc;
    hb200_weight_i8* w = nullptr;
    if ((rc = weight_new(n_rows, n_cols, &w))) return rc;
    rc = launch_i8_load(q_dev, ld_q, scales_dev, (int)n_rows, (int)n_cols, w->plane, w->scales, (cudaStream_t)stream);
    return weight_finish(w, rc, (cudaStream_t)stream, out);
    I8_END
}

extern "C" int hb200_weight_i8_quantize_dev(size_t n_rows, size_t n_cols, const float* w_dev, size_t ld_w, void* stream, hb200_weight_i8_t* out) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!out) { set_error("null output handle"); return HB200_ERR_NULL; }
    if ((rc = check_rows(n_rows, n_cols))) return rc;
    if ((rc = check_ld("ld_w", ld_w, n_cols))) return rc;
    if (n_rows > 0 && !w_dev) { set_error("null weight values"); return HB200_ERR_NULL; }
    I8_USE(current_slot());
    if (n_rows > 0 && (rc = check_memory("weight values", w_dev))) return rc;
    hb200_weight_i8* w = nullptr;
    if ((rc = weight_new(n_rows, n_cols, &w))) return rc;
    I8Rows p = {};
    p.x = w_dev;
    p.ld = ld_w;
    p.n_cols = (int)n_cols;
    p.plane = w->plane;
    p.scales = w->scales;
    rc = launch_i8_rows(I8_QUANTIZE, p, (int)n_rows, (cudaStream_t)stream);
    return weight_finish(w, rc, (cudaStream_t)stream, out);
    I8_END
}

extern "C" int hb200_weight_i8_store_dev(hb200_weight_i8_t w, int8_t* q_dev, size_t ld_q, float* scales_dev, void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!w) { set_error("null weight handle"); return HB200_ERR_NULL; }
    if (q_dev && (rc = check_ld("ld_q", ld_q, w->n_cols))) return rc;
    I8_USE_OF(w);
    return launch_i8_store(w->plane, w->scales, (int)w->n_rows, (int)w->n_cols, q_dev, ld_q, scales_dev, (cudaStream_t)stream);
    I8_END
}

extern "C" int hb200_weight_i8_free(hb200_weight_i8_t w) {
    I8_BEGIN
    if (!w) return HB200_OK;
    I8_USE(w->slot);
    weight_delete(w);
    return HB200_OK;
    I8_END
}

extern "C" int hb200_weight_i8_info(hb200_weight_i8_t w, size_t* n_rows, size_t* n_cols, size_t* resident_bytes, int* device) {
    if (!w) { set_error("null weight handle"); return HB200_ERR_NULL; }
    if (n_rows) *n_rows = w->n_rows;
    if (n_cols) *n_cols = w->n_cols;
    if (resident_bytes) *resident_bytes = w->resident_bytes;
    if (device) *device = w->device;
    return HB200_OK;
}

// ------------------------------------------------------------- activations --

extern "C" int hb200_act_i8_create(size_t max_seq_len, size_t n_cols, hb200_act_i8_t* out) {
    I8_BEGIN
    if (!out) { set_error("null output handle"); return HB200_ERR_NULL; }
    if (max_seq_len == 0) { set_error("activation of 0 tokens"); return HB200_ERR_BAD_SHAPE; }
    int rc = check_cols(n_cols);
    if (rc) return rc;
    if (max_seq_len > HB200_MAX_SEQ_LEN) { set_error("activation of %zu tokens (limit %d)", max_seq_len, HB200_MAX_SEQ_LEN); return HB200_ERR_TOO_LARGE; }
    if ((rc = need_init())) return rc;
    I8_USE(current_slot());
    hb200_act_i8* a = new hb200_act_i8();
    a->slot = current_slot();
    a->device = bound_device();
    a->max_seq = max_seq_len;
    a->n_cols = n_cols;
    a->kb = (int)((n_cols + 127) / 128);
    const size_t groups = (max_seq_len + 7) / 8;
    a->plane.tile_stride = 1024;
    a->plane.kb_stride = groups * 1024;
    a->plane.row_shift = 3;
    const size_t bytes = (size_t)a->kb * a->plane.kb_stride, sbytes = groups * 8 * sizeof(float);
    cudaError_t e = cudaMalloc(&a->plane.q, bytes + sbytes);  // the scales behind the plane
    if (e == cudaSuccess) e = cudaMemset(a->plane.q, 0, bytes + sbytes);
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) {
        set_error("activation allocation failed: %s", cudaGetErrorString(e));
        cudaGetLastError();
        if (a->plane.q) cudaFree(a->plane.q);
        delete a;
        return HB200_ERR_CUDA;
    }
    a->scales = reinterpret_cast<float*>(a->plane.q + bytes);
    rc = encode_i8_plane(&a->map64, a->plane.q, groups * 8, a->kb, a->plane.kb_stride, 64);
    if (!rc) rc = encode_i8_plane(&a->map128, a->plane.q, groups * 8, a->kb, a->plane.kb_stride, 128);
    if (rc) {
        cudaFree(a->plane.q);
        delete a;
        return rc;
    }
    *out = a;
    return HB200_OK;
    I8_END
}

extern "C" int hb200_act_i8_free(hb200_act_i8_t a) {
    I8_BEGIN
    if (!a) return HB200_OK;
    I8_USE(a->slot);
    if (a->plane.q) cudaFree(a->plane.q);
    delete a;
    return HB200_OK;
    I8_END
}

extern "C" int hb200_act_i8_info(hb200_act_i8_t a, size_t* max_seq_len, size_t* n_cols, int* device) {
    if (!a) { set_error("null activation handle"); return HB200_ERR_NULL; }
    if (max_seq_len) *max_seq_len = a->max_seq;
    if (n_cols) *n_cols = a->n_cols;
    if (device) *device = a->device;
    return HB200_OK;
}

extern "C" int hb200_act_i8_quantize_dev(hb200_act_i8_t a, const float* x_dev, size_t ld_x, size_t seq_len, void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!a) { set_error("null activation handle"); return HB200_ERR_NULL; }
    if ((rc = check_seq(a, seq_len))) return rc;
    if ((rc = check_ld("ld_x", ld_x, a->n_cols))) return rc;
    if (seq_len == 0) return HB200_OK;
    if (!x_dev) { set_error("null pointer"); return HB200_ERR_NULL; }
    I8_USE_OF(a);
    I8Rows p = rows_of(a);
    p.x = x_dev;
    p.ld = ld_x;
    return launch_i8_rows(I8_QUANTIZE, p, (int)seq_len, (cudaStream_t)stream);
    I8_END
}

extern "C" int hb200_act_i8_add_rms_norm_dev(hb200_act_i8_t a, const float* x_dev, const float* residual_dev, size_t ld_x, const float* weight_dev,
                                             float eps, size_t seq_len, float* sum_dev, size_t ld_sum, void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!a) { set_error("null activation handle"); return HB200_ERR_NULL; }
    if ((rc = check_seq(a, seq_len))) return rc;
    if ((rc = check_ld("ld_x", ld_x, a->n_cols))) return rc;
    if (sum_dev && (rc = check_ld("ld_sum", ld_sum, a->n_cols))) return rc;
    if (!(eps > 0.0f && eps <= FLT_MAX)) { set_error("eps %g: a positive finite number", (double)eps); return HB200_ERR_BAD_SHAPE; }
    if (sum_dev && ld_sum != ld_x && (sum_dev == x_dev || sum_dev == residual_dev)) {
        set_error("the sum overwrites an input row by row: ld_sum %zu must be ld_x %zu", ld_sum, ld_x);
        return HB200_ERR_BAD_SHAPE;
    }
    if (seq_len == 0) return HB200_OK;
    if (!x_dev || !weight_dev) { set_error("null pointer"); return HB200_ERR_NULL; }
    I8_USE_OF(a);
    I8Rows p = rows_of(a);
    p.x = x_dev;
    p.y = residual_dev;
    p.ld = ld_x;
    p.weight = weight_dev;
    p.eps = eps;
    p.sum = sum_dev;
    p.ld_sum = ld_sum;
    return launch_i8_rows(I8_ADD_RMS_NORM, p, (int)seq_len, (cudaStream_t)stream);
    I8_END
}

extern "C" int hb200_act_i8_silu_mul_dev(hb200_act_i8_t a, const float* gate_dev, const float* up_dev, size_t ld, size_t seq_len, void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!a) { set_error("null activation handle"); return HB200_ERR_NULL; }
    if ((rc = check_seq(a, seq_len))) return rc;
    if ((rc = check_ld("ld", ld, a->n_cols))) return rc;
    if (seq_len == 0) return HB200_OK;
    if (!gate_dev || !up_dev) { set_error("null pointer"); return HB200_ERR_NULL; }
    I8_USE_OF(a);
    I8Rows p = rows_of(a);
    p.x = gate_dev;
    p.y = up_dev;
    p.ld = ld;
    return launch_i8_rows(I8_SILU_MUL, p, (int)seq_len, (cudaStream_t)stream);
    I8_END
}

extern "C" int hb200_act_i8_load_dev(hb200_act_i8_t a, const int8_t* q_dev, size_t ld_q, const float* scales_dev, size_t seq_len, void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!a) { set_error("null activation handle"); return HB200_ERR_NULL; }
    if ((rc = check_seq(a, seq_len))) return rc;
    if ((rc = check_ld("ld_q", ld_q, a->n_cols))) return rc;
    if (seq_len == 0) return HB200_OK;
    if (!q_dev || !scales_dev) { set_error("null pointer"); return HB200_ERR_NULL; }
    I8_USE_OF(a);
    return launch_i8_load(q_dev, ld_q, scales_dev, (int)seq_len, (int)a->n_cols, a->plane, a->scales, (cudaStream_t)stream);
    I8_END
}

extern "C" int hb200_act_i8_store_dev(hb200_act_i8_t a, int8_t* q_dev, size_t ld_q, float* scales_dev, size_t seq_len, void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!a) { set_error("null activation handle"); return HB200_ERR_NULL; }
    if ((rc = check_seq(a, seq_len))) return rc;
    if (q_dev && (rc = check_ld("ld_q", ld_q, a->n_cols))) return rc;
    if (seq_len == 0) return HB200_OK;
    if (!q_dev && !scales_dev) { set_error("nothing to store into"); return HB200_ERR_NULL; }
    I8_USE_OF(a);
    return launch_i8_store(a->plane, a->scales, (int)seq_len, (int)a->n_cols, q_dev, ld_q, scales_dev, (cudaStream_t)stream);
    I8_END
}

extern "C" int hb200_act_i8_dequantize_dev(hb200_act_i8_t a, float* out_dev, size_t ld_out, size_t seq_len, void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!a) { set_error("null activation handle"); return HB200_ERR_NULL; }
    if ((rc = check_seq(a, seq_len))) return rc;
    if ((rc = check_ld("ld_out", ld_out, a->n_cols))) return rc;
    if (seq_len == 0) return HB200_OK;
    if (!out_dev) { set_error("null output"); return HB200_ERR_NULL; }
    I8_USE_OF(a);
    return launch_i8_dequantize(a->plane, a->scales, (int)seq_len, (int)a->n_cols, out_dev, ld_out, (cudaStream_t)stream);
    I8_END
}

// ----------------------------------------------------------------- product --

extern "C" int hb200_matmul_i8_dev(hb200_weight_i8_t w, hb200_act_i8_t a, size_t seq_len, float* out_dev, size_t ld_out, int accumulate,
                                   void* stream) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if ((rc = check_product(w, a, seq_len, ld_out))) return rc;
    if (seq_len == 0 || w->n_rows == 0) return HB200_OK;
    if (!out_dev) { set_error("null output"); return HB200_ERR_NULL; }
    I8_USE_OF(w);
    return product(w, a, seq_len, out_dev, ld_out, accumulate, (cudaStream_t)stream);
    I8_END
}

extern "C" int hb200_matmul_i8(hb200_weight_i8_t w, const float* x, size_t seq_len, float* out) {
    I8_BEGIN
    int rc = need_init();
    if (rc) return rc;
    if (!w) { set_error("null weight handle"); return HB200_ERR_NULL; }
    if (seq_len > HB200_MAX_SEQ_LEN) { set_error("seq_len %zu (limit %d)", seq_len, HB200_MAX_SEQ_LEN); return HB200_ERR_TOO_LARGE; }
    if (seq_len == 0 || w->n_rows == 0) return HB200_OK;
    if (!x || !out) { set_error("null buffer"); return HB200_ERR_NULL; }
    I8_USE_OF(w);
    Staging& g = g_staging[w->slot];
    const size_t in_bytes = seq_len * w->n_cols * sizeof(float), out_bytes = seq_len * w->n_rows * sizeof(float);
    if ((rc = grow_floats(&g.x, &g.x_bytes, in_bytes))) return rc;
    if ((rc = grow_floats(&g.out, &g.out_bytes, out_bytes))) return rc;
    if (!g.act || g.act->n_cols != w->n_cols || g.act->max_seq < seq_len) {
        hb200_act_i8_t old = g.act;
        g.act = nullptr;
        if ((rc = hb200_act_i8_free(old))) return rc;
        if ((rc = hb200_act_i8_create(seq_len, w->n_cols, &g.act))) return rc;
    }
    cudaStream_t st = slot_stream();
    HB_CUDA(cudaMemcpyAsync(g.x, x, in_bytes, cudaMemcpyHostToDevice, st));
    I8Rows p = rows_of(g.act);
    p.x = g.x;
    p.ld = w->n_cols;
    if ((rc = launch_i8_rows(I8_QUANTIZE, p, (int)seq_len, st))) return rc;
    if ((rc = product(w, g.act, seq_len, g.out, w->n_rows, 0, st))) return rc;
    HB_CUDA(cudaMemcpyAsync(out, g.out, out_bytes, cudaMemcpyDeviceToHost, st));
    HB_CUDA(cudaStreamSynchronize(st));
    return take_device_status();  // every product kernel has bounded waits
    I8_END
}

extern "C" const char* hb200_matmul_i8_kernel(size_t n_rows, size_t n_cols, size_t seq_len) {
    if (n_rows == 0 || n_cols == 0 || seq_len == 0 || n_rows > HB200_I8_MAX_ROWS || n_cols > HB200_I8_MAX_COLS || seq_len > HB200_MAX_SEQ_LEN)
        return "none";
    return i8_gemm_kernel_name((int)n_rows, (int)((n_cols + 127) / 128), (int)seq_len);
}

namespace hb200 {
void i8_release_slot(int slot) {
    Staging& g = g_staging[slot];
    if (g.x) cudaFree(g.x);
    if (g.out) cudaFree(g.out);
    if (g.act) {
        if (g.act->plane.q) cudaFree(g.act->plane.q);
        delete g.act;
    }
    g = Staging();
}

#ifdef HB200_BOUNDS
int i8_failure_selftest() {
    // 9 tokens x 2048 columns x 200 rows: two row tiles, each cut over the eight CTAs of a cluster; all operands 1, all scales one float
    constexpr size_t TOK = 9, COLS = 2048, ROWS = 200;
    cudaStream_t st = slot_stream();
    int8_t* q = nullptr;
    float *s = nullptr, *out = nullptr;
    hb200_weight_i8_t w = nullptr;
    hb200_act_i8_t a = nullptr;
    std::vector<float> got(TOK * ROWS);
    HB_CUDA(cudaMalloc(&q, ROWS * COLS));
    HB_CUDA(cudaMalloc(&s, ROWS * sizeof(float)));
    HB_CUDA(cudaMalloc(&out, got.size() * sizeof(float)));
    HB_CUDA(cudaMemset(q, 1, ROWS * COLS));
    HB_CUDA(cudaMemset(s, 0x3F, ROWS * sizeof(float)));
    HB_CUDA(cudaDeviceSynchronize());
    int rc = hb200_weight_i8_upload_dev(ROWS, COLS, q, COLS, s, st, &w);
    if (!rc) rc = hb200_act_i8_create(TOK, COLS, &a);
    if (!rc) rc = hb200_act_i8_load_dev(a, q, COLS, s, TOK, st);
    for (int rank = -1; rank < 8 && !rc; rank++) {
        HB_CUDA(cudaMemsetAsync(out, 0, got.size() * sizeof(float), st));
        if ((rc = product(w, a, TOK, out, ROWS, 0, st, rank + 1))) break;
        HB_CUDA(cudaMemcpyAsync(got.data(), out, got.size() * sizeof(float), cudaMemcpyDeviceToHost, st));
        HB_CUDA(cudaStreamSynchronize(st));
        const int want = rank < 0 ? HB200_OK : HB200_ERR_TIMEOUT, status = take_device_status();
        size_t stored = 0;
        for (float v : got) stored += v != 0.0f;
        if (status != want || stored != (rank < 0 ? got.size() : 0)) {
            set_error("8-bit product self-test: rank %d reports a failure, status %d, %zu of %zu outputs stored", rank, status, stored, got.size());
            rc = HB200_ERR_CUDA;
        }
    }
    if (a) hb200_act_i8_free(a);
    if (w) hb200_weight_i8_free(w);
    cudaFree(q); cudaFree(s); cudaFree(out);
    return rc;
}
#endif
}  // namespace hb200
