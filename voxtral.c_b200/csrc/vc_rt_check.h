// vc_rt_check.h - what the row operators' entry points share: checks of
// arguments, the device of a call, reports.
#pragma once

#include "vc_runtime.h"

namespace vc {
namespace rt {

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }
inline bool aligned4(const void *p) { return ((uintptr_t)p & 3u) == 0; }   // as an int or an fp32 is
inline int elem_size(int dtype) { return dtype == ELEM_F32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype == ELEM_F32 || dtype == ELEM_BF16 || dtype == ELEM_F16; }

// Launches go to the library's device of the calling thread, whichever device
// the caller's other code made current.
class DeviceGuard {
  public:
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&before_) != cudaSuccess) before_ = -1;
        if (before_ != device) ok_ = cudaSetDevice(device) == cudaSuccess;
        else before_ = -1;
    }
    ~DeviceGuard() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
    bool ok() const { return ok_; }

  private:
    int before_ = -1;
    bool ok_ = true;
};

// [a, a + an) and [b, b + bn) share a byte
inline bool overlap(const void *a, double an, const void *b, double bn) {
    const double x = (double)(uintptr_t)a, y = (double)(uintptr_t)b;
    return a && b && x < y + bn && y < x + an;
}

// parents: 0 refused, 1 optional, 2 required
inline int check_rows(const char *who, const vox_cuda_rows *r, int n_streams, int ring, int parents, RowsView *out) {
    if (!r || !r->pos) {
        set_error("%s: no rows or positions", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (!aligned4(r->pos) || !aligned4(r->row_start) || !aligned4(r->parent)) {
        set_error("%s: positions, row ranges and parents must be aligned as int is", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (r->n_rows < 0 || r->max_rows < 0 || r->max_rows > r->n_rows || (r->n_rows > 0 && r->max_rows < 1)) {
        set_error("%s: bad row counts (%d rows, at most %d of a stream)", who, r->n_rows, r->max_rows);
        return VOX_CUDA_ERR_ARG;
    }
    if (!r->row_start && r->n_rows > 0 && (r->n_rows != n_streams || r->max_rows != 1)) {
        set_error("%s: without row_start there is one row for each of the %d streams, not %d", who, n_streams, r->n_rows);
        return VOX_CUDA_ERR_ARG;
    }
    if ((parents == 2 && !r->parent) || (parents == 0 && r->parent)) {
        set_error(parents ? "%s: a tree needs the rows' parents" : "%s: the rows of a window have no parents", who);
        return VOX_CUDA_ERR_ARG;
    }
    if (r->parent && r->max_rows > kTreeMax) {
        set_error("%s: a tree holds at most %d rows of a stream, not %d", who, kTreeMax, r->max_rows);
        return VOX_CUDA_ERR_ARG;
    }
    if (r->max_rows > ring) {
        set_error("%s: a ring of %d positions cannot hold %d rows", who, ring, r->max_rows);
        return VOX_CUDA_ERR_CAPACITY;
    }
    out->pos = r->pos;
    out->start = r->row_start;
    out->parent = r->parent;
    out->n_rows = r->n_rows;
    out->max_rows = r->max_rows;
    return VOX_CUDA_OK;
}

inline int check_layer(const char *who, int layer, int n_layers) {
    if (layer >= 0 && layer < n_layers) return VOX_CUDA_OK;
    set_error("%s: layer %d of %d", who, layer, n_layers);
    return VOX_CUDA_ERR_ARG;
}

inline int check_heads(const char *who, int n_heads, int n_kv_heads) {
    if (n_heads >= 1 && n_heads % n_kv_heads == 0 && n_heads / n_kv_heads <= kMaxGroup) return VOX_CUDA_OK;
    set_error("%s: %d heads over %d KV heads (a multiple of them, at most %d times as many)", who, n_heads, n_kv_heads,
              kMaxGroup);
    return VOX_CUDA_ERR_ARG;
}

// A wait that ran out in the kernel of an earlier call of this thread is
// reported once; that call's rows are NaN.
inline int check_waits(const char *who, DevCtx *c) {
    if (!__atomic_exchange_n(c->op_err + op_slot(), 0u, __ATOMIC_RELAXED)) return VOX_CUDA_OK;
    set_error("%s: a device-side wait of an earlier call of this thread timed out (its rows are void: NaN)", who);
    return VOX_CUDA_ERR_CUDA;
}

inline int launched(const char *who, cudaError_t e) {
    if (e == cudaSuccess) return VOX_CUDA_OK;
    cudaGetLastError();   // reported here, not by whoever asks next
    set_error("%s: %s", who, cudaGetErrorString(e));
    return VOX_CUDA_ERR_CUDA;
}

}  // namespace rt
}  // namespace vc
