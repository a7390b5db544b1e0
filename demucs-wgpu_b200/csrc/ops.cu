// The operator entry points of include/dmx.h (dmx_ops_*, dmx_layer_norm*,
// dmx_quantize_rows, dmx_quantized_linear): argument checks, the device guard
// and the status codes around the launchers of ops.h. Nothing here throws
// across the boundary, allocates device memory after dmx_ops_create, or waits
// (dmx_ops_check excepted), so calls may be captured into a CUDA graph.
#include <atomic>
#include <chrono>
#include <cmath>
#include <thread>

#include "kernels.h"
#include "ops.h"
#include "runtime.cuh"

using namespace dmx;

struct dmx_ops {
  int device = 0;
  int* err = nullptr;  // raised by a bounded wait that gave up
};

namespace dmx {

int sm_count() {
  static std::atomic<int> count[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  int n = count[dev].load();
  if (n == 0) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    count[dev].store(n);
  }
  return n;
}

void check_cuda(cudaError_t e) {
  if (e == cudaSuccess) return;
  cudaGetLastError();
  throw Error(DMX_ERR_CUDA, std::string("an operator's kernel could not be launched: ") + cudaGetErrorString(e));
}

}  // namespace dmx

namespace {

// Makes the context's device current for a call and puts the caller's back.
struct OnDevice {
  int before = 0, device;
  explicit OnDevice(int d) : device(d) {
    CK(cudaGetDevice(&before));
    if (before != device) CK(cudaSetDevice(device));
  }
  ~OnDevice() {
    if (before != device) cudaSetDevice(before);
  }
};

// Largest row count, row length and pitch taken: offsets stay far inside 64 bits.
constexpr int64_t kMaxRows = INT32_MAX, kMaxCols = INT32_MAX / 4, kMaxPitch = 1ll << 31;
// 128 * 128 * k must stay below 2^31
constexpr int64_t kMaxInner = 131071;

[[noreturn]] void refuse(const char* what, const std::string& why) {
  throw Error(DMX_ERR_INVALID, std::string(what) + ": " + why);
}

size_t type_bytes(const char* what, const char* name, int type) {
  if (type == DMX_TYPE_F32) return 4;
  if (type == DMX_TYPE_F16 || type == DMX_TYPE_BF16) return 2;
  refuse(what, std::string(name) + " must be DMX_TYPE_F32, DMX_TYPE_F16 or DMX_TYPE_BF16");
}

void check_shape(const char* what, int64_t rows, int64_t cols) {
  if (rows < 0 || rows > kMaxRows) refuse(what, "rows must be in [0, 2^31 - 1]");
  if (cols < 1 || cols > kMaxCols) refuse(what, "cols must be in [1, 2^29 - 1]");
}

// A row-major operand: present, aligned to its elements, pitch at least its row.
void check_rows(const char* what, const char* name, const void* p, size_t align, int64_t ld,
                int64_t cols) {
  if (!p) refuse(what, std::string(name) + " is null");
  if (reinterpret_cast<uintptr_t>(p) % align)
    refuse(what, std::string(name) + " is not aligned to " + std::to_string(align) + " bytes");
  if (ld < cols || ld > kMaxPitch)
    refuse(what, std::string(name) + "_ld must be in [row length, 2^31]");
}

void check_vector(const char* what, const char* name, const void* p, size_t align, bool needed) {
  if (!p) {
    if (needed) refuse(what, std::string(name) + " is null");
    return;
  }
  if (reinterpret_cast<uintptr_t>(p) % align)
    refuse(what, std::string(name) + " is not aligned to its elements");
}

// x and y may be one buffer only element for element.
void check_in_place(const char* what, const void* x, int x_type, int64_t x_ld, const void* y,
                    int y_type, int64_t y_ld) {
  if (x == y && (x_type != y_type || x_ld != y_ld))
    refuse(what, "in place needs one type and one pitch");
}

void check_call(const char* what, const dmx_ops* ops, const void* args) {
  if (!ops) refuse(what, "ops is null");
  if (!args) refuse(what, "args is null");
}

// The fields that dmx_layer_norm and dmx_layer_norm_quantize share.
template <typename Args>
void set_norm(const char* what, const Args* g, RowArgs* a) {
  if (g->weight || g->bias) {
    const size_t b = type_bytes(what, "param_type", g->param_type);
    check_vector(what, "weight", g->weight, b, false);
    check_vector(what, "bias", g->bias, b, false);
  }
  if (!(g->eps >= 0.f) || std::isinf(g->eps)) refuse(what, "eps must be finite and not negative");
  check_vector(what, "mean", g->mean, 4, false);
  check_vector(what, "rstd", g->rstd, 4, false);
  a->norm = true;
  a->weight = g->weight;
  a->bias = g->bias;
  a->param_type = g->param_type;
  a->eps = g->eps;
  a->mean = g->mean;
  a->rstd = g->rstd;
  a->rows = g->rows;
  a->cols = (int)g->cols;
}

// The fields that dmx_quantize_rows and dmx_layer_norm_quantize share.
template <typename Args>
void set_quantized(const char* what, const Args* g, size_t x_bytes, RowArgs* a) {
  a->x = g->x;
  a->x_type = g->x_type;
  a->x_ld = g->x_ld ? g->x_ld : g->cols;
  a->q = g->q;
  a->q_ld = g->q_ld ? g->q_ld : g->cols;
  a->scale = g->scale;
  check_rows(what, "x", a->x, x_bytes, a->x_ld, g->cols);
  check_rows(what, "q", a->q, 1, a->q_ld, g->cols);
  check_vector(what, "scale", g->scale, 4, true);
  if (static_cast<const void*>(g->q) == g->x) refuse(what, "q must not be x");
}

template <typename F>
dmx_status guarded(F&& f) {
  try {
    f();
    return DMX_OK;
  } catch (const Error& e) {
    return fail(e);
  } catch (const std::exception& e) {
    return fail_std(e);
  }
}

}  // namespace

extern "C" {

dmx_status dmx_ops_create(int device, dmx_ops** out) {
  return guarded([&] {
    if (!out) refuse("dmx_ops_create", "out is null");
    *out = nullptr;
    int count = 0;
    CK(cudaGetDeviceCount(&count));
    if (device < 0 || device >= count) refuse("dmx_ops_create", "no such device");
    OnDevice on(device);
    std::unique_ptr<dmx_ops> o(new dmx_ops());
    o->device = device;
    CK(cudaMalloc(&o->err, sizeof(int)));
    const cudaError_t e = cudaMemset(o->err, 0, sizeof(int));
    if (e != cudaSuccess) {
      cudaFree(o->err);
      CK(e);
    }
    CK(cudaDeviceSynchronize());  // the flag is clear before any stream's first call
    *out = o.release();
  });
}

void dmx_ops_destroy(dmx_ops* ops) {
  if (!ops) return;
  int before = 0;
  cudaGetDevice(&before);
  cudaSetDevice(ops->device);
  cudaFree(ops->err);  // waits for the device's work in flight
  cudaSetDevice(before);
  delete ops;
}

dmx_status dmx_ops_check(dmx_ops* ops, void* stream) {
  return guarded([&] {
    if (!ops) refuse("dmx_ops_check", "ops is null");
    OnDevice on(ops->device);
    const auto s = static_cast<cudaStream_t>(stream);
    const auto deadline = std::chrono::steady_clock::now() + std::chrono::seconds(600);
    while (true) {
      const cudaError_t q = cudaStreamQuery(s);
      if (q == cudaSuccess) break;
      if (q != cudaErrorNotReady) CK(q);
      if (std::chrono::steady_clock::now() > deadline)
        throw Error(DMX_ERR_TIMEOUT, "dmx_ops_check: the stream did not drain within the deadline");
      std::this_thread::sleep_for(std::chrono::microseconds(20));
    }
    int code = 0;
    CK(cudaMemcpyAsync(&code, ops->err, sizeof(int), cudaMemcpyDeviceToHost, s));
    CK(cudaStreamSynchronize(s));
    if (code == 0) return;
    CK(cudaMemsetAsync(ops->err, 0, sizeof(int), s));
    CK(cudaStreamSynchronize(s));
    throw Error(DMX_ERR_TIMEOUT,
                std::string(code == kSelftestCode ? "the self-test kernel" : "dmx_quantized_linear") +
                    ": a bounded wait gave up (code " + std::to_string(code) +
                    "); what dmx_quantized_linear wrote on any stream since the last check is not valid");
  });
}

dmx_status dmx_ops_selftest_wait_timeout(dmx_ops* ops, int wait_ms, void* stream) {
  return guarded([&] {
    const char* what = "dmx_ops_selftest_wait_timeout";
    if (!ops) refuse(what, "ops is null");
    if (wait_ms < 1 || wait_ms > 5000) refuse(what, "wait_ms must be in [1, 5000]");
    OnDevice on(ops->device);
    check_cuda(launch_selftest_wait((uint64_t)wait_ms * 1000000ull, kSelftestCode, ops->err,
                                    static_cast<cudaStream_t>(stream)));
  });
}

dmx_status dmx_layer_norm(dmx_ops* ops, const dmx_layer_norm_args* g, void* stream) {
  return guarded([&] {
    const char* what = "dmx_layer_norm";
    check_call(what, ops, g);
    check_shape(what, g->rows, g->cols);
    RowArgs a;
    const size_t xb = type_bytes(what, "x_type", g->x_type);
    const size_t yb = type_bytes(what, "y_type", g->y_type);
    set_norm(what, g, &a);
    if (g->rows == 0) return;
    a.x = g->x;
    a.x_type = g->x_type;
    a.x_ld = g->x_ld ? g->x_ld : g->cols;
    a.y = g->y;
    a.y_type = g->y_type;
    a.y_ld = g->y_ld ? g->y_ld : g->cols;
    check_rows(what, "x", a.x, xb, a.x_ld, g->cols);
    check_rows(what, "y", a.y, yb, a.y_ld, g->cols);
    check_in_place(what, a.x, a.x_type, a.x_ld, a.y, a.y_type, a.y_ld);
    OnDevice on(ops->device);
    launch_rows(a, static_cast<cudaStream_t>(stream));
  });
}

size_t dmx_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
  if (rows < 0 || rows > kMaxRows || cols < 1 || cols > kMaxCols) return 0;
  return norm_grad_workspace(rows, cols);
}

dmx_status dmx_layer_norm_backward(dmx_ops* ops, const dmx_layer_norm_backward_args* g,
                                   void* stream) {
  return guarded([&] {
    const char* what = "dmx_layer_norm_backward";
    check_call(what, ops, g);
    check_shape(what, g->rows, g->cols);
    const size_t dyb = type_bytes(what, "dy_type", g->dy_type);
    const size_t xb = type_bytes(what, "x_type", g->x_type);
    if (g->weight)
      check_vector(what, "weight", g->weight, type_bytes(what, "param_type", g->param_type), false);
    check_vector(what, "dweight", g->dweight, 4, false);
    check_vector(what, "dbias", g->dbias, 4, false);
    NormGradArgs a;
    a.dy = g->dy;
    a.dy_type = g->dy_type;
    a.dy_ld = g->dy_ld ? g->dy_ld : g->cols;
    a.x = g->x;
    a.x_type = g->x_type;
    a.x_ld = g->x_ld ? g->x_ld : g->cols;
    a.weight = g->weight;
    a.param_type = g->param_type;
    a.mean = g->mean;
    a.rstd = g->rstd;
    a.rows = g->rows;
    a.cols = (int)g->cols;
    a.dx = g->dx;
    a.dx_ld = g->dx_ld ? g->dx_ld : g->cols;
    a.dweight = g->dweight;
    a.dbias = g->dbias;
    a.partials = static_cast<float*>(g->workspace);
    if (g->rows > 0) {
      check_rows(what, "dy", a.dy, dyb, a.dy_ld, g->cols);
      check_rows(what, "x", a.x, xb, a.x_ld, g->cols);
      check_vector(what, "mean", a.mean, 4, true);
      check_vector(what, "rstd", a.rstd, 4, true);
      if (a.dx) {
        check_rows(what, "dx", a.dx, xb, a.dx_ld, g->cols);
        check_in_place(what, a.dy, a.dy_type, a.dy_ld, a.dx, a.x_type, a.dx_ld);
        check_in_place(what, a.x, a.x_type, a.x_ld, a.dx, a.x_type, a.dx_ld);
      }
      if (a.dweight || a.dbias) {
        if (g->workspace_bytes < norm_grad_workspace(g->rows, g->cols))
          refuse(what, "the workspace is smaller than dmx_layer_norm_backward_workspace says");
        check_vector(what, "workspace", g->workspace, 16, true);
      }
    }
    OnDevice on(ops->device);
    launch_norm_grad(a, static_cast<cudaStream_t>(stream));
  });
}

dmx_status dmx_quantize_rows(dmx_ops* ops, const dmx_quantize_rows_args* g, void* stream) {
  return guarded([&] {
    const char* what = "dmx_quantize_rows";
    check_call(what, ops, g);
    check_shape(what, g->rows, g->cols);
    const size_t xb = type_bytes(what, "x_type", g->x_type);
    check_vector(what, "col_scale", g->col_scale, 4, false);
    if (g->rows == 0) return;
    RowArgs a;
    a.rows = g->rows;
    a.cols = (int)g->cols;
    a.col_scale = g->col_scale;
    set_quantized(what, g, xb, &a);
    OnDevice on(ops->device);
    launch_rows(a, static_cast<cudaStream_t>(stream));
  });
}

dmx_status dmx_layer_norm_quantize(dmx_ops* ops, const dmx_layer_norm_quantize_args* g,
                                   void* stream) {
  return guarded([&] {
    const char* what = "dmx_layer_norm_quantize";
    check_call(what, ops, g);
    check_shape(what, g->rows, g->cols);
    const size_t xb = type_bytes(what, "x_type", g->x_type);
    RowArgs a;
    set_norm(what, g, &a);
    if (g->rows == 0) return;
    set_quantized(what, g, xb, &a);
    OnDevice on(ops->device);
    launch_rows(a, static_cast<cudaStream_t>(stream));
  });
}

dmx_status dmx_quantized_linear(dmx_ops* ops, const dmx_quantized_linear_args* g, void* stream) {
  return guarded([&] {
    const char* what = "dmx_quantized_linear";
    check_call(what, ops, g);
    if (g->rows < 0 || g->rows > kMaxRows) refuse(what, "rows must be in [0, 2^31 - 1]");
    if (g->out_features < 1 || g->out_features > kMaxCols)
      refuse(what, "out_features must be in [1, 2^29 - 1]");
    if (g->in_features < 1 || g->in_features > kMaxInner)
      refuse(what, "in_features must be in [1, 131071], the longest exact 32-bit sum");
    if (g->activation != DMX_ACT_NONE && g->activation != DMX_ACT_GELU)
      refuse(what, "activation must be DMX_ACT_NONE or DMX_ACT_GELU");
    const size_t ob = type_bytes(what, "out_type", g->out_type);
    check_vector(what, "x_scale", g->x_scale, 4, false);
    check_vector(what, "w_scale", g->w_scale, 4, false);
    check_vector(what, "bias", g->bias, 4, false);
    if (g->rows == 0) return;
    LinearArgs a;
    a.x = g->x;
    a.x_ld = g->x_ld ? g->x_ld : g->in_features;
    a.x_scale = g->x_scale;
    a.w = g->w;
    a.w_ld = g->w_ld ? g->w_ld : g->in_features;
    a.w_scale = g->w_scale;
    a.bias = g->bias;
    a.rows = g->rows;
    a.n = (int)g->out_features;
    a.k = (int)g->in_features;
    a.gelu = g->activation == DMX_ACT_GELU;
    a.residual = g->residual;
    a.residual_ld = g->residual_ld ? g->residual_ld : g->out_features;
    a.out = g->out;
    a.out_type = g->out_type;
    a.out_ld = g->out_ld ? g->out_ld : g->out_features;
    a.err = ops->err;
    check_rows(what, "x", a.x, 16, a.x_ld, a.k);
    check_rows(what, "w", a.w, 16, a.w_ld, a.k);
    if (a.x_ld % 16 || a.w_ld % 16) refuse(what, "x_ld and w_ld must be multiples of 16 bytes");
    check_rows(what, "out", a.out, ob, a.out_ld, a.n);
    if (a.residual) {
      check_rows(what, "residual", a.residual, ob, a.residual_ld, a.n);
      check_in_place(what, a.residual, a.out_type, a.residual_ld, a.out, a.out_type, a.out_ld);
    }
    if (a.out == a.x || a.out == a.w) refuse(what, "out must not be x or w");
    OnDevice on(ops->device);
    if (!launch_quantized_linear(a, static_cast<cudaStream_t>(stream)))
      throw Error(DMX_ERR_CUDA, "dmx_quantized_linear: a tensor map could not be encoded");
  });
}

}  // extern "C"
