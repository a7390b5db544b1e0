// The operator entry points of include/dmx.h (dmx_ops_*, dmx_layer_norm*,
// dmx_quantize_rows, dmx_quantized_linear): argument checks, the device guard
// and the status codes around the launchers of ops.h. Nothing here throws
// across the boundary, allocates device memory after dmx_ops_create, or waits
// (dmx_ops_check excepted), so calls may be captured into a CUDA graph.
#include <cmath>
#include <chrono>
#include <thread>

#include "ops.h"
#include "runtime.cuh"

using namespace dmx;

struct dmx_ops {
  int device = 0;
  int* err = nullptr;  // raised by a bounded wait that gave up
};

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
// 127 * 128 * k must stay below 2^31 for every pair of int8 rows, -128 included
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

void check_norm(const char* what, const RowArgs& a) {
  if (a.weight || a.bias) {
    const size_t b = type_bytes(what, "param_type", a.param_type);
    check_vector(what, "weight", a.weight, b, false);
    check_vector(what, "bias", a.bias, b, false);
  }
  if (!(a.eps >= 0.f) || std::isinf(a.eps)) refuse(what, "eps must be finite and not negative");
  check_vector(what, "mean", a.mean, 4, false);
  check_vector(what, "rstd", a.rstd, 4, false);
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
    throw Error(DMX_ERR_TIMEOUT, "dmx_quantized_linear: a bounded wait gave up (code " +
                                     std::to_string(code) + "); its outputs are not valid");
  });
}

dmx_status dmx_layer_norm(dmx_ops* ops, const void* x, int x_type, int64_t x_ld,
                          const void* weight, const void* bias, int param_type, int64_t rows,
                          int64_t cols, float eps, void* y, int y_type, int64_t y_ld, float* mean,
                          float* rstd, void* stream) {
  return guarded([&] {
    const char* what = "dmx_layer_norm";
    if (!ops) refuse(what, "ops is null");
    check_shape(what, rows, cols);
    RowArgs a;
    const size_t xb = type_bytes(what, "x_type", x_type), yb = type_bytes(what, "y_type", y_type);
    a.norm = true;
    a.weight = weight;
    a.bias = bias;
    a.param_type = param_type;
    a.eps = eps;
    a.mean = mean;
    a.rstd = rstd;
    check_norm(what, a);
    if (rows == 0) return;
    check_rows(what, "x", x, xb, x_ld, cols);
    check_rows(what, "y", y, yb, y_ld, cols);
    check_in_place(what, x, x_type, x_ld, y, y_type, y_ld);
    a.x = x;
    a.x_type = x_type;
    a.x_ld = x_ld;
    a.rows = rows;
    a.cols = (int)cols;
    a.y = y;
    a.y_type = y_type;
    a.y_ld = y_ld;
    OnDevice on(ops->device);
    launch_rows(a, static_cast<cudaStream_t>(stream));
    CK(cudaGetLastError());
  });
}

size_t dmx_layer_norm_backward_workspace(int64_t rows, int64_t cols) {
  if (rows < 0 || rows > kMaxRows || cols < 1 || cols > kMaxCols) return 0;
  return norm_grad_workspace(rows, cols);
}

dmx_status dmx_layer_norm_backward(dmx_ops* ops, const void* dy, int dy_type, int64_t dy_ld,
                                   const void* x, int x_type, int64_t x_ld, const void* weight,
                                   int param_type, const float* mean, const float* rstd,
                                   int64_t rows, int64_t cols, void* dx, int64_t dx_ld,
                                   float* dweight, float* dbias, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  return guarded([&] {
    const char* what = "dmx_layer_norm_backward";
    if (!ops) refuse(what, "ops is null");
    check_shape(what, rows, cols);
    const size_t dyb = type_bytes(what, "dy_type", dy_type), xb = type_bytes(what, "x_type", x_type);
    if (weight) check_vector(what, "weight", weight, type_bytes(what, "param_type", param_type), false);
    check_vector(what, "dweight", dweight, 4, false);
    check_vector(what, "dbias", dbias, 4, false);
    NormGradArgs a;
    if (rows > 0) {
      check_rows(what, "dy", dy, dyb, dy_ld, cols);
      check_rows(what, "x", x, xb, x_ld, cols);
      check_vector(what, "mean", mean, 4, true);
      check_vector(what, "rstd", rstd, 4, true);
      if (dx) {
        check_rows(what, "dx", dx, xb, dx_ld, cols);
        check_in_place(what, dy, dy_type, dy_ld, dx, x_type, dx_ld);
        check_in_place(what, x, x_type, x_ld, dx, x_type, dx_ld);
      }
      if (dweight || dbias) {
        if (workspace_bytes < norm_grad_workspace(rows, cols))
          refuse(what, "the workspace is smaller than dmx_layer_norm_backward_workspace says");
        check_vector(what, "workspace", workspace, 16, true);
      }
    }
    a.dy = dy;
    a.dy_type = dy_type;
    a.dy_ld = dy_ld;
    a.x = x;
    a.x_type = x_type;
    a.x_ld = x_ld;
    a.weight = weight;
    a.param_type = param_type;
    a.mean = mean;
    a.rstd = rstd;
    a.rows = rows;
    a.cols = (int)cols;
    a.dx = dx;
    a.dx_ld = dx_ld;
    a.dweight = dweight;
    a.dbias = dbias;
    a.partials = static_cast<float*>(workspace);
    OnDevice on(ops->device);
    launch_norm_grad(a, static_cast<cudaStream_t>(stream));
    CK(cudaGetLastError());
  });
}

dmx_status dmx_quantize_rows(dmx_ops* ops, const void* x, int x_type, int64_t x_ld,
                             const float* col_scale, int64_t rows, int64_t cols, int8_t* q,
                             int64_t q_ld, float* scale, void* stream) {
  return guarded([&] {
    const char* what = "dmx_quantize_rows";
    if (!ops) refuse(what, "ops is null");
    check_shape(what, rows, cols);
    RowArgs a;
    const size_t xb = type_bytes(what, "x_type", x_type);
    check_vector(what, "col_scale", col_scale, 4, false);
    if (rows == 0) return;
    check_rows(what, "x", x, xb, x_ld, cols);
    check_rows(what, "q", q, 1, q_ld, cols);
    check_vector(what, "scale", scale, 4, true);
    if (static_cast<const void*>(q) == x) refuse(what, "q must not be x");
    a.x = x;
    a.x_type = x_type;
    a.x_ld = x_ld;
    a.col_scale = col_scale;
    a.rows = rows;
    a.cols = (int)cols;
    a.q = q;
    a.q_ld = q_ld;
    a.scale = scale;
    OnDevice on(ops->device);
    launch_rows(a, static_cast<cudaStream_t>(stream));
    CK(cudaGetLastError());
  });
}

dmx_status dmx_layer_norm_quantize(dmx_ops* ops, const void* x, int x_type, int64_t x_ld,
                                   const void* weight, const void* bias, int param_type,
                                   int64_t rows, int64_t cols, float eps, int8_t* q, int64_t q_ld,
                                   float* scale, float* mean, float* rstd, void* stream) {
  return guarded([&] {
    const char* what = "dmx_layer_norm_quantize";
    if (!ops) refuse(what, "ops is null");
    check_shape(what, rows, cols);
    RowArgs a;
    const size_t xb = type_bytes(what, "x_type", x_type);
    a.norm = true;
    a.weight = weight;
    a.bias = bias;
    a.param_type = param_type;
    a.eps = eps;
    a.mean = mean;
    a.rstd = rstd;
    check_norm(what, a);
    if (rows == 0) return;
    check_rows(what, "x", x, xb, x_ld, cols);
    check_rows(what, "q", q, 1, q_ld, cols);
    check_vector(what, "scale", scale, 4, true);
    if (static_cast<const void*>(q) == x) refuse(what, "q must not be x");
    a.x = x;
    a.x_type = x_type;
    a.x_ld = x_ld;
    a.rows = rows;
    a.cols = (int)cols;
    a.q = q;
    a.q_ld = q_ld;
    a.scale = scale;
    OnDevice on(ops->device);
    launch_rows(a, static_cast<cudaStream_t>(stream));
    CK(cudaGetLastError());
  });
}

dmx_status dmx_quantized_linear(dmx_ops* ops, const int8_t* x, int64_t x_ld, const float* x_scale,
                                const int8_t* w, int64_t w_ld, const float* w_scale,
                                const float* bias, int64_t rows, int64_t out_features,
                                int64_t in_features, int activation, const void* residual,
                                int64_t residual_ld, void* out, int out_type, int64_t out_ld,
                                void* stream) {
  return guarded([&] {
    const char* what = "dmx_quantized_linear";
    if (!ops) refuse(what, "ops is null");
    if (rows < 0 || rows > kMaxRows) refuse(what, "rows must be in [0, 2^31 - 1]");
    if (out_features < 1 || out_features > kMaxCols)
      refuse(what, "out_features must be in [1, 2^29 - 1]");
    if (in_features < 1 || in_features > kMaxInner)
      refuse(what, "in_features must be in [1, 131071], the longest exact 32-bit sum");
    if (activation != DMX_ACT_NONE && activation != DMX_ACT_GELU)
      refuse(what, "activation must be DMX_ACT_NONE or DMX_ACT_GELU");
    const size_t ob = type_bytes(what, "out_type", out_type);
    check_vector(what, "x_scale", x_scale, 4, false);
    check_vector(what, "w_scale", w_scale, 4, false);
    check_vector(what, "bias", bias, 4, false);
    if (rows == 0) return;
    check_rows(what, "x", x, 16, x_ld, in_features);
    check_rows(what, "w", w, 16, w_ld, in_features);
    if (x_ld % 16 || w_ld % 16) refuse(what, "x_ld and w_ld must be multiples of 16 bytes");
    check_rows(what, "out", out, ob, out_ld, out_features);
    if (residual) {
      check_rows(what, "residual", residual, ob, residual_ld, out_features);
      check_in_place(what, residual, out_type, residual_ld, out, out_type, out_ld);
    }
    if (out == x || out == w) refuse(what, "out must not be x or w");
    LinearArgs a;
    a.x = x;
    a.x_ld = x_ld;
    a.x_scale = x_scale;
    a.w = w;
    a.w_ld = w_ld;
    a.w_scale = w_scale;
    a.bias = bias;
    a.rows = rows;
    a.n = (int)out_features;
    a.k = (int)in_features;
    a.gelu = activation == DMX_ACT_GELU;
    a.residual = residual;
    a.residual_ld = residual_ld;
    a.out = out;
    a.out_type = out_type;
    a.out_ld = out_ld;
    a.err = ops->err;
    OnDevice on(ops->device);
    if (!launch_quantized_linear(a, static_cast<cudaStream_t>(stream)))
      throw Error(DMX_ERR_CUDA, "dmx_quantized_linear: a tensor map could not be encoded");
    CK(cudaGetLastError());
  });
}

}  // extern "C"
