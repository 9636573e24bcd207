// Entry points of the feed-forward operators: argument checks, operand staging, order of launches.
#include <string>

#include "ffn.cuh"

using namespace exob200;

namespace {

bool refuse(const char* fn, bool cond, const std::string& what, int code = EXO_B200_ERR_INVALID_ARGUMENT) {
  if (cond) set_error(code, std::string(fn) + ": " + what);
  return cond;
}

// Nothing is thrown through a C entry (a failing allocation of a message, a mutex): it becomes the call's error.
template <class F>
void guarded(const char* fn, F body) {
  try {
    clear_error();
    body();
  } catch (...) {
    try {
      set_error(EXO_B200_ERR_CUDA, std::string(fn) + ": host-side failure");
    } catch (...) {
    }
  }
}

// sums of K products of int8 fit int32 up to here: 131071 * 128 * 128 < 2^31
constexpr int_fast32_t kMaxI8K = 131071;

bool bad_sizes(const char* fn, int_fast32_t a, int_fast32_t b, int_fast32_t c, const char* names) {
  return refuse(fn, a < 1 || b < 1 || c < 1, std::string(names) + " must be >= 1") ||
         refuse(fn, a > INT32_MAX - 512 || b > INT32_MAX - 512 || c > INT32_MAX - 512, "size out of range",
                EXO_B200_ERR_UNSUPPORTED);
}
bool bad_act(const char* fn, int_fast32_t act) {
  return refuse(fn, act < EXO_B200_ACT_SILU || act > EXO_B200_ACT_GELU_TANH,
                "activation must be one of EXO_B200_ACT_SILU, _GELU, _GELU_TANH");
}

// A thread that is capturing in the strict modes may not allocate, nor ask for much else, until the capture ends; what a
// first call sets up (the context's status word, its pool, kernel attributes) touches no stream, so it may.
class RelaxedCapture {
 public:
  RelaxedCapture() { exchange(); }
  ~RelaxedCapture() { exchange(); }
  RelaxedCapture(const RelaxedCapture&) = delete;
  RelaxedCapture& operator=(const RelaxedCapture&) = delete;

 private:
  void exchange() {
    if (cudaThreadExchangeStreamCaptureMode(&mode_) != cudaSuccess) cudaGetLastError();
  }
  cudaStreamCaptureMode mode_ = cudaStreamCaptureModeRelaxed;
};

// The operands of one call: in() and out() take them in any order before anything is enqueued, done() returns the
// results of host calls.  dev(i) is operand i's device address, nullptr for one that was NULL.
class Operands {
 public:
  Operands(const char* fn, void* ctxt) : fn_(fn), use_(resolve_context(ctxt)) {}
  exo_b200_Context* ctx() const { return use_.get(); }

  Operands& in(const void* p, size_t bytes, size_t align) { return add(p, bytes, align, false, false); }
  Operands& maybe_in(const void* p, size_t bytes, size_t align) { return add(p, bytes, align, false, true); }
  Operands& out(void* p, size_t bytes, size_t align) { return add(p, bytes, align, true, false); }
  Operands& maybe_out(void* p, size_t bytes, size_t align) { return add(p, bytes, align, true, true); }

  // Checks every pointer before the first copy, so that a refused call has touched nothing.
  bool stage() {
    if (!ctx() || bad_) return false;
    bool host = false;
    for (int i = 0; i < n_; i++) {
      if (!op_[i].user) continue;
      cudaPointerAttributes attr;
      const bool known = cudaPointerGetAttributes(&attr, op_[i].user) == cudaSuccess;
      if (!known) cudaGetLastError();
      if (known && attr.type == cudaMemoryTypeDevice && attr.device != ctx()->device) {
        set_error(EXO_B200_ERR_INVALID_ARGUMENT, std::string(fn_) + ": operand " + std::to_string(i + 1) +
                                                     " belongs to device " + std::to_string(attr.device) +
                                                     " but the context is on device " + std::to_string(ctx()->device));
        return false;
      }
      on_device_[i] = known && (attr.type == cudaMemoryTypeDevice || attr.type == cudaMemoryTypeManaged);
      host = host || !on_device_[i];
    }
    if (host && stream_is_capturing(ctx()->stream)) {
      set_error(EXO_B200_ERR_UNSUPPORTED, std::string(fn_) + ": host operands on a stream that is being captured");
      return false;
    }
    for (int i = 0; i < n_; i++) {
      if (!op_[i].user) continue;
      if (on_device_[i]) {
        op_[i].dev = const_cast<void*>(op_[i].user);
        op_[i].staged = false;
      } else if (!stage_in(ctx(), i, op_[i].user, op_[i].bytes, !out_[i], &op_[i])) {
        return fail();
      }
    }
    return true;
  }
  template <class P>
  P* dev(int i) const {
    return static_cast<P*>(op_[i].dev);
  }
  // The result of the launches; on success copies staged outputs back.
  void done(cudaError_t e) {
    bool staged = false;
    if (e != cudaSuccess) {
      // a launcher that has said why (a tensor map, an allocation) keeps its message
      if (last_error_code() == EXO_B200_OK) check_cuda(e, fn_);
      cudaGetLastError();
      fail();
      return;
    }
    for (int i = 0; i < n_; i++) {
      if (!op_[i].user || !op_[i].staged) continue;
      staged = true;
      if (out_[i] && !stage_out(ctx(), op_[i])) {
        fail();
        return;
      }
    }
    finish(ctx(), staged);
  }

 private:
  Operands& add(const void* p, size_t bytes, size_t align, bool out, bool optional) {
    op_[n_] = Operand{p, nullptr, bytes, false};
    out_[n_] = out;
    n_++;
    if (bad_) return *this;
    bad_ = refuse(fn_, !p && !optional, "NULL tensor (operand " + std::to_string(n_) + ")") ||
           refuse(fn_, (reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0,
                  "operand " + std::to_string(n_) + " is not aligned to its element");
    return *this;
  }
  // copies in flight may still read the caller's buffers: wait for them, keep the error
  bool fail() {
    bool staged = false;
    for (int i = 0; i < n_; i++) staged = staged || op_[i].staged;
    if (staged) {
      cudaStreamSynchronize(ctx()->stream);
      cudaGetLastError();
    }
    return false;
  }

  const char* fn_;
  RelaxedCapture relaxed_;  // before the context is looked up
  ContextUse use_;
  Operand op_[kStageSlots];
  bool out_[kStageSlots], on_device_[kStageSlots];
  int n_ = 0;
  bool bad_ = false;
};

size_t mul(int_fast32_t a, int_fast32_t b, size_t e) { return (size_t)a * (size_t)b * e; }

void quantize(const char* fn, void* ctxt, int_fast32_t M, int_fast32_t K, const void* X, bool bf16, int8_t* Q,
              float* scale) {
  if (bad_sizes(fn, M, K, 1, "M and K")) return;
  const size_t e = bf16 ? 2 : 4;
  Operands o(fn, ctxt);
  if (!o.in(X, mul(M, K, e), e).out(Q, mul(M, K, 1), 1).out(scale, mul(M, 1, 4), 4).stage()) return;
  o.done(ffn::launch_quantize_rows(o.ctx(), M, K, o.dev<void>(0), bf16, o.dev<int8_t>(1), o.dev<float>(2)));
}

void gemm_scaled(const char* fn, void* ctxt, int_fast32_t M, int_fast32_t N, int_fast32_t K, const int8_t* A,
                 const int8_t* B, const float* row_scale, const float* col_scale, const float* bias, void* C,
                 bool f32) {
  if (bad_sizes(fn, M, N, K, "M, N, K")) return;
  if (refuse(fn, K > kMaxI8K, "K above 131071 would overflow the int32 sums", EXO_B200_ERR_UNSUPPORTED)) return;
  const size_t e = f32 ? 4 : 2;
  Operands o(fn, ctxt);
  if (!o.in(A, mul(M, K, 1), 1)
           .in(B, mul(N, K, 1), 1)
           .in(row_scale, mul(M, 1, 4), 4)
           .in(col_scale, mul(N, 1, 4), 4)
           .maybe_in(bias, mul(N, 1, 4), 4)
           .out(C, mul(M, N, e), e)
           .stage())
    return;
  ffn::Problem p{};
  p.M = M, p.N = N, p.K = K;
  p.a0 = o.dev<void>(0), p.b0 = o.dev<void>(1);
  p.row_scale = o.dev<float>(2), p.col_scale = o.dev<float>(3), p.bias = o.dev<float>(4);
  p.c0 = o.dev<void>(5);
  o.done(ffn::launch_product(o.ctx(), ffn::SCALED, f32, p, false));
}

void linear(const char* fn, void* ctxt, int_fast32_t M, int_fast32_t N, int_fast32_t K, const void* X,
            const int8_t* B, const float* col_scale, const float* bias, int8_t* Q, float* row_scale, void* Y,
            bool f32) {
  if (bad_sizes(fn, M, N, K, "M, N, K")) return;
  if (refuse(fn, K > kMaxI8K, "K above 131071 would overflow the int32 sums", EXO_B200_ERR_UNSUPPORTED)) return;
  const size_t e = f32 ? 4 : 2;
  Operands o(fn, ctxt);
  if (!o.in(X, mul(M, K, e), e)
           .in(B, mul(N, K, 1), 1)
           .in(col_scale, mul(N, 1, 4), 4)
           .maybe_in(bias, mul(N, 1, 4), 4)
           .out(Q, mul(M, K, 1), 1)
           .out(row_scale, mul(M, 1, 4), 4)
           .out(Y, mul(M, N, e), e)
           .stage())
    return;
  ffn::Problem p{};
  p.M = M, p.N = N, p.K = K;
  p.a0 = o.dev<void>(4), p.b0 = o.dev<void>(1);
  p.row_scale = o.dev<float>(5), p.col_scale = o.dev<float>(2), p.bias = o.dev<float>(3);
  p.c0 = o.dev<void>(6);
  cudaError_t err;
  if (ffn::linear_rows_wanted(p, f32)) {
    err = ffn::launch_linear_rows(o.ctx(), f32, p, o.dev<void>(0));
  } else {
    err = ffn::launch_quantize_rows(o.ctx(), M, K, o.dev<void>(0), !f32, o.dev<int8_t>(4), o.dev<float>(5));
    if (err == cudaSuccess) err = ffn::launch_product(o.ctx(), ffn::SCALED, f32, p, true);
  }
  o.done(err);
}

void gated(void* ctxt, int_fast32_t activation, int_fast32_t M, int_fast32_t F, int_fast32_t K,
                    const uint16_t* X, const uint16_t* Wg, const uint16_t* Wu, uint16_t* H, uint16_t* G, uint16_t* U) {
  const char* fn = "gated_bf16_exo";
  if (bad_act(fn, activation) || bad_sizes(fn, M, F, K, "M, F, K")) return;
  if (refuse(fn, !G != !U, "G and U are kept together: give both or neither")) return;
  Operands o(fn, ctxt);
  if (!o.in(X, mul(M, K, 2), 2)
           .in(Wg, mul(F, K, 2), 2)
           .in(Wu, mul(F, K, 2), 2)
           .out(H, mul(M, F, 2), 2)
           .maybe_out(G, mul(M, F, 2), 2)
           .maybe_out(U, mul(M, F, 2), 2)
           .stage())
    return;
  ffn::Problem p{};
  p.M = M, p.N = F, p.K = K;
  p.a0 = o.dev<void>(0), p.b0 = o.dev<void>(1), p.b1 = o.dev<void>(2);
  p.c0 = o.dev<void>(3), p.c1 = o.dev<void>(4), p.c2 = o.dev<void>(5);
  p.act = (int)activation;
  o.done(ffn::launch_product(o.ctx(), ffn::GATED, false, p, false));
}

void gated_backward(void* ctxt, int_fast32_t activation, int_fast32_t M, int_fast32_t F, int_fast32_t K,
                             const uint16_t* X, const uint16_t* Wg, const uint16_t* Wu, const uint16_t* G,
                             const uint16_t* U, const uint16_t* dH, uint16_t* dG, uint16_t* dU, uint16_t* dX,
                             uint16_t* dWg, uint16_t* dWu) {
  const char* fn = "gated_bf16_backward_exo";
  if (bad_act(fn, activation) || bad_sizes(fn, M, F, K, "M, F, K")) return;
  if (refuse(fn, !dWg != !dWu, "dWg and dWu are computed together: give both or neither")) return;
  Operands o(fn, ctxt);
  if (!o.in(X, mul(M, K, 2), 2)
           .in(Wg, mul(F, K, 2), 2)
           .in(Wu, mul(F, K, 2), 2)
           .in(G, mul(M, F, 2), 2)
           .in(U, mul(M, F, 2), 2)
           .in(dH, mul(M, F, 2), 2)
           .out(dG, mul(M, F, 2), 2)
           .out(dU, mul(M, F, 2), 2)
           .maybe_out(dX, mul(M, K, 2), 2)
           .maybe_out(dWg, mul(F, K, 2), 2)
           .maybe_out(dWu, mul(F, K, 2), 2)
           .stage())
    return;
  cudaError_t e = ffn::launch_gate_backward(o.ctx(), (int)activation, M * F, o.dev<uint16_t>(3), o.dev<uint16_t>(4),
                                            o.dev<uint16_t>(5), o.dev<uint16_t>(6), o.dev<uint16_t>(7));
  if (e == cudaSuccess)
    e = ffn::launch_gradients(o.ctx(), M, F, K, o.dev<void>(0), o.dev<void>(1), o.dev<void>(2), o.dev<void>(6),
                              o.dev<void>(7), o.dev<void>(8), o.dev<void>(9), o.dev<void>(10));
  o.done(e);
}

void gated_i8(void* ctxt, int_fast32_t activation, int_fast32_t M, int_fast32_t F, int_fast32_t K,
                       const int8_t* A, const int8_t* Bg, const int8_t* Bu, const float* row_scale,
                       const float* gate_scale, const float* up_scale, uint16_t* H) {
  const char* fn = "gated_i8_bf16_exo";
  if (bad_act(fn, activation) || bad_sizes(fn, M, F, K, "M, F, K")) return;
  if (refuse(fn, K > kMaxI8K, "K above 131071 would overflow the int32 sums", EXO_B200_ERR_UNSUPPORTED)) return;
  Operands o(fn, ctxt);
  if (!o.in(A, mul(M, K, 1), 1)
           .in(Bg, mul(F, K, 1), 1)
           .in(Bu, mul(F, K, 1), 1)
           .in(row_scale, mul(M, 1, 4), 4)
           .in(gate_scale, mul(F, 1, 4), 4)
           .in(up_scale, mul(F, 1, 4), 4)
           .out(H, mul(M, F, 2), 2)
           .stage())
    return;
  ffn::Problem p{};
  p.M = M, p.N = F, p.K = K;
  p.a0 = o.dev<void>(0), p.b0 = o.dev<void>(1), p.b1 = o.dev<void>(2);
  p.row_scale = o.dev<float>(3), p.col_scale = o.dev<float>(4), p.col_scale1 = o.dev<float>(5);
  p.c0 = o.dev<void>(6);
  p.act = (int)activation;
  o.done(ffn::launch_product(o.ctx(), ffn::GATED_I8, false, p, false));
}

}  // namespace

extern "C" {

void quantize_rows_bf16_exo(void* ctxt, int_fast32_t M, int_fast32_t K, const uint16_t* X, int8_t* Q, float* scale) {
  guarded("quantize_rows_bf16_exo", [&] { quantize("quantize_rows_bf16_exo", ctxt, M, K, X, true, Q, scale); });
}
void quantize_rows_f32_exo(void* ctxt, int_fast32_t M, int_fast32_t K, const float* X, int8_t* Q, float* scale) {
  guarded("quantize_rows_f32_exo", [&] { quantize("quantize_rows_f32_exo", ctxt, M, K, X, false, Q, scale); });
}

void gemm_i8_scaled_bf16_exo(void* ctxt, int_fast32_t M, int_fast32_t N, int_fast32_t K, const int8_t* A,
                             const int8_t* B, const float* row_scale, const float* col_scale, const float* bias,
                             uint16_t* C) {
  guarded("gemm_i8_scaled_bf16_exo", [&] {
    gemm_scaled("gemm_i8_scaled_bf16_exo", ctxt, M, N, K, A, B, row_scale, col_scale, bias, C, false);
  });
}
void gemm_i8_scaled_f32_exo(void* ctxt, int_fast32_t M, int_fast32_t N, int_fast32_t K, const int8_t* A,
                            const int8_t* B, const float* row_scale, const float* col_scale, const float* bias,
                            float* C) {
  guarded("gemm_i8_scaled_f32_exo", [&] {
    gemm_scaled("gemm_i8_scaled_f32_exo", ctxt, M, N, K, A, B, row_scale, col_scale, bias, C, true);
  });
}

void linear_i8_bf16_exo(void* ctxt, int_fast32_t M, int_fast32_t N, int_fast32_t K, const uint16_t* X, const int8_t* B,
                        const float* col_scale, const float* bias, int8_t* Q, float* row_scale, uint16_t* Y) {
  guarded("linear_i8_bf16_exo", [&] {
    linear("linear_i8_bf16_exo", ctxt, M, N, K, X, B, col_scale, bias, Q, row_scale, Y, false);
  });
}
void linear_i8_f32_exo(void* ctxt, int_fast32_t M, int_fast32_t N, int_fast32_t K, const float* X, const int8_t* B,
                       const float* col_scale, const float* bias, int8_t* Q, float* row_scale, float* Y) {
  guarded("linear_i8_f32_exo", [&] {
    linear("linear_i8_f32_exo", ctxt, M, N, K, X, B, col_scale, bias, Q, row_scale, Y, true);
  });
}

void gated_bf16_exo(void* ctxt, int_fast32_t activation, int_fast32_t M, int_fast32_t F, int_fast32_t K,
                    const uint16_t* X, const uint16_t* Wg, const uint16_t* Wu, uint16_t* H, uint16_t* G, uint16_t* U) {
  guarded("gated_bf16_exo", [&] { gated(ctxt, activation, M, F, K, X, Wg, Wu, H, G, U); });
}

void gated_bf16_backward_exo(void* ctxt, int_fast32_t activation, int_fast32_t M, int_fast32_t F, int_fast32_t K,
                             const uint16_t* X, const uint16_t* Wg, const uint16_t* Wu, const uint16_t* G,
                             const uint16_t* U, const uint16_t* dH, uint16_t* dG, uint16_t* dU, uint16_t* dX,
                             uint16_t* dWg, uint16_t* dWu) {
  guarded("gated_bf16_backward_exo",
          [&] { gated_backward(ctxt, activation, M, F, K, X, Wg, Wu, G, U, dH, dG, dU, dX, dWg, dWu); });
}

void gated_i8_bf16_exo(void* ctxt, int_fast32_t activation, int_fast32_t M, int_fast32_t F, int_fast32_t K,
                       const int8_t* A, const int8_t* Bg, const int8_t* Bu, const float* row_scale,
                       const float* gate_scale, const float* up_scale, uint16_t* H) {
  guarded("gated_i8_bf16_exo",
          [&] { gated_i8(ctxt, activation, M, F, K, A, Bg, Bu, row_scale, gate_scale, up_scale, H); });
}

}  // extern "C"
