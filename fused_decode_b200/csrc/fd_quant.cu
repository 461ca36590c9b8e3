// Rows to 8 bits (e4m3) with one fp32 scale per row, fused into the operator
// that produces the row: plain rows, RMSNorm / add+RMSNorm, SwiGLU.
//
//   a     = max(max_j |y_j|, 2^-64)
//   scale = a / 448                       (448: the largest finite e4m3 value)
//   q_j   = e4m3(y_j * (448 / a))         (to nearest even, saturating)
//
// y stays in fp32: it is rounded once, to 8 bits (half a step, relative 2^-4).
// The floor 2^-64 keeps 448 / a finite and gives a row of zeros a scale above
// zero and zeros as values.  A NaN anywhere in y makes the scale NaN.
//
// The row maximum is taken over the bit patterns of |y| as unsigned integers:
// they order like the values, and a NaN's pattern is above every number's, so
// it carries through where fmaxf would drop it.
#include "fd_rowgrid.cuh"

#include <cuda_fp8.h>

#include <algorithm>

using namespace fd;

namespace {

constexpr float kMax8 = 448.f;
constexpr float kAmaxFloor = 5.421010862427522e-20f;  // 2^-64

// What a row is before its quantisation.
enum RowOp { ROW_PLAIN = 0, ROW_RMS = 1, ROW_ADD_RMS = 2, ROW_SWIGLU = 3 };

struct QuantArgs {
  RowsArg x;   // plain, norms: the input; SwiGLU: gate
  RowsArg r;   // add+RMSNorm: residual; SwiGLU: up
  RowsArg q;   // e4m3 output
  RowsArg ro;  // add+RMSNorm: residual_out
  float* scale;  // one per row, in row order
  int64_t B, C, rows, n;
  const void* w;
  int32_t w_dtype;
  int64_t w_stride;
  float eps;
};

FD_DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The floor under the row maximum (a NaN stays one).
FD_DEV float floor_amax(float a) { return a <= kAmaxFloor ? kAmaxFloor : a; }

FD_DEV uint8_t to_e4m3(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

// ============================================================== any layout
// One CTA of 256 threads per row, element by element: any strides, any n.
// Bound by latency: the row is read once for its statistics and once more
// (from L1 or L2) to be written.
constexpr int kGenThreads = 256;

FD_DEV float block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < kGenThreads / 32; ++w) t += red[w];
  return t;
}

FD_DEV uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t t = 0;
  for (int w = 0; w < kGenThreads / 32; ++w) t = max(t, red[w]);
  return t;
}

template <typename T, int OP>
__global__ void __launch_bounds__(kGenThreads) quant_generic_kernel(QuantArgs a) {
  __shared__ float red_sum[kGenThreads / 32];
  __shared__ uint32_t red_max[kGenThreads / 32];
  const int64_t row = blockIdx.x;
  grid_dep_wait();
  grid_dep_launch();
  constexpr bool kNorm = OP == ROW_RMS || OP == ROW_ADD_RMS;
  constexpr bool kTwo = OP == ROW_ADD_RMS || OP == ROW_SWIGLU;
  const T* xr = row_ptr<T>(a.x, row, a.B, a.C);
  const T* rr = kTwo ? row_ptr<T>(a.r, row, a.B, a.C) : nullptr;
  // the row before the norm's scale and weight
  auto raw = [&](int64_t j) {
    const float v = to_f32(xr[j * a.x.col]);
    if (OP == ROW_ADD_RMS) return v + to_f32(rr[j * a.r.col]);
    if (OP == ROW_SWIGLU) return silu_mul(v, to_f32(rr[j * a.r.col]));
    return v;
  };
  float inv = 1.f;
  if (kNorm) {
    float sumsq = 0.f;
    for (int64_t j = threadIdx.x; j < a.n; j += kGenThreads) {
      const float s = raw(j);
      sumsq += s * s;
    }
    inv = rsqrtf(block_sum(sumsq, red_sum) / static_cast<float>(a.n) + a.eps);
  }
  auto value = [&](int64_t j, float s) {
    return kNorm ? s * inv * load_as_f32(a.w, a.w_dtype, j * a.w_stride) : s;
  };
  uint32_t top = 0;
  for (int64_t j = threadIdx.x; j < a.n; j += kGenThreads) top = max(top, abs_bits(value(j, raw(j))));
  const float amax = floor_amax(__uint_as_float(block_max(top, red_max)));
  const float up = kMax8 / amax;
  uint8_t* qr = row_ptr<uint8_t>(a.q, row, a.B, a.C);
  T* ror = OP == ROW_ADD_RMS ? row_ptr<T>(a.ro, row, a.B, a.C) : nullptr;
  for (int64_t j = threadIdx.x; j < a.n; j += kGenThreads) {
    const float s = raw(j);  // read before residual_out, which may be the residual itself
    if (OP == ROW_ADD_RMS) ror[j * a.ro.col] = from_f32<T>(s);
    qr[j * a.q.col] = to_e4m3(value(j, s) * up);
  }
  if (threadIdx.x == 0) a.scale[row] = amax / kMax8;
}

// ============================================================== host side
int from_cuda(cudaError_t e) { return e == cudaSuccess ? FD_OK : FD_ERR_LAUNCH; }

template <int OP>
int launch_quant(const fd_rows* x, const fd_rows* r, const fd_rows* q, const fd_rows* ro, float* scale, const void* w,
                 int32_t w_dtype, int64_t w_stride, float eps, void* stream) {
  using namespace fd_host;
  if (!x || !q || !scale) return FD_ERR_ARG;
  if (!half_dtype(x->dtype) || q->dtype != FD_E4M3 || !same_grid(x, q)) return FD_ERR_ARG;
  if ((OP == ROW_ADD_RMS || OP == ROW_SWIGLU) && (!r || !same_grid(x, r) || r->dtype != x->dtype)) return FD_ERR_ARG;
  if (OP == ROW_ADD_RMS && (!ro || !same_grid(x, ro) || ro->dtype != x->dtype)) return FD_ERR_ARG;
  if ((OP == ROW_RMS || OP == ROW_ADD_RMS) && (!valid_dtype(w_dtype) || (!w && x->n > 0))) return FD_ERR_ARG;
  const int64_t rows = x->a * x->b * x->c;
  if (rows <= 0 || x->n < 0) return FD_OK;
  if (rows > 0x7fffffffLL) return FD_ERR_UNSUPPORTED;
  QuantArgs a;
  a.x = rows_arg(x);
  a.r = rows_arg(r);
  a.q = rows_arg(q);
  a.ro = rows_arg(ro);
  a.scale = scale;
  a.B = x->b;
  a.C = x->c;
  a.rows = rows;
  a.n = x->n;
  a.w = w;
  a.w_dtype = w_dtype;
  a.w_stride = w_stride;
  a.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 blocks(static_cast<unsigned>(rows));
  return from_cuda(x->dtype == FD_BF16
                       ? launch_pdl(quant_generic_kernel<__nv_bfloat16, OP>, blocks, kGenThreads, 0, st, a)
                       : launch_pdl(quant_generic_kernel<__half, OP>, blocks, kGenThreads, 0, st, a));
}

}  // namespace

// ================================================================ C ABI
extern "C" {

int fd_quantize_fp8_out(const fd_rows* x, const fd_rows* out, float* scale, void* stream) {
  return launch_quant<ROW_PLAIN>(x, nullptr, out, nullptr, scale, nullptr, FD_F32, 0, 0.f, stream);
}

int fd_rms_fp8_out(const fd_rows* x, const fd_rows* residual, const void* weight, int32_t w_dtype, int64_t w_stride,
                   const fd_rows* out, float* scale, const fd_rows* residual_out, float eps, void* stream) {
  if (!residual != !residual_out) return FD_ERR_ARG;
  if (residual)
    return launch_quant<ROW_ADD_RMS>(x, residual, out, residual_out, scale, weight, w_dtype, w_stride, eps, stream);
  return launch_quant<ROW_RMS>(x, nullptr, out, nullptr, scale, weight, w_dtype, w_stride, eps, stream);
}

int fd_swiglu_fp8_out(const fd_rows* gate, const fd_rows* up, const fd_rows* out, float* scale, void* stream) {
  return launch_quant<ROW_SWIGLU>(gate, up, out, nullptr, scale, nullptr, FD_F32, 0, 0.f, stream);
}

}  // extern "C"
