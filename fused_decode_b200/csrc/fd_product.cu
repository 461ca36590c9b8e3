// Matrix products with an epilogue, any number of rows:
//   y[m, n] = round(act(sum_k x[m, k] w[n, k] (* xs[m] * ws[n]) + bias[n]) + row_add[m, n])
// 16-bit operands (f16 or bf16), or e4m3 operands with one fp32 scale per row
// of x and per row of w.  Sums are fp32; the result is rounded once.
#include "fd_stream.cuh"

#include <cuda_fp8.h>

#include <algorithm>

using namespace fd;

namespace {

using fd_stream::mma16816;

// ============================================================== epilogue
struct Epilogue {
  const float* xs;  // e4m3 operands: scale of each row of x (nullptr: none)
  const float* ws;  //                and of each row of w
  const void* bias;
  int32_t bias_dtype;
  int64_t sbias;
  const void* ra;
  int32_t ra_dtype;
  int64_t srm, srn;
  void* y;
  int64_t sym, syn;
  int64_t m, n;
  int32_t act;
};

// v * sigmoid(z), with exp(-|z|) so that nothing overflows (see silu_mul for
// the accuracy of __expf and __fdividef).
FD_DEV float gated(float v, float z) {
  const float e = __expf(-fabsf(z));
  const float r = __fdividef(1.0f, 1.0f + e);
  return v * (z >= 0.f ? r : e * r);
}

FD_DEV float activate(float v, int act) {
  switch (act) {
    case FD_ACT_RELU: return v < 0.f ? 0.f : v;  // a NaN stays one
    case FD_ACT_SILU: return gated(v, v);
    case FD_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    // 0.5 v (1 + tanh(u)) = v sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3)
    case FD_ACT_GELU_TANH: return gated(v, 1.5957691216057308f * (v + 0.044715f * v * v * v));
    default: return v;
  }
}

// One output element from its fp32 sum.  row_add is read before y is written
// by the same thread, so y may be row_add.
template <typename T, bool FP8>
FD_DEV void finish(const Epilogue& e, int64_t m, int64_t n, float v) {
  if (FP8) v = v * e.xs[m] * e.ws[n];
  if (e.bias) v += load_as_f32(e.bias, e.bias_dtype, n * e.sbias);
  v = activate(v, e.act);
  if (e.ra) v += load_as_f32(e.ra, e.ra_dtype, m * e.srm + n * e.srn);
  static_cast<T*>(e.y)[m * e.sym + n * e.syn] = from_f32<T>(v);
}

// ============================================================== any layout
// Any strides, alignments and sizes: 64 x 64 tiles of y, operands gathered
// element by element into shared memory, mma.sync m16n8k16 (four warps of
// 32 x 32).  e4m3 operands are widened to f16, which holds every e4m3 value.
// For layouts that TMA cannot address; bound by the scalar loads.
struct GenericArgs {
  const void* x;
  int64_t sxm, sxk;
  const void* w;
  int64_t swn, swk;
  int64_t k;
  Epilogue epi;
};

constexpr int kGenTile = 64;
constexpr int kGenK = 32;
constexpr int kGenPitch = kGenK + 8;  // 80-byte rows: the eight rows of a fragment load fall in eight bank groups

template <bool FP8>
FD_DEV uint16_t load_operand(const void* p, int64_t i) {
  if (FP8) return __nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(p)[i], __NV_E4M3).x;
  return static_cast<const uint16_t*>(p)[i];
}

// TX: element type of the 16-bit operands (f16 for e4m3).  T: output.
template <typename TX, typename T, bool FP8>
__global__ void __launch_bounds__(128) product_generic_kernel(GenericArgs a) {
  __shared__ __align__(16) uint16_t xt[kGenTile][kGenPitch];
  __shared__ __align__(16) uint16_t wt[kGenTile][kGenPitch];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q = lane & 3;
  const int wm = (warp & 1) * 32, wn = (warp >> 1) * 32;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kGenTile;
  grid_dep_wait();
  grid_dep_launch();
  for (int64_t m0 = static_cast<int64_t>(blockIdx.y) * kGenTile; m0 < a.epi.m;
       m0 += static_cast<int64_t>(gridDim.y) * kGenTile) {
    float acc[2][4][4] = {};
    for (int64_t k0 = 0; k0 < a.k; k0 += kGenK) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kGenTile * kGenK / 128; ++i) {
        const int r = (tid + i * 128) / kGenK, c = (tid + i * 128) % kGenK;
        const int64_t kk = k0 + c;
        xt[r][c] = m0 + r < a.epi.m && kk < a.k ? load_operand<FP8>(a.x, (m0 + r) * a.sxm + kk * a.sxk) : 0;
        wt[r][c] = n0 + r < a.epi.n && kk < a.k ? load_operand<FP8>(a.w, (n0 + r) * a.swn + kk * a.swk) : 0;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kGenK; kk += 16) {
        uint32_t fa[2][4], fb[4][2];
        auto word = [&](const uint16_t (*t)[kGenPitch], int r, int c) {
          return *reinterpret_cast<const uint32_t*>(&t[r][c]);
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = wm + 16 * i + g;
          fa[i][0] = word(xt, r, kk + 2 * q);
          fa[i][1] = word(xt, r + 8, kk + 2 * q);
          fa[i][2] = word(xt, r, kk + 2 * q + 8);
          fa[i][3] = word(xt, r + 8, kk + 2 * q + 8);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = wn + 8 * j + g;
          fb[j][0] = word(wt, r, kk + 2 * q);
          fb[j][1] = word(wt, r, kk + 2 * q + 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma16816<TX>(acc[i][j], fa[i][0], fa[i][1], fa[i][2], fa[i][3], fb[j][0], fb[j][1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int64_t m = m0 + wm + 16 * i + g + 8 * (c >> 1);
          const int64_t n = n0 + wn + 8 * j + 2 * q + (c & 1);
          if (m < a.epi.m && n < a.epi.n) finish<T, FP8>(a.epi, m, n, acc[i][j][c]);
        }
  }
}

// ============================================================== host side
int from_cuda(cudaError_t e) { return e == cudaSuccess ? FD_OK : FD_ERR_LAUNCH; }

template <typename TX, typename T, bool FP8>
int launch_generic(const GenericArgs& a, cudaStream_t st) {
  const int64_t nb = (a.epi.n + kGenTile - 1) / kGenTile, mb = (a.epi.m + kGenTile - 1) / kGenTile;
  if (nb > 0x7fffffffLL) return FD_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(nb), static_cast<unsigned>(std::min<int64_t>(mb, 65535)));
  return from_cuda(fd_host::launch_pdl(product_generic_kernel<TX, T, FP8>, grid, 128, 0, st, a));
}

bool epilogue_ok(const Epilogue& e) {
  return e.y && fd_host::valid_dtype(e.bias_dtype) && fd_host::valid_dtype(e.ra_dtype) && e.act >= FD_ACT_NONE &&
         e.act <= FD_ACT_GELU_TANH;
}

// in_dtype: f16, bf16 or e4m3 (then e.xs and e.ws are set and out_dtype is the
// output's; for 16-bit operands out_dtype = in_dtype).
int product(const GenericArgs& a, int in_dtype, int out_dtype, cudaStream_t st) {
  const Epilogue& e = a.epi;
  if (e.m < 0 || e.n < 0 || a.k < 0) return FD_ERR_ARG;
  if (e.m == 0 || e.n == 0) return FD_OK;
  if (!epilogue_ok(e) || !fd_host::half_dtype(out_dtype) || (a.k > 0 && (!a.x || !a.w))) return FD_ERR_ARG;
  const bool bf = out_dtype == FD_BF16;
  if (in_dtype == FD_E4M3)
    return bf ? launch_generic<__half, __nv_bfloat16, true>(a, st) : launch_generic<__half, __half, true>(a, st);
  return bf ? launch_generic<__nv_bfloat16, __nv_bfloat16, false>(a, st)
            : launch_generic<__half, __half, false>(a, st);
}

// ---- post_attn_mlp_fp8's intermediates in the caller's workspace
struct MlpBuffers {
  size_t q, scale, gate_up, mid, mid_scale, bytes;
};
MlpBuffers mlp_buffers(int64_t m, int64_t h, int64_t i) {
  auto up = [](size_t v) { return (v + 255) & ~size_t{255}; };
  MlpBuffers b;
  b.q = 0;
  b.scale = b.q + up(static_cast<size_t>(m) * h);
  b.gate_up = b.scale + up(static_cast<size_t>(m) * 4);
  b.mid = b.gate_up + up(static_cast<size_t>(m) * 2 * i * 2);
  b.mid_scale = b.mid + up(static_cast<size_t>(m) * i);
  b.bytes = b.mid_scale + up(static_cast<size_t>(m) * 4);
  return b;
}

}  // namespace

// ================================================================ C ABI
extern "C" {

int fd_linear_act_out(const void* x, int64_t sxm, int64_t sxk, const void* w, int64_t swn, int64_t swk,
                      const void* bias, int32_t bias_dtype, int64_t sbias, const void* row_add, int32_t ra_dtype,
                      int64_t srm, int64_t srn, void* y, int64_t sym, int64_t syn, int32_t dtype, int32_t act,
                      int64_t m, int64_t n, int64_t k, void* stream) {
  if (!fd_host::half_dtype(dtype)) return FD_ERR_ARG;
  const Epilogue e{nullptr, nullptr, bias, bias_dtype, sbias, row_add, ra_dtype, srm, srn, y, sym, syn, m, n, act};
  return product({x, sxm, sxk, w, swn, swk, k, e}, dtype, dtype, static_cast<cudaStream_t>(stream));
}

int fd_linear_fp8_out(const void* x, int64_t sxm, int64_t sxk, const float* x_scale, const void* w, int64_t swn,
                      int64_t swk, const float* w_scale, const void* bias, int32_t bias_dtype, int64_t sbias,
                      const void* row_add, int32_t ra_dtype, int64_t srm, int64_t srn, void* y, int64_t sym,
                      int64_t syn, int32_t out_dtype, int32_t act, int64_t m, int64_t n, int64_t k, void* stream) {
  if (m > 0 && n > 0 && (!x_scale || !w_scale)) return FD_ERR_ARG;
  const Epilogue e{x_scale, w_scale, bias, bias_dtype, sbias, row_add, ra_dtype, srm, srn, y, sym, syn, m, n, act};
  return product({x, sxm, sxk, w, swn, swk, k, e}, FD_E4M3, out_dtype, static_cast<cudaStream_t>(stream));
}

size_t fd_post_attn_mlp_fp8_workspace_bytes(int64_t m, int64_t h, int64_t i) {
  if (m < 0 || h < 0 || i < 0) return 0;
  return mlp_buffers(m, h, i).bytes;
}

int fd_post_attn_mlp_fp8_out(const void* hidden, int64_t s_hidden, const void* norm_w, int32_t norm_dtype,
                             int64_t s_norm, const void* w_gate_up, int64_t s_gu, const float* gate_up_scale,
                             const void* w_down, int64_t s_down, const float* down_scale, void* out, int32_t dtype,
                             int64_t m, int64_t h, int64_t i, float eps, void* workspace, size_t workspace_bytes,
                             void* stream) {
  if (m < 0 || h < 0 || i < 0 || !fd_host::half_dtype(dtype)) return FD_ERR_ARG;
  if (m == 0 || h == 0) return FD_OK;
  if (i == 0 || !hidden || !norm_w || !w_gate_up || !gate_up_scale || !w_down || !down_scale || !out)
    return FD_ERR_ARG;
  const MlpBuffers b = mlp_buffers(m, h, i);
  if (!workspace || !fd_host::aligned16(workspace) || workspace_bytes < b.bytes) return FD_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  auto grid = [&](void* p, int dt, int64_t stride, int64_t n) {
    return fd_rows{p, dt, 0, 1, 1, m, 0, 0, stride, 1, n};
  };
  float* scale = reinterpret_cast<float*>(ws + b.scale);
  float* mid_scale = reinterpret_cast<float*>(ws + b.mid_scale);
  char* gu = ws + b.gate_up;
  const fd_rows rx = grid(const_cast<void*>(hidden), dtype, s_hidden, h), rq = grid(ws + b.q, FD_E4M3, h, h);
  const fd_rows rg = grid(gu, dtype, 2 * i, i), ru = grid(gu + 2 * i, dtype, 2 * i, i);
  const fd_rows rm = grid(ws + b.mid, FD_E4M3, i, i);
  int r = fd_rms_fp8_out(&rx, nullptr, norm_w, norm_dtype, s_norm, &rq, scale, nullptr, eps, stream);
  if (r == FD_OK)
    r = fd_linear_fp8_out(ws + b.q, h, 1, scale, w_gate_up, s_gu, 1, gate_up_scale, nullptr, 0, 0, nullptr, 0, 0, 0,
                          gu, 2 * i, 1, dtype, FD_ACT_NONE, m, 2 * i, h, stream);
  if (r == FD_OK) r = fd_swiglu_fp8_out(&rg, &ru, &rm, mid_scale, stream);
  if (r == FD_OK)
    r = fd_linear_fp8_out(ws + b.mid, i, 1, mid_scale, w_down, s_down, 1, down_scale, nullptr, 0, 0, hidden, dtype,
                          s_hidden, 1, out, h, 1, dtype, FD_ACT_NONE, m, h, i, stream);
  return r;
}

}  // extern "C"
