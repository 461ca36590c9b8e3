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
// Maxima keep a NaN: max.NaN between a thread's elements, and between lanes the
// bit patterns of the magnitudes as unsigned integers, which order like the
// values with a NaN's above every number's.
#include "fd_rowgrid.cuh"

#include <cuda_fp8.h>

#include <algorithm>

using namespace fd;

namespace {

constexpr float kMax8 = 448.f;
constexpr float kAmaxFloor = 5.421010862427522e-20f;  // 2^-64

// What a row is before its quantisation.
enum RowOp { ROW_PLAIN = 0, ROW_RMS = 1, ROW_ADD_RMS = 2, ROW_SWIGLU = 3 };

// Whether the next kernel on the stream may start before this one has finished.
// Not behind residual_out: a 16-bit tensor may be the weight of a linear_decode,
// which streams its weight before it waits.  add_rms_norm_fp8 of one row and the
// 8-bit product behind it, 4096 x 4096: 9.7 us, with an early start 8.4; with a
// start behind a fence 9.8.
template <int OP>
constexpr bool kEarlyNext = OP != ROW_ADD_RMS;

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

// silu(g) * u by the hardware's exp2 and reciprocal, flushing subnormals: for
// g towards -inf the exponential overflows to infinity and the sigmoid to 0.
// The exponential's error grows with its argument: relative 2^-22 and
// |g| 2^-24, where the row is rounded to 2^-4.
FD_DEV float silu_mul_fast(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r * u;
}

// max(a, |b|) that keeps a NaN.
FD_DEV float max_abs(float a, float b) {
  float v;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(fabsf(b)));
  return v;
}

// The floor under the row maximum (a NaN stays one).
FD_DEV float floor_amax(float a) { return a <= kAmaxFloor ? kAmaxFloor : a; }

FD_DEV uint8_t to_e4m3(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }

// ============================================================== any layout
// One CTA per row, element by element: any strides, any n.  A row of up to
// THREADS * EACH elements stays in registers; of a longer one the rest is read
// again (from L1 or L2) for the maximum and for the values.  Coalesced where the
// elements are contiguous, so rows that vectors cannot address (odd widths, odd
// offsets) still stream: SwiGLU of 2100 x 14335 76 us, add_rms_norm_fp8 of 8192 x
// 4095 75 us.
FD_DEV float block_sum(float v, int warps, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < warps; ++w) t += red[w];
  return t;
}

FD_DEV float block_max(float v, int warps, float* red) {
  v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < warps; ++w) t = max_abs(t, red[w]);
  return t;
}

template <typename T, int OP, int THREADS, int EACH, bool CONTIG>
__global__ void __launch_bounds__(THREADS) quant_generic_kernel(QuantArgs a) {
  __shared__ float red_sum[32], red_max[32];
  constexpr int warps = THREADS / 32;
  const int64_t row = blockIdx.x;
  grid_dep_wait();
  if (kEarlyNext<OP>) grid_dep_launch();
  constexpr bool kNorm = OP == ROW_RMS || OP == ROW_ADD_RMS;
  constexpr bool kTwo = OP == ROW_ADD_RMS || OP == ROW_SWIGLU;
  const T* xr = row_ptr<T>(a.x, row, a.B, a.C);
  const T* rr = kTwo ? row_ptr<T>(a.r, row, a.B, a.C) : nullptr;
  uint8_t* qr = row_ptr<uint8_t>(a.q, row, a.B, a.C);
  T* ror = OP == ROW_ADD_RMS ? row_ptr<T>(a.ro, row, a.B, a.C) : nullptr;
  // element j of a row with last-dimension stride col (1 where CONTIG)
  auto at = [](int64_t j, int64_t col) { return CONTIG ? j : j * col; };
  // the row before the norm's scale and weight
  auto raw = [&](int64_t j) {
    const float v = to_f32(xr[at(j, a.x.col)]);
    if (OP == ROW_ADD_RMS) return v + to_f32(rr[at(j, a.r.col)]);
    if (OP == ROW_SWIGLU) return silu_mul_fast(v, to_f32(rr[at(j, a.r.col)]));
    return v;
  };
  const int n = static_cast<int>(min(a.n, static_cast<int64_t>(THREADS) * EACH));  // elements in registers
  const int t = threadIdx.x;
  float s[EACH], w[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) s[i] = t + i * THREADS < n ? raw(t + i * THREADS) : 0.f;
  if (kNorm) {
    auto weights = [&](auto* p) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) w[i] = t + i * THREADS < n ? to_f32(p[at(t + i * THREADS, a.w_stride)]) : 0.f;
    };
    if (a.w_dtype == FD_F32) weights(static_cast<const float*>(a.w));
    else if (a.w_dtype == FD_BF16) weights(static_cast<const __nv_bfloat16*>(a.w));
    else weights(static_cast<const __half*>(a.w));
  }
  const int64_t rest = t + static_cast<int64_t>(EACH) * THREADS;
  float inv = 1.f;
  if (kNorm) {
    float sumsq = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) sumsq += s[i] * s[i];
    for (int64_t j = rest; j < a.n; j += THREADS) {
      const float v = raw(j);
      sumsq += v * v;
    }
    inv = rsqrtf(block_sum(sumsq, warps, red_sum) / static_cast<float>(a.n) + a.eps);
  }
  auto value = [&](int64_t j, float v) {
    return kNorm ? v * inv * load_as_f32(a.w, a.w_dtype, j * a.w_stride) : v;
  };
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (t + i * THREADS < n) top = max_abs(top, kNorm ? s[i] * inv * w[i] : s[i]);
  for (int64_t j = rest; j < a.n; j += THREADS) top = max_abs(top, value(j, raw(j)));
  const float amax = floor_amax(block_max(top, warps, red_max));
  const float up = kMax8 / amax;
  // every element was read before its residual_out, which may be the residual itself
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int j = t + i * THREADS;
    if (j < n) {
      if (OP == ROW_ADD_RMS) ror[at(j, a.ro.col)] = from_f32<T>(s[i]);
      qr[at(j, a.q.col)] = to_e4m3((kNorm ? s[i] * inv * w[i] : s[i]) * up);
    }
  }
  for (int64_t j = rest; j < a.n; j += THREADS) {
    const float v = raw(j);
    if (OP == ROW_ADD_RMS) ror[at(j, a.ro.col)] = from_f32<T>(v);
    qr[at(j, a.q.col)] = to_e4m3(value(j, v) * up);
  }
  if (t == 0) a.scale[row] = amax / kMax8;
}

// ============================================================== vectors of 8
// Rows of 16-byte vectors, each handled by `wpr` warps: every thread keeps VPT
// vectors of the row in registers, so the inputs are read from HBM once.  The
// norm needs the sum of squares before any y is known; since
// max|s * inv * w| = inv * max|s * w|, both reductions run over the row
// together, at the price of one more pass over the registers for a row whose
// s * w is not finite.  Bound by HBM for many rows, by one round trip to memory
// and the reduction for few.
struct QuantVecArgs {
  QuantArgs g;
  int32_t wpr;  // warps per row
  int32_t rpc;  // rows per CTA
  int32_t nv;   // vectors per row
};

struct RowStats {
  float sum;
  float top;  // maximum of the magnitudes
};

// Sum and maximum over the warps of a row's group; every warp of the CTA takes part.
FD_DEV RowStats group_reduce(RowStats s, int wpr, int group, float* red_sum, float* red_top) {
  s.sum = warp_sum(s.sum);
  s.top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(s.top)));
  if (wpr > 1) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) {
      red_sum[warp] = s.sum;
      red_top[warp] = s.top;
    }
    __syncthreads();
    s = {0.f, 0.f};
    for (int w = 0; w < wpr; ++w) {
      s.sum += red_sum[group * wpr + w];
      s.top = max_abs(s.top, red_top[group * wpr + w]);
    }
  }
  return s;
}

FD_DEV uint2 pack8_e4m3(const float* f) {
  auto two = [](float a, float b) -> uint32_t {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  };
  return make_uint2(two(f[0], f[1]) | two(f[2], f[3]) << 16, two(f[4], f[5]) | two(f[6], f[7]) << 16);
}

// A row in registers, VPT vectors to a thread (vector j = t + i * threads): its
// statistics, then its values.
template <typename T, int OP, int VPT>
struct RowRegs {
  static constexpr bool kNorm = OP == ROW_RMS || OP == ROW_ADD_RMS;
  static constexpr bool kTwo = OP == ROW_ADD_RMS || OP == ROW_SWIGLU;
  float s[VPT][8];  // the row before the norm's scale and weight
  uint4 w16[VPT];   // the norm weight, where it is of 16 bits

  // issued with the row's loads, not after they have arrived
  FD_DEV void ask_weight(const QuantArgs& g, int i, int j) {
    if (kNorm && g.w_dtype != FD_F32) w16[i] = __ldg(static_cast<const uint4*>(g.w) + j);
  }
  FD_DEV void weight(const QuantArgs& g, int i, int j, float* w) const {
    if (g.w_dtype == FD_F32) load8_as_f32(static_cast<const float*>(g.w) + 8 * j, FD_F32, w);
    else if (g.w_dtype == FD_BF16) unpack8<__nv_bfloat16>(w16[i], w);
    else unpack8<__half>(w16[i], w);
  }
  // vector i (the row's vector j) from its packed inputs
  FD_DEV void take(const QuantArgs& g, int i, int j, const uint4& x, const uint4& r, RowStats* st) {
    unpack8<T>(x, s[i]);
    if (kTwo) {
      float f[8];
      unpack8<T>(r, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[i][e] = OP == ROW_SWIGLU ? silu_mul_fast(s[i][e], f[e]) : s[i][e] + f[e];
    }
    if (kNorm) {
      float w[8];
      weight(g, i, j, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        st->sum += s[i][e] * s[i][e];
        st->top = max_abs(st->top, s[i][e] * w[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) st->top = max_abs(st->top, s[i][e]);
    }
  }
  // (row maximum, 1 / rms) from the row's statistics.  Where s * w overflowed,
  // or holds an infinity or a NaN, `again` reduces the maximum of the products
  // themselves, as the definition orders them.
  template <typename Again>
  FD_DEV float amax(const QuantArgs& g, RowStats st, int t, int threads, int nv, bool live, float* inv, Again again) {
    if (!kNorm) return st.top;
    *inv = rsqrtf(st.sum / static_cast<float>(g.n) + g.eps);
    if (st.top < __uint_as_float(0x7f800000u)) return st.top * *inv;
    RowStats more{0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = t + i * threads;
      if (live && j < nv) {
        float w[8];
        weight(g, i, j, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) more.top = max_abs(more.top, s[i][e] * *inv * w[e]);
      }
    }
    return again(more).top;
  }
  FD_DEV void put(const QuantArgs& g, int i, int j, float inv, float up, uint8_t* q) const {
    float o[8];
    if (kNorm) {
      float w[8];
      weight(g, i, j, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = s[i][e] * inv * w[e] * up;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = s[i][e] * up;
    }
    *reinterpret_cast<uint2*>(q + 8 * j) = pack8_e4m3(o);
  }
};

template <typename T, int OP, int VPT, bool FLAT>
__global__ void __launch_bounds__(1024) quant_vec_kernel(QuantVecArgs a) {
  __shared__ float red_sum[2][32], red_top[2][32];
  using Row = RowRegs<T, OP, VPT>;
  const int group_threads = 32 * a.wpr;
  const int group = threadIdx.x / group_threads;
  const int t = threadIdx.x - group * group_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * a.rpc + group;
  const bool live = row < a.g.rows;
  const RowIdx ri = split_row<FLAT>(live ? row : 0, a.g.B, a.g.C);
  grid_dep_wait();
  if (kEarlyNext<OP>) grid_dep_launch();

  Row v;
  RowStats st{0.f, 0.f};
  if (live) {
    const T* xr = reinterpret_cast<const T*>(a.g.x.ptr) + offset_of(a.g.x, ri);
    const T* rr = Row::kTwo ? reinterpret_cast<const T*>(a.g.r.ptr) + offset_of(a.g.r, ri) : nullptr;
    uint4 xv[VPT], rv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = t + i * group_threads;
      if (j < a.nv) {
        xv[i] = ld_plain16(xr + 8 * j);
        if (Row::kTwo) rv[i] = ld_plain16(rr + 8 * j);
        v.ask_weight(a.g, i, j);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = t + i * group_threads;
      if (j < a.nv) v.take(a.g, i, j, xv[i], rv[i], &st);
    }
    if (OP == ROW_ADD_RMS) {
      T* ror = reinterpret_cast<T*>(a.g.ro.ptr) + offset_of(a.g.ro, ri);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = t + i * group_threads;
        if (j < a.nv) st_stream16(ror + 8 * j, pack8<T>(v.s[i]));
      }
    }
  }
  st = group_reduce(st, a.wpr, group, red_sum[0], red_top[0]);
  // With one warp a row, whether the maximum is reduced again may differ
  // between a CTA's rows, and stays within the warp; with more there is one row
  // to a CTA.
  float inv = 1.f;
  const float amax = floor_amax(v.amax(a.g, st, t, group_threads, a.nv, live, &inv, [&](RowStats more) {
    return group_reduce(more, a.wpr, group, red_sum[1], red_top[1]);
  }));
  if (!live) return;
  const float up = kMax8 / amax;
  uint8_t* qr = reinterpret_cast<uint8_t*>(a.g.q.ptr) + offset_of(a.g.q, ri);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = t + i * group_threads;
    if (j < a.nv) v.put(a.g, i, j, inv, up, qr);
  }
  if (t == 0) a.g.scale[row] = amax / kMax8;
}

// ============================================================== host side
int from_cuda(cudaError_t e) { return e == cudaSuccess ? FD_OK : FD_ERR_LAUNCH; }

// e4m3 rows that can be written 8 values at a time.
bool rows_vec8(const fd_rows* q) {
  if (q->col != 1 || reinterpret_cast<uintptr_t>(q->ptr) % 8) return false;
  return !((q->a > 1 && q->sa % 8) || (q->b > 1 && q->sb % 8) || (q->c > 1 && q->sc % 8));
}

template <typename T, int OP, int VPT>
cudaError_t launch_vec2(const QuantVecArgs& a, bool flat, cudaStream_t st) {
  const dim3 threads(32 * a.wpr * a.rpc);
  const dim3 blocks(static_cast<unsigned>((a.g.rows + a.rpc - 1) / a.rpc));
  return flat ? fd_host::launch_pdl(quant_vec_kernel<T, OP, VPT, true>, blocks, threads, 0, st, a)
              : fd_host::launch_pdl(quant_vec_kernel<T, OP, VPT, false>, blocks, threads, 0, st, a);
}

// Vectors per thread and warps per row, nv <= 4096.  Many rows run best with four
// vectors to a thread (add_rms_norm_fp8 8192 x 4096: 42.2 us, with one, two or
// eight 59, 45, 49).  Few rows run best with many threads (1 x 4096: 2.3 us, with
// four vectors 3.3): one vector each where 16 warps then hold the row, else two,
// else four as for many rows (8 x 14336: 14 warps, 3.2 us).
template <typename T, int OP>
cudaError_t launch_vec(QuantVecArgs a, bool flat, cudaStream_t st) {
  const int nv = a.nv;
  a.wpr = 1;
  a.rpc = 4;
  if (nv <= 32) return launch_vec2<T, OP, 1>(a, flat, st);
  if (nv <= 64) return launch_vec2<T, OP, 2>(a, flat, st);
  a.rpc = 1;
  auto warps = [&](int vpt) { return (nv + 32 * vpt - 1) / (32 * vpt); };
  const bool few = a.g.rows <= fd_host::sm_count();
  if (few && warps(1) <= 16) {
    a.wpr = warps(1);
    return launch_vec2<T, OP, 1>(a, flat, st);
  }
  if (few && warps(2) <= 16) {
    a.wpr = warps(2);
    return launch_vec2<T, OP, 2>(a, flat, st);
  }
  a.wpr = warps(4);  // <= 32
  return launch_vec2<T, OP, 4>(a, flat, st);
}

// Threads and register elements for a row of any layout: enough for the row, or
// the most there are; with more rows than SMs fewer threads with more elements,
// so that several rows share an SM.
template <typename T, int OP, bool CONTIG>
cudaError_t launch_generic(const QuantArgs& a, cudaStream_t st) {
  auto go = [&](auto* kernel, int threads) {
    return fd_host::launch_pdl(kernel, dim3(static_cast<unsigned>(a.rows)), dim3(threads), 0, st, a);
  };
  const bool many = a.rows > fd_host::sm_count();
  if (a.n <= 1024) return go(quant_generic_kernel<T, OP, 128, 8, CONTIG>, 128);
  if (many && a.n <= 4096) return go(quant_generic_kernel<T, OP, 256, 16, CONTIG>, 256);
  if (many && a.n <= 8192) return go(quant_generic_kernel<T, OP, 512, 16, CONTIG>, 512);
  if (a.n <= 8192) return go(quant_generic_kernel<T, OP, 1024, 8, CONTIG>, 1024);
  return go(quant_generic_kernel<T, OP, 1024, 16, CONTIG>, 1024);
}

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
  const bool norm = OP == ROW_RMS || OP == ROW_ADD_RMS;
  if (x->n > 0 && x->n % 8 == 0 && x->n <= 32768 && rows_vec16(x) && rows_vec8(q) &&
      (OP == ROW_PLAIN || OP == ROW_RMS || rows_vec16(r)) && (OP != ROW_ADD_RMS || rows_vec16(ro)) &&
      (!norm || (w_stride == 1 && aligned16(w)))) {
    const QuantVecArgs v{a, 1, 1, static_cast<int32_t>(x->n / 8)};
    const bool flat = x->a == 1 && x->b == 1;
    return from_cuda(x->dtype == FD_BF16 ? launch_vec<__nv_bfloat16, OP>(v, flat, st)
                                         : launch_vec<__half, OP>(v, flat, st));
  }
  const bool contig = x->col == 1 && q->col == 1 && (!r || r->col == 1) && (!ro || ro->col == 1) && (!norm || w_stride == 1);
  const bool bf = x->dtype == FD_BF16;
  if (contig)
    return from_cuda(bf ? launch_generic<__nv_bfloat16, OP, true>(a, st) : launch_generic<__half, OP, true>(a, st));
  return from_cuda(bf ? launch_generic<__nv_bfloat16, OP, false>(a, st) : launch_generic<__half, OP, false>(a, st));
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
