// Matrix products with an epilogue, any number of rows:
//   y[m, n] = round(act(sum_k x[m, k] w[n, k] (* xs[m] * ws[n]) + bias[n]) + row_add[m, n])
// 16-bit operands (f16 or bf16), or e4m3 operands with one fp32 scale per row
// of x and per row of w.  Sums are fp32; the result is rounded once.
#include "fd_stream.cuh"

#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

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

template <typename T>
FD_DEV constexpr int dtype_of() {
  return std::is_same<T, __nv_bfloat16>::value ? FD_BF16 : FD_F16;
}

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

// ============================================================== tensor cores
// Shared by the two tcgen05 kernels below.  Both operands lie row by row along
// K, in shared-memory tiles of 128-byte rows (64 16-bit or 128 8-bit elements)
// with the 128-byte swizzle TMA writes; one instruction takes 32 bytes of K.
constexpr int kBoxBytes = 128;  // K bytes of a tile row
constexpr int kMaxRing = 12;
constexpr int kSliceBytes = 32;  // K bytes of one tcgen05.mma

// None of the product kernels lets the next kernel start before it has finished
// (grid_dep_launch): y may be the weight of a linear_decode, which streams its
// weight before it waits.  It costs 0.9 us between products of 4096 x 4096.
constexpr int kStatusWait = 1;  // a bounded wait expired: the call's output is invalid
__device__ int g_product_status;

// Shared-memory descriptor of a K-major tile: start address / 16, rows of 8
// (1024 bytes) apart, descriptor version 1, 128-byte swizzle.
FD_DEV uint64_t tile_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (uint64_t{1} << 16) | (uint64_t{1024 >> 4} << 32) |
         (uint64_t{1} << 46) | (uint64_t{2} << 61);
}

// Instruction descriptor: fp32 accumulator, both operands K-major of one
// element format (kind::f16: 0 f16, 1 bf16; kind::f8f6f4: 0 e4m3), rows x cols.
inline uint32_t mma_desc(int format, int rows, int cols) {
  return (1u << 4) | (static_cast<uint32_t>(format) << 7) | (static_cast<uint32_t>(format) << 10) |
         (static_cast<uint32_t>(cols >> 3) << 17) | (static_cast<uint32_t>(rows >> 4) << 24);
}

template <int CTAS>
FD_DEV void tmem_alloc(uint32_t* slot, uint32_t cols) {
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fd_stream::smem_addr(slot)),
                 "r"(cols)
                 : "memory");
  else
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fd_stream::smem_addr(slot)),
                 "r"(cols)
                 : "memory");
}
template <int CTAS>
FD_DEV void tmem_free(uint32_t addr, uint32_t cols) {
  if constexpr (CTAS == 1) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
  } else {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
  }
}
FD_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
FD_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// d (+)= a b^T over one 32-byte slice of K; issued by one thread.
template <bool FP8, int CTAS>
FD_DEV void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, bool add) {
#define FD_TC_MMA(group, kind)                                                                              \
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::" group ".kind::" kind       \
               " [%0], %1, %2, %3, p;\n}" ::"r"(d),                                                         \
               "l"(a), "l"(b), "r"(desc), "r"(static_cast<int>(add))                                        \
               : "memory")
  if constexpr (FP8 && CTAS == 1) FD_TC_MMA("1", "f8f6f4");
  else if constexpr (FP8) FD_TC_MMA("2", "f8f6f4");
  else if constexpr (CTAS == 1) FD_TC_MMA("1", "f16");
  else FD_TC_MMA("2", "f16");
#undef FD_TC_MMA
}
// Arrive on `bar` once every earlier MMA of this thread has completed; with
// two CTAs, on the same barrier of the cluster's CTAs in `mask`.
template <int CTAS>
FD_DEV void tc_commit(uint64_t* bar, uint16_t mask = 0) {
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     fd_stream::smem_addr(bar))
                 : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            fd_stream::smem_addr(bar)),
        "h"(mask)
        : "memory");
}

// 16 consecutive accumulator columns of this warp's 32 lanes (tcgen05.ld
// reads lanes 32 * (warp % 4) + lane), arrived on return: the wait is in the
// same statement, so that no use of the values can be moved before it.
FD_DEV void tc_load16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
// One lane of a converged warp, chosen by elect.sync.  TMA and tcgen05
// instructions take warp-uniform operands; issued under `if (lane == 0)`
// instead, a step of four MMAs and its commit measured about 700 cycles whatever
// the tile, under elect.sync as little as its MMAs take (4096 x 14336 x 4096 in
// 16 bits: 340 -> 312 us, 1 x 28672 x 4096: 59 -> 49 us).
FD_DEV bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
FD_DEV int warp_index() { return __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0); }

// Bring a tile into L2 only.  L2 is where all SMs' accesses meet, so this may run
// before the kernel that writes the tile has finished.
FD_DEV void tma_prefetch_2d(const CUtensorMap* map, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}

FD_DEV void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
FD_DEV int dtype_size(int dtype) { return dtype == FD_F32 ? 4 : 2; }

FD_DEV void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
FD_DEV void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
FD_DEV float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Wait (bounded) for the phase of `bar` with this parity.  Every role calls
// grid_dep_wait before its first such wait, so the bound covers this kernel's own
// work alone, however long the kernels ahead take.  It is looked at every 256
// tries.  Acquiring at CTA scope is enough where the other CTA of
// a pair signals, too: what these barriers pass on is shared-memory tiles
// written by TMA and accumulators in tensor memory, never plain stores.
constexpr int64_t kWaitClocks = 4000000000ll;  // 2 s at the highest clock
FD_DEV bool wait_more(uint32_t addr, uint32_t parity) {
  const int64_t t0 = clock64();
  do {
    for (int i = 0; i < 256; ++i)
      if (fd_stream::mbar_try(addr, parity)) return true;
  } while (clock64() - t0 < kWaitClocks);
  return false;
}
FD_DEV bool wait_phase(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = fd_stream::smem_addr(bar);
  return fd_stream::mbar_try(addr, parity) || wait_more(addr, parity);
}

// The ring stage of a role's next step, and how often the ring has come round:
// counted up, since dividing the step number takes longer than a step.
struct RingPos {
  int stage;
  uint32_t phase;
  FD_DEV void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

FD_DEV bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort);

// Wait for the step at `p`, and look at the ring's later stages with the other
// lanes: how many steps in a row (at most `most`) have arrived, 0 once any role
// has given up.  One look costs about 150 ns, as much as issuing a step's MMAs.
// The lane that issues the MMAs has itself looked at one stage only: __syncwarp
// passes the other lanes' acquires on to it, which the vote alone does not.
FD_DEV int wait_steps(uint64_t* bars, RingPos p, int stages, int most, volatile int* abort) {
  const int lane = threadIdx.x & 31;
  most = min(most, stages);
  int s = p.stage + lane;
  uint32_t phase = p.phase;
  if (s >= stages) {
    s -= stages;
    phase ^= 1;
  }
  const uint32_t addr = fd_stream::smem_addr(bars + (lane < most ? s : p.stage));
  if (lane >= most) phase = p.phase;
  uint32_t here = __ballot_sync(0xffffffffu, fd_stream::mbar_try(addr, phase));
  if (!(here & 1)) {
    if (!wait_or_abort(bars + p.stage, p.phase, abort)) return 0;
    here = 1;
  }
  __syncwarp();
  return min(here == 0xffffffffu ? 32 : __ffs(~here) - 1, most);
}

// A warp's wait: false, for all of its lanes, once any role of this CTA has given up.
FD_DEV bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const uint32_t addr = fd_stream::smem_addr(bar);
  bool done = fd_stream::mbar_try(addr, parity);
  if (!done && !*abort) done = wait_more(addr, parity);
  if (__all_sync(0xffffffffu, done)) return true;
  *abort = 1;
  if ((threadIdx.x & 31) == 0) atomicOr(&g_product_status, kStatusWait);
  return false;
}

template <int N>
FD_DEV void activate_all(float* v, int act) {
  switch (act) {
#define FD_ACT_CASE(a)                                  \
  case a:                                               \
    _Pragma("unroll") for (int j = 0; j < N; ++j) v[j] = activate(v[j], a); \
    break;
    FD_ACT_CASE(FD_ACT_RELU)
    FD_ACT_CASE(FD_ACT_SILU)
    FD_ACT_CASE(FD_ACT_GELU)
    FD_ACT_CASE(FD_ACT_GELU_TANH)
#undef FD_ACT_CASE
    default: break;
  }
}

constexpr int kMaxSplit = 8;  // CTAs, or pairs, that share a tile's K steps

// Four consecutive columns of y from their sums.
template <typename T, bool FP8>
FD_DEV void finish4(const Epilogue& e, bool vec, int64_t m, int64_t n, const float* sum) {
  if (!vec || n + 4 > e.n) {
    for (int j = 0; j < 4 && n + j < e.n; ++j) finish<T, FP8>(e, m, n + j, sum[j]);
    return;
  }
  float v[4];
  const float xs = FP8 ? e.xs[m] : 1.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = FP8 ? sum[j] * xs * e.ws[n + j] : sum[j];
    if (e.bias) v[j] += load_as_f32(e.bias, e.bias_dtype, (n + j) * e.sbias);
  }
  activate_all<4>(v, e.act);
  if (e.ra) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const T*>(e.ra) + m * e.srm + n);
    const float2 lo = unpack2<T>(w.x), hi = unpack2<T>(w.y);
    v[0] += lo.x; v[1] += lo.y; v[2] += hi.x; v[3] += hi.y;
  }
  *reinterpret_cast<uint2*>(static_cast<T*>(e.y) + m * e.sym + n) =
      make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

// The partial tiles of a cluster's `parts` sharers, `rows` floats to a column
// at `part` in each: sharer `rank` takes the columns rank, rank + parts, ... below
// `live`, sums them in sharer order and finishes them, `threads` threads at
// work.  Sharer p is the cluster's CTA p * step + side.  Rows past the last row
// of w are not read: every remote load then feeds a store to y, so none is still
// under way when this CTA tells its peers that they may exit.
template <typename T, bool FP8>
FD_DEV void join_parts(const Epilogue& e, bool vec, const float* part, int rows, int live, int rank, int parts, int step,
                       int side, int64_t m0, int64_t n0, int tid, int threads) {
  const int quads = rows / 4, mine = live > rank ? (live - rank - 1) / parts + 1 : 0;
  for (int i = tid; i < mine * quads; i += threads) {
    const int c = rank + i / quads * parts, r = i % quads * 4;
    if (n0 + r >= e.n) continue;
    float4 from[kMaxSplit];  // all on their way before the first is added
#pragma unroll
    for (int p = 0; p < kMaxSplit; ++p)
      from[p] = p < parts ? ld_cluster_f4(fd_stream::cluster_map(part + c * rows + r, p * step + side))
                          : make_float4(0.f, 0.f, 0.f, 0.f);
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < kMaxSplit; ++p) {
      v[0] += from[p].x; v[1] += from[p].y; v[2] += from[p].z; v[3] += from[p].w;
    }
    finish4<T, FP8>(e, vec, m0 + c, n0 + r, v);
  }
}

// N columns of a tile straight from tensor memory, `live` of them in use, one
// row n of w to a thread: consecutive lanes write consecutive elements of y,
// whatever its layout.  xs: the scales of the N rows of x.  The columns' offsets
// from the first are 32-bit (N is 16, and the host keeps row strides of y and
// row_add below 2^27 elements).
template <typename T, bool FP8, int N>
FD_DEV void emit_columns(const Epilogue& e, float* v, int64_t m, int live, int64_t n, const float* xs, float ws,
                         float bias) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = FP8 ? fmaf(v[j] * xs[j], ws, bias) : v[j] + bias;
  activate_all<N>(v, e.act);
  const uint32_t sym = static_cast<uint32_t>(e.sym), srm = static_cast<uint32_t>(e.srm);
  T* y = static_cast<T*>(e.y) + m * e.sym + n * e.syn;
  if (live >= N && (!e.ra || e.ra_dtype == dtype_of<T>())) {
    if (e.ra) {  // all on their way before the first is added
      const T* ra = static_cast<const T*>(e.ra) + m * e.srm + n * e.srn;
      T r[N];
#pragma unroll
      for (int j = 0; j < N; ++j) r[j] = ra[j * srm];
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += to_f32(r[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) y[j * sym] = from_f32<T>(v[j]);
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < live) {
      if (e.ra) v[j] += load_as_f32(e.ra, e.ra_dtype, (m + j) * e.srm + n * e.srn);
      y[j * sym] = from_f32<T>(v[j]);
    }
}

// ============================================================== few rows
// Products bound by the weight's bytes.  The weight's rows are cut into tiles
// of R rows (any multiple of 8 up to 256) so that the tiles, or the tiles times
// the CTAs that share the K steps of each, number the SMs: every SM streams
// the same share of the weight.  A tile's rows are the MMA's rows (one or two
// blocks of 128; rows beyond R are whatever shared memory holds, and nothing
// reads their sums), up to 80 rows of x its columns.  Each CTA streams its part
// through a TMA ring (one warp for w, one for x, one issuing MMAs).  Where a
// thread-block cluster shares a tile's K steps, the partial tiles meet through
// distributed shared memory and every CTA sums some columns of all partials in
// rank order: the same bits every time, and no workspace that two streams or
// graphs could share.  Otherwise a CTA goes over several tiles where there are
// more than SMs, the epilogue of one under the stream of the next.
constexpr int kBlockRows = 128;  // rows of one MMA
constexpr int kSplitThreads = 256;

struct SplitArgs {
  Epilogue e;
  int64_t tiles;
  int32_t rows;    // R
  int32_t blocks;  // MMA row blocks per tile
  int32_t cols;    // rows of x, rounded up to 16 (MMA columns)
  int32_t steps;   // K steps of a tile, 128 bytes each
  int32_t stages;
  int32_t split;   // CTAs per tile
  int32_t accs;    // accumulators (2: the epilogue overlaps the next tile)
  int32_t box_elems;
  uint32_t desc;
  uint32_t tmem_cols;
  int32_t ahead;   // steps of w brought into L2 before the kernel before this one has finished
  int32_t vec;     // y and row_add take 4 columns at a time
};

template <typename T, bool FP8>
__global__ void __launch_bounds__(kSplitThreads, 1)
    product_split_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                         const __grid_constant__ SplitArgs a) {
  using namespace fd_stream;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kMaxRing], empty[kMaxRing], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = a.split > 1 ? cluster_ctarank() : 0;
  const int64_t first = blockIdx.x / a.split, stride = gridDim.x / a.split;
  const int s0 = static_cast<int>(static_cast<int64_t>(rank) * a.steps / a.split);
  const int count = static_cast<int>(static_cast<int64_t>(rank + 1) * a.steps / a.split) - s0;
  const uint32_t wbytes = a.rows * kBoxBytes, xbytes = a.cols * kBoxBytes, stage_bytes = wbytes + xbytes;
  const uint32_t acc_cols = a.blocks * a.cols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    abort = 0;
    bar_init_fence();
  }
  if (warp == 3) tmem_alloc<1>(&tmem_slot, a.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp <= 1) {
    const CUtensorMap* map = warp == 0 ? &wmap : &xmap;
    const uint32_t bytes = warp == 0 ? wbytes : xbytes;
    const uint64_t policy = evict_first_policy();
    if (elect_one()) prefetch_map(map);
    grid_dep_wait();
    RingPos p{0, 0};
    int64_t i = 0;
    bool ok = true;
    for (int64_t t = first; t < a.tiles && ok; t += stride) {
      const int32_t row = warp == 0 ? static_cast<int32_t>(t * a.rows) : 0;
      for (int k = 0; k < count; ++k, ++i, p.next(a.stages)) {
        if (i >= a.stages && !wait_or_abort(&empty[p.stage], p.phase ^ 1, &abort)) {
          ok = false;
          break;
        }
        uint8_t* dst = ring + p.stage * stage_bytes + (warp == 0 ? 0 : wbytes);
        if (elect_one()) {
          mbar_expect_tx(&full[p.stage], bytes);
          if (warp == 0) tma_load_2d(dst, map, (s0 + k) * a.box_elems, row, &full[p.stage], policy);
          else tma_load_2d_plain(dst, map, (s0 + k) * a.box_elems, row, &full[p.stage]);
        }
        __syncwarp();
      }
    }
    // every copy of this CTA has landed and been read before it may exit
    bool read = true;
    for (int64_t j = i > a.stages ? i - a.stages : 0; j < i; ++j) {
      read = read && wait_phase(&empty[j % a.stages], (j / a.stages) & 1);
      if (!read) wait_phase(&full[j % a.stages], (j / a.stages) & 1);
    }
    __syncwarp();
  } else if (warp == 2) {
    const uint64_t ring_desc = tile_desc(smem_addr(ring));  // addresses in 16-byte units: below 2^14
    // No operand arrives before the kernels ahead have finished: only from there
    // on does a wait's bound say anything.
    grid_dep_wait();
    RingPos p{0, 0};
    bool ok = true;
    int it = 0;
    for (int64_t t = first; t < a.tiles && ok; t += stride, ++it) {
      const int b = a.accs == 2 ? it & 1 : 0, turn = a.accs == 2 ? it >> 1 : it;
      if (!wait_or_abort(&acc_empty[b], (turn & 1) ^ 1, &abort)) break;
      tc_fence_after();
      const uint32_t d = tmem + b * acc_cols;
      for (int k = 0; k < count;) {
        const int here = wait_steps(full, p, a.stages, count - k, &abort);
        if (here == 0) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int j = 0; j < here; ++j, ++k, p.next(a.stages)) {
          const uint64_t w = ring_desc + p.stage * (stage_bytes / 16), x = w + wbytes / 16;
          if (elect_one()) {
            for (int r = 0; r < a.blocks; ++r)
#pragma unroll
              for (int kk = 0; kk < kBoxBytes; kk += kSliceBytes)
                tc_mma<FP8, 1>(d + r * a.cols, w + (r * kBlockRows * kBoxBytes + kk) / 16, x + kk / 16, a.desc,
                               k + kk > 0);
            tc_commit<1>(&empty[p.stage]);
            if (k + 1 == count) tc_commit<1>(&acc_full[b]);
          }
          __syncwarp();
        }
      }
    }
  } else if (warp == 3) {
    for (int i = 0; i < min(count, a.ahead); ++i)
      if (elect_one()) tma_prefetch_2d(&wmap, (s0 + i) * a.box_elems, static_cast<int32_t>(first * a.rows));
    __syncwarp();
  }
  grid_dep_wait();
  const int live = static_cast<int>(a.e.m);  // columns in use
  if (warp >= 4) {  // the first tile's part of the epilogue's operands into L2, under its MMAs
    const int et = threadIdx.x - 128;
    const int64_t n0 = first * a.rows;
    const int rows = static_cast<int>(min(static_cast<int64_t>(a.rows), a.e.n - n0));
    for (int r = et; r < rows; r += 128) {
      if (FP8) prefetch_l2(a.e.ws + n0 + r);
      if (a.e.bias) prefetch_l2(static_cast<const char*>(a.e.bias) + (n0 + r) * a.e.sbias * dtype_size(a.e.bias_dtype));
    }
    if (et < live) {
      if (FP8) prefetch_l2(a.e.xs + et);
      if (a.e.ra && a.e.srn == 1 && et % a.split == static_cast<int>(rank)) {
        const int es = dtype_size(a.e.ra_dtype);
        const char* p = static_cast<const char*>(a.e.ra) + (et * a.e.srm + n0) * es;
        for (int o = 0; o < rows * es; o += 128) prefetch_l2(p + o);
      }
    }
    __syncwarp();
  }
  if (a.split == 1) {
    // straight from tensor memory: a thread per row of the tile
    if (warp >= 4) {
      bool ok = true;
      int it = 0;
      for (int64_t t = first; t < a.tiles; t += stride, ++it) {
        const int b = a.accs == 2 ? it & 1 : 0, turn = a.accs == 2 ? it >> 1 : it;
        float ws2[2] = {1.f, 1.f}, bias2[2] = {0.f, 0.f};  // of this thread's row in either block
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          const int r = blk * kBlockRows + (warp - 4) * 32 + lane;
          const int64_t n = t * a.rows + r;
          if (r >= a.rows || n >= a.e.n) continue;
          if (FP8) ws2[blk] = a.e.ws[n];
          if (a.e.bias) bias2[blk] = load_as_f32(a.e.bias, a.e.bias_dtype, n * a.e.sbias);
        }
        ok = ok && wait_or_abort(&acc_full[b], turn & 1, &abort);
        if (!ok) break;
        tc_fence_after();
        for (int blk = 0; blk < a.blocks; ++blk) {
          const int r = blk * kBlockRows + (warp - 4) * 32 + lane;
          const int64_t n = t * a.rows + r;
          const bool row_ok = r < a.rows && n < a.e.n;
          const float ws = blk ? ws2[1] : ws2[0], bias = blk ? bias2[1] : bias2[0];
          const uint32_t acc = tmem + (static_cast<uint32_t>((warp - 4) * 32) << 16) + b * acc_cols + blk * a.cols;
          for (int c = 0; c < live; c += 16) {
            float v[16], xs[16];
            __syncwarp();
            tc_load16(acc + c, reinterpret_cast<uint32_t*>(v));
            if (!row_ok) continue;
            if (FP8) {
#pragma unroll
              for (int j = 0; j < 16; ++j) xs[j] = c + j < live ? a.e.xs[c + j] : 0.f;
            }
            emit_columns<T, FP8, 16>(a.e, v, c, live - c, n, xs, ws, bias);
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[b]);
      }
    }
  } else {
    // partial tiles in the ring's memory, a column of R floats after another
    float* part = reinterpret_cast<float*>(ring);
    const bool ok = wait_or_abort(&acc_full[0], 0, &abort);
    tc_fence_after();
    if (warp >= 4 && ok) {
      for (int blk = 0; blk < a.blocks; ++blk) {
        const int r = blk * kBlockRows + (warp - 4) * 32 + lane;
        const uint32_t acc = tmem + (static_cast<uint32_t>((warp - 4) * 32) << 16) + blk * a.cols;
        for (int c = 0; c < live; c += 16) {
          uint32_t v[16];
          __syncwarp();
          tc_load16(acc + c, v);
          if (r < a.rows) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (c + j < live) part[(c + j) * a.rows + r] = __uint_as_float(v[j]);
          }
        }
        __syncwarp();
      }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    join_parts<T, FP8>(a.e, a.vec, part, a.rows, live, rank, a.split, 1, 0, 0, first * a.rows, threadIdx.x,
                       kSplitThreads);
    __syncwarp();
    // The other CTAs may still be reading this one's partial.  Relaxed, here and
    // in the pair kernel: nothing is passed on, every value read from a peer is in
    // a store to y that comes before the arrival, and a release would wait for
    // those stores.
    cluster_arrive_relaxed();
    cluster_wait();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_free<1>(tmem, a.tmem_cols);
  }
}

// ============================================================== many rows
// Pairs of CTAs (cta_group::2) on tiles of 256 rows of w by up to 256 rows of x
// (any multiple of 32, so that a ragged batch fills its tiles): each CTA holds
// 128 rows of the w tile and half of the x tile, so a pair reads every operand
// byte from shared memory half as often as two single CTAs would.  Persistent:
// a pair walks over its tiles with two accumulators in tensor memory, the
// epilogue of one tile under the MMAs of the next.  Rows of w are the MMA's rows
// because the accumulator then has consecutive elements of a row of y in
// consecutive lanes: one path of coalesced stores for any layout of y.
// An SM takes in about 115 GB/s from L2 whatever it multiplies; where there are
// fewer tiles than pairs, the pairs of a cluster share the K steps of one tile,
// and each sums its part of the columns over all partials, in rank order,
// through distributed shared memory.
constexpr int kPairRows = 256;
constexpr int kPairCols = 256;     // at most
constexpr int kEpilogueWarps = 8;  // a multiple of 4: warp w reads the tensor memory lanes of w % 4
constexpr int kPairThreads = 128 + 32 * kEpilogueWarps;  // TMA, MMA, tensor memory, one idle warp
// Accumulator columns an epilogue warp handles at once: with 32 the code of a
// chunk is as long again and 8192 x 4096 x 512 takes 34 us, with 16 it takes 30.
constexpr int kChunk = 16;

struct PairArgs {
  Epilogue e;
  int32_t steps;  // 128-byte boxes along K
  int32_t cols;   // rows of x per tile
  int32_t stages;
  int32_t split;  // pairs that share a tile
  int32_t box_elems;
  uint32_t desc;
  int64_t mt, nt;  // tiles along m (x) and n (w)
  int32_t group;   // m tiles walked together
  int32_t vec;     // y and row_add take 4 columns at a time
};

// Tile t of the walk: `group` m tiles side by side for every n tile, so that
// the pairs at work share both operands' tiles in L2.
FD_DEV void pair_tile(const PairArgs& a, int64_t t, int64_t* mi, int64_t* ni) {
  const uint32_t per = static_cast<uint32_t>(a.group) * static_cast<uint32_t>(a.nt), tile = static_cast<uint32_t>(t);
  const uint32_t g = tile / per, in = tile - g * per;
  const uint32_t rows = min(static_cast<uint32_t>(a.group), static_cast<uint32_t>(a.mt) - g * a.group);
  const uint32_t n = in / rows;
  *mi = g * a.group + (in - n * rows);
  *ni = n;
}

FD_DEV void tma_load_pair(void* dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(fd_stream::smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Relaxed: the accumulator's columns are in registers by then, and a release
// would wait for the warp's stores to y (about 2 us a tile).
FD_DEV void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <typename T, bool FP8>
__global__ void __launch_bounds__(kPairThreads, 1)
    product_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                        const __grid_constant__ PairArgs a) {
  using namespace fd_stream;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kMaxRing], empty[kMaxRing], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort;
  __shared__ __align__(16) float s_xs[2][kPairCols];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  const int warp = warp_index(), lane = threadIdx.x & 31;
  // a cluster's CTAs: pairs of neighbours, the first of a pair issues its MMAs
  const uint32_t crank = cluster_ctarank(), side = crank & 1, pair = crank >> 1;
  const uint16_t both = static_cast<uint16_t>(3u << (pair * 2));
  const int half_cols = a.cols / 2;
  const uint32_t wbytes = 128 * kBoxBytes, xbytes = half_cols * kBoxBytes, stage_bytes = wbytes + xbytes;
  const int64_t tiles = a.mt * a.nt, stride = gridDim.x / (2 * a.split), first = blockIdx.x / (2 * a.split);
  const int s0 = static_cast<int>(static_cast<int64_t>(pair) * a.steps / a.split);
  const int count = static_cast<int>(static_cast<int64_t>(pair + 1) * a.steps / a.split) - s0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kEpilogueWarps);  // of both CTAs
    }
    abort = 0;
    bar_init_fence();
  }
  if (warp == 2) tmem_alloc<2>(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_arrive_relaxed();  // the cluster's barriers exist (bar_init_fence) before any is signalled
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  grid_dep_wait();

  if (warp == 0) {
    if (elect_one()) {
      prefetch_map(&wmap);
      prefetch_map(&xmap);
    }
    const uint32_t bars = cluster_map(full, crank - side);
    RingPos p{0, 0};
    int64_t i = 0;
    bool ok = true;
    for (int64_t t = first; t < tiles && ok; t += stride) {
      int64_t mi, ni;
      pair_tile(a, t, &mi, &ni);
      const int32_t wr = static_cast<int32_t>(ni * kPairRows + side * 128);
      const int32_t xr = static_cast<int32_t>(mi * a.cols + side * half_cols);
      for (int k = 0; k < count; ++k, ++i, p.next(a.stages)) {
        if (i >= a.stages && !wait_or_abort(&empty[p.stage], p.phase ^ 1, &abort)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t bar = bars + p.stage * 8;
          // the first CTA's barrier counts the bytes of both
          if (side == 0) mbar_expect_tx(&full[p.stage], 2 * stage_bytes);
          uint8_t* dst = ring + p.stage * stage_bytes;
          tma_load_pair(dst, &wmap, (s0 + k) * a.box_elems, wr, bar);
          tma_load_pair(dst + wbytes, &xmap, (s0 + k) * a.box_elems, xr, bar);
        }
        __syncwarp();
      }
    }
    // every stage has landed and been read, and its barrier signalled, before the pair may exit
    bool read = true;
    for (int64_t j = i > a.stages ? i - a.stages : 0; j < i; ++j) {
      read = read && wait_phase(&empty[j % a.stages], (j / a.stages) & 1);
      if (!read && side == 0) wait_phase(&full[j % a.stages], (j / a.stages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (side == 0) {
      const uint64_t ring_desc = tile_desc(smem_addr(ring));
      RingPos p{0, 0};
      int it = 0;
      bool ok = true;
      for (int64_t t = first; t < tiles && ok; t += stride, ++it) {
        const int b = it & 1;
        if (!wait_or_abort(&acc_empty[b], ((it >> 1) & 1) ^ 1, &abort)) break;
        tc_fence_after();
        const uint32_t d = tmem + b * kPairCols;
        for (int k = 0; k < count;) {
          const int here = wait_steps(full, p, a.stages, count - k, &abort);
          if (here == 0) {
            ok = false;
            break;
          }
          tc_fence_after();
          for (int j = 0; j < here; ++j, ++k, p.next(a.stages)) {
            const uint64_t w = ring_desc + p.stage * (stage_bytes / 16), x = w + wbytes / 16;
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < kBoxBytes; kk += kSliceBytes)
                tc_mma<FP8, 2>(d, w + kk / 16, x + kk / 16, a.desc, k + kk > 0);
              tc_commit<2>(&empty[p.stage], both);
              if (k + 1 == count) tc_commit<2>(&acc_full[b], both);
            }
            __syncwarp();
          }
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int q = warp & 3, turn = (warp - 4) >> 2, et = threadIdx.x - 128;
    // a tile's place, this thread's scales (of row n of w, and of the tile's row
    // et of x) and bias: loaded a tile ahead
    struct Edge {
      int64_t m0, n;
      int live;
      float ws, bias, xs;
    };
    auto edge_of = [&](int64_t t) {
      Edge g{0, 0, 0, 1.f, 0.f, 0.f};
      if (t >= tiles) return g;
      int64_t mi, ni;
      pair_tile(a, t, &mi, &ni);
      g.m0 = mi * a.cols;
      g.n = ni * kPairRows + side * 128 + q * 32 + lane;
      g.live = static_cast<int>(min(static_cast<int64_t>(a.cols), a.e.m - g.m0));
      if (g.n < a.e.n) {
        if (FP8) g.ws = a.e.ws[g.n];
        if (a.e.bias) g.bias = load_as_f32(a.e.bias, a.e.bias_dtype, g.n * a.e.sbias);
      }
      if (et < g.live) {
        if (FP8) g.xs = a.e.xs[g.m0 + et];
        // row et of the tile's part of row_add into L2: the loads themselves keep
        // too few bytes in flight for HBM's latency
        if (a.e.ra && a.e.srn == 1 && a.e.srm != 0) {
          const int es = dtype_size(a.e.ra_dtype);
          const int64_t n0 = ni * kPairRows + side * 128;
          const char* p = static_cast<const char*>(a.e.ra) + ((g.m0 + et) * a.e.srm + n0) * es;
          const int bytes = static_cast<int>(min(int64_t{128}, a.e.n - n0)) * es;
          for (int o = 0; o < bytes; o += 128) prefetch_l2(p + o);
        }
      }
      return g;
    };
    static_assert(kPairCols <= 32 * kEpilogueWarps, "one row of x to a thread");
    int it = 0;
    bool ok = true;
    Edge next = edge_of(first);
    for (int64_t t = first; t < tiles; t += stride, ++it) {
      const int b = it & 1;
      const Edge g = next;
      const int64_t m0 = g.m0, n = g.n;
      const int live = g.live;
      const bool row_ok = n < a.e.n;
      if (FP8) {
        if (et < kPairCols) s_xs[b][et] = g.xs;
        named_sync(1, 32 * kEpilogueWarps);
      }
      next = edge_of(t + stride);
      // after an expired wait the warps still meet at every tile's barrier
      ok = ok && wait_or_abort(&acc_full[b], (it >> 1) & 1, &abort);
      if (!ok) continue;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16) + b * kPairCols;
      // the partial tile of a shared one: a column of 128 rows after another, in the ring's memory
      float* part = reinterpret_cast<float*>(ring) + q * 32 + lane;
      auto freed = [&]() {  // this warp has read its part: once from all, the accumulator takes the tile after next
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(cluster_map(&acc_empty[b], crank - side));
      };
      constexpr int kRound = kEpilogueWarps / 4 * kChunk;
      for (int c = turn * kChunk; c < live; c += kRound) {
        float v[kChunk];
        tc_load16(acc + c, reinterpret_cast<uint32_t*>(v));
        if (c + kRound >= live) freed();
        if (a.split > 1) {
#pragma unroll
          for (int j = 0; j < kChunk; ++j)
            if (c + j < live) part[(c + j) * 128] = v[j];
        } else if (row_ok) {
          emit_columns<T, FP8, kChunk>(a.e, v, m0 + c, live - c, n, s_xs[b] + c, g.ws, g.bias);
        }
        __syncwarp();
      }
      if (turn * kChunk >= live) freed();
    }
    __syncwarp();
  }
  if (a.split > 1) {
    cluster_arrive();  // every partial is written
    cluster_wait();
    int64_t mi, ni;
    pair_tile(a, first, &mi, &ni);
    const int64_t m0 = mi * a.cols;
    const int live = static_cast<int>(min(static_cast<int64_t>(a.cols), a.e.m - m0));
    join_parts<T, FP8>(a.e, a.vec, reinterpret_cast<float*>(ring), 128, live, pair, a.split, 2, side, m0,
                       ni * kPairRows + side * 128, threadIdx.x, kPairThreads);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive_relaxed();  // the cluster's last signals, MMAs and reads of partials are over on all sides
  cluster_wait();
  if (warp == 2) {
    tc_fence_after();
    tmem_free<2>(tmem, 512);
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

// ---- the tensor-core kernels
// A [rows, k] operand as a tensor map of 128-byte boxes: elements outside read
// as zero.  Needs unit stride along K, and 16-byte aligned rows.
bool operand_map(CUtensorMap* map, const void* p, int64_t rows, int64_t k, int64_t stride, int64_t k_stride, int es,
                 int box_rows) {
  if (rows == 1) stride = (k * es + 15) / 16 * 16 / es;  // never followed
  if ((k_stride != 1 && k != 1) || !fd_host::aligned16(p) || stride * es % 16 != 0 || stride < k) return false;
  if (rows > 0x7fffffffLL || k > 0x7fffffffLL || stride * es >= (int64_t{1} << 40)) return false;
  auto fn = fd_stream::encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * es};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(kBoxBytes / es), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t unit[2] = {1, 1};
  return fn(map, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(p),
            dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr size_t kSplitSmemMax = 226 * 1024;
constexpr size_t kPairSmem = 217 * 1024;  // all of an SM's, as it takes all of its tensor memory
// Tensor memory has 512 columns an SM and an allocation waits for them.  A CTA
// takes at least this much shared memory for each column, its share of the
// SM's 228 KB: no SM ever holds CTAs that want more columns than there are, so
// no allocation waits for a CTA that is itself waiting for a peer.
constexpr size_t kSmemPerTmemCol = 228 * 1024 / 512;

constexpr int kMaxDevices = 64;

// Let a kernel have up to `bytes` of dynamic shared memory: once per device.
template <auto kKernel>
cudaError_t allow_smem(size_t bytes) {
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kMaxDevices && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && dev < kMaxDevices) done[dev].store(true, std::memory_order_release);
  return e;
}

void set_cluster(cudaLaunchAttribute* attr, int size) {
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = static_cast<unsigned>(size);
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
}

// Clusters of `size` CTAs (2 to 8) that fit on the device at once, one CTA per
// SM: asked once per device.
template <auto kKernel>
int64_t cluster_slots(int threads, size_t smem, int size) {
  static std::atomic<int> known[kMaxDevices][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return 1;
  int n = known[dev][size].load(std::memory_order_relaxed);
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(size));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  set_cluster(&attr[0], size);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (allow_smem<kKernel>(smem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess ||
      n < 1) {
    (void)cudaGetLastError();
    n = 1;
  }
  known[dev][size].store(n, std::memory_order_relaxed);
  return n;
}

template <auto kKernel, typename Args>
cudaError_t launch_cluster(dim3 grid, int threads, int cluster, size_t smem, size_t smem_max, cudaStream_t st,
                           const CUtensorMap& m0, const CUtensorMap& m1, const Args& a) {
  const cudaError_t e = allow_smem<kKernel>(smem_max);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  set_cluster(&attr[1], cluster);
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kKernel, m0, m1, a);
}

int mma_format(int in_dtype) { return in_dtype == FD_BF16 ? 1 : 0; }

// Rows of y (and of row_add, where there is one) as vectors of `width` elements of the output's type.
bool epilogue_vec(const Epilogue& e, int out_dtype, int width) {
  auto rows = [&](const void* p, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % (2 * width) == 0 && (e.m == 1 || stride % width == 0);
  };
  if (e.syn != 1 || !rows(e.y, e.sym)) return false;
  return !e.ra || (e.ra_dtype == out_dtype && e.srn == 1 && rows(e.ra, e.srm));
}

// Rows of x up to which the split kernel serves a product.  Each of its CTAs
// takes in (R + rows of x) * 128 bytes a step, so the pair kernel, which shares
// the x tile between two CTAs, wins once x is no longer small beside R.  Split
// against pair at 64, 80, 96 and 128 rows: 4096 x 4096 in 16 bits 11.8 / 12.8,
// 12.6 / 13.5, 14.0 / 13.7, 15.1 / 13.8 us; 28672 x 4096 in 8 bits 24.1 / 24.5,
// 25.4 / 26.0, 26.6 / 25.1, 29.1 / 26.1 us.  One number for every N and type: both
// widths change over between 80 and 96 rows, and others were not measured.
constexpr int64_t kSplitMaxM = 80;

// Few rows.  FD_ERR_UNSUPPORTED: a layout TMA cannot address.
template <typename T, bool FP8>
int launch_split(const GenericArgs& g, int in_dtype, int out_dtype, cudaStream_t st) {
  constexpr int es = FP8 ? 1 : 2;
  constexpr int64_t max_rows = 256;
  const Epilogue& e = g.epi;
  SplitArgs a;
  a.e = e;
  a.cols = static_cast<int32_t>((e.m + 15) / 16 * 16);
  a.box_elems = kBoxBytes / es;
  const int sms = fd_host::sm_count();
  const int64_t steps = (g.k + a.box_elems - 1) / a.box_elems;
  // CTAs per tile: tiles of about 128 rows (an MMA takes as long for fewer)
  // that fill the SMs, 8 steps at least to each CTA
  a.split = 1;
  while (a.split < kMaxSplit && e.n * a.split * 2 <= static_cast<int64_t>(sms) * kBlockRows && steps >= a.split * 8)
    a.split *= 2;
  // R: equal tiles in one wave of CTAs, or in the fewest
  const int64_t slots = a.split > 1 ? cluster_slots<product_split_kernel<T, FP8>>(kSplitThreads, kSplitSmemMax, a.split) : sms;
  const int64_t waves = a.split > 1 ? 1 : (e.n + slots * max_rows - 1) / (slots * max_rows);
  const int64_t rows = std::min<int64_t>(((e.n + slots * waves - 1) / (slots * waves) + 7) / 8 * 8, max_rows);
  a.rows = static_cast<int32_t>(rows);
  a.blocks = a.rows > kBlockRows ? 2 : 1;
  a.tiles = (e.n + rows - 1) / rows;
  if (steps > 0x7fffffffLL || a.tiles > 0x7fffff) return FD_ERR_UNSUPPORTED;
  a.steps = static_cast<int32_t>(steps);
  a.desc = mma_desc(FP8 ? 0 : mma_format(in_dtype), kBlockRows, a.cols);
  const uint32_t acc = a.blocks * a.cols;
  a.accs = a.split == 1 && a.tiles > sms && 2 * acc <= 256 ? 2 : 1;
  a.tmem_cols = 32;
  while (a.tmem_cols < a.accs * acc) a.tmem_cols *= 2;
  a.vec = epilogue_vec(e, out_dtype, 4);
  // A ring of all the shared memory, and the first steps brought into L2 ahead
  // of the wait: four cost nothing where this kernel starts late, eight delay its
  // own copies (4096 x 4096 in 8 bits 7.6 against 8.7 us, without any 7.7; the MLP
  // of one row, behind its row kernels, 39.0 against 39.5 and 41.4).
  a.ahead = 4;
  const size_t stage = static_cast<size_t>(kBoxBytes) * (a.rows + a.cols);
  a.stages = static_cast<int32_t>(std::min<size_t>(kMaxRing, 216 * 1024 / stage));
  const size_t part = a.split > 1 ? static_cast<size_t>(e.m) * a.rows * 4 : 0;
  // an MMA reads whole blocks of 128 rows, past the last stage's R
  const size_t reads = (a.stages - 1) * stage + static_cast<size_t>(kBoxBytes) * a.blocks * kBlockRows;
  const size_t smem = std::max(a.tmem_cols * kSmemPerTmemCol, std::max(std::max(a.stages * stage, reads), part) + 1024);
  if (smem > kSplitSmemMax) return FD_ERR_UNSUPPORTED;
  CUtensorMap wm, xm;
  if (!operand_map(&wm, g.w, e.n, g.k, g.swn, g.swk, es, a.rows) ||
      !operand_map(&xm, g.x, e.m, g.k, g.sxm, g.sxk, es, a.cols))
    return FD_ERR_UNSUPPORTED;
  const int64_t grid = a.split > 1 ? a.tiles * a.split : std::min<int64_t>(a.tiles, sms);
  return from_cuda(launch_cluster<product_split_kernel<T, FP8>>(dim3(static_cast<unsigned>(grid)), kSplitThreads,
                                                                a.split, smem, kSplitSmemMax, st, wm, xm, a));
}

template <typename T, bool FP8>
int launch_pair(const GenericArgs& g, int in_dtype, int out_dtype, cudaStream_t st) {
  constexpr int es = FP8 ? 1 : 2;
  const Epilogue& e = g.epi;
  PairArgs a;
  a.e = e;
  a.box_elems = kBoxBytes / es;
  const int64_t steps = (g.k + a.box_elems - 1) / a.box_elems;
  const int pairs = fd_host::sm_count() / 2;
  a.nt = (e.n + kPairRows - 1) / kPairRows;
  // Rows of x per tile and pairs per tile, by the time they should take: a step
  // measured 0.12 us + 0.98 ns per column (0.245 at 128 columns, 0.37 at 256,
  // MMAs, L2 and the power limit together, so for a GPU under steady load; 8 and
  // 16 bits alike, since a step is 128 bytes of K in either), a tile's start and
  // end 0.5 us, the exchange of partials 0.5 us + 6 ns per column.
  double best = 0;
  a.cols = 0;
  a.split = 1;
  for (int split = 1; split <= 4 && (split == 1 || steps >= 4 * split); split *= 2) {
    const int64_t slots = split > 1 ? cluster_slots<product_pair_kernel<T, FP8>>(kPairThreads, kPairSmem, 2 * split) : pairs;
    for (int64_t most = kPairCols; most >= 32; most -= 32) {
      const int64_t mt = (e.m + most - 1) / most;
      const int64_t c = ((e.m + mt - 1) / mt + 31) / 32 * 32;  // as many tiles, evenly filled
      const int64_t tiles = (e.m + c - 1) / c * a.nt;
      const int64_t waves = (tiles + slots - 1) / slots;
      if (split > 1 && waves > 1) continue;
      const double cost = waves * ((steps + split - 1) / split * (0.12 + 0.00098 * c) + 0.5) +
                          (split > 1 ? 0.5 + 0.006 * c : 0.0);
      if (a.cols == 0 || cost < best) {
        best = cost;
        a.cols = static_cast<int32_t>(c);
        a.split = split;
      }
    }
  }
  a.mt = (e.m + a.cols - 1) / a.cols;
  a.group = 16;
  if (steps > 0x7fffffffLL || e.m > 0x7fffff00LL || e.n > 0x7fffff00LL || (a.mt + 16) * a.nt > 0x7fffffffLL)
    return FD_ERR_UNSUPPORTED;
  a.steps = static_cast<int32_t>(steps);
  a.desc = mma_desc(FP8 ? 0 : mma_format(in_dtype), kPairRows, a.cols);
  a.vec = epilogue_vec(e, out_dtype, 4);
  const size_t stage = static_cast<size_t>(kBoxBytes) * (128 + a.cols / 2);
  a.stages = static_cast<int32_t>(std::min<size_t>(kMaxRing, 216 * 1024 / stage));
  CUtensorMap wm, xm;
  if (!operand_map(&wm, g.w, e.n, g.k, g.swn, g.swk, es, 128) ||
      !operand_map(&xm, g.x, e.m, g.k, g.sxm, g.sxk, es, a.cols / 2))
    return FD_ERR_UNSUPPORTED;
  const int64_t grid = 2 * a.split * (a.split > 1 ? a.mt * a.nt : std::min<int64_t>(pairs, a.mt * a.nt));
  return from_cuda(launch_cluster<product_pair_kernel<T, FP8>>(dim3(static_cast<unsigned>(grid)), kPairThreads,
                                                               2 * a.split, kPairSmem, kPairSmem, st, wm, xm, a));
}

template <typename TX, typename T, bool FP8>
int launch_product(const GenericArgs& g, int in_dtype, int out_dtype, cudaStream_t st) {
  int r = FD_ERR_UNSUPPORTED;
  // emit_columns' 32-bit column offsets
  const bool near = g.epi.sym >= 0 && g.epi.srm >= 0 && std::max(g.epi.sym, g.epi.srm) < (int64_t{1} << 27);
  if (g.k > 0 && near) {
    r = g.epi.m <= kSplitMaxM ? launch_split<T, FP8>(g, in_dtype, out_dtype, st)
                              : launch_pair<T, FP8>(g, in_dtype, out_dtype, st);
  }
  return r == FD_ERR_UNSUPPORTED ? launch_generic<TX, T, FP8>(g, st) : r;
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
    return bf ? launch_product<__half, __nv_bfloat16, true>(a, in_dtype, out_dtype, st)
              : launch_product<__half, __half, true>(a, in_dtype, out_dtype, st);
  return bf ? launch_product<__nv_bfloat16, __nv_bfloat16, false>(a, in_dtype, out_dtype, st)
            : launch_product<__half, __half, false>(a, in_dtype, out_dtype, st);
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

int fd_product_status(int32_t* status, void* stream) {
  if (!status) return FD_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int32_t v = 0;
  if (cudaMemcpyFromSymbolAsync(&v, g_product_status, sizeof(v), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return FD_ERR_DEVICE;
  *status = v;
  return FD_OK;
}

int fd_product_reset(void* stream) {
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_product_status) != cudaSuccess) return FD_ERR_DEVICE;
  return from_cuda(cudaMemsetAsync(p, 0, sizeof(int32_t), static_cast<cudaStream_t>(stream)));
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
