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

// ============================================================== tensor cores
// Shared by the two tcgen05 kernels below.  Both operands lie row by row along
// K, in shared-memory tiles of 128-byte rows (64 16-bit or 128 8-bit elements)
// with the 128-byte swizzle TMA writes; one instruction takes 32 bytes of K.
constexpr int kBoxBytes = 128;  // K bytes of a tile row
constexpr int kMaxRing = 10;
constexpr int kSliceBytes = 32;  // K bytes of one tcgen05.mma

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
// two CTAs, on the same barrier of both.
template <int CTAS>
FD_DEV void tc_commit(uint64_t* bar) {
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     fd_stream::smem_addr(bar))
                 : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            fd_stream::smem_addr(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}

// 16 / 32 consecutive accumulator columns of this warp's 32 lanes (tcgen05.ld
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
FD_DEV void tc_load32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}

FD_DEV void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
FD_DEV void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
FD_DEV float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Wait (bounded) for the phase of `bar` with this parity.  The bound is looked
// at every 256 tries.  Acquiring at CTA scope is enough where the other CTA of
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
  int stage = 0;
  uint32_t phase = 0;
  FD_DEV void next(int stages) {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// A wait of one role: false once any role of this CTA has given up.
FD_DEV bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const uint32_t addr = fd_stream::smem_addr(bar);
  if (fd_stream::mbar_try(addr, parity)) return true;
  if (*abort) return false;
  if (wait_more(addr, parity)) return true;
  *abort = 1;
  atomicOr(&g_product_status, kStatusWait);
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

// ============================================================== few rows
// Weight-stationary tiles for products bound by the weight's bytes: 128 rows
// of w are the MMA's rows, up to 256 rows of x (a multiple of 16) its columns,
// and the K steps of a tile are divided among the CTAs of a thread-block
// cluster.  Each CTA streams its part of the tile through a TMA ring (one warp
// for w, one for x, one issuing MMAs), the partial tiles meet through
// distributed shared memory, where every CTA sums some columns of all partials
// in rank order: the same bits every time, and no workspace that two streams
// or graphs could share.
constexpr int kTileRows = 128;
constexpr int kSplitThreads = 256;
constexpr int kMaxSplit = 8;

struct SplitArgs {
  Epilogue e;
  int32_t steps;   // K steps of a tile (boxes * 128 bytes each)
  int32_t cols;    // rows of x per tile (MMA columns)
  int32_t boxes;   // 128-byte boxes per step
  int32_t stages;
  int32_t split;   // CTAs per tile
  int32_t box_elems;
  uint32_t desc;
  uint32_t tmem_cols;
  int32_t w_early;  // the kernel before this one does not write w
};

template <typename T, bool FP8>
__global__ void __launch_bounds__(kSplitThreads, 1)
    product_split_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                         const __grid_constant__ SplitArgs a) {
  using namespace fd_stream;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kMaxRing], empty[kMaxRing], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = a.split > 1 ? cluster_ctarank() : 0;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x / a.split) * kTileRows;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * a.cols;
  const int s0 = static_cast<int>(static_cast<int64_t>(rank) * a.steps / a.split);
  const int count = static_cast<int>(static_cast<int64_t>(rank + 1) * a.steps / a.split) - s0;
  const uint32_t wbytes = a.boxes * kTileRows * kBoxBytes, xbytes = a.boxes * a.cols * kBoxBytes;
  const uint32_t stage_bytes = wbytes + xbytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    abort = 0;
    bar_init_fence();
  }
  if (warp == 3) tmem_alloc<1>(&tmem_slot, a.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp <= 1) {
    if (lane == 0) {
      const CUtensorMap* map = warp == 0 ? &wmap : &xmap;
      prefetch_map(map);
      const uint32_t bytes = warp == 0 ? wbytes : xbytes, box = bytes / a.boxes;
      const int32_t row = static_cast<int32_t>(warp == 0 ? n0 : m0);
      const uint64_t policy = evict_first_policy();
      if (warp == 1 || !a.w_early) grid_dep_wait();
      RingPos p;
      int i = 0;
      for (; i < count; ++i, p.next(a.stages)) {
        const int s = p.stage;
        if (i >= a.stages && !wait_or_abort(&empty[s], p.phase ^ 1, &abort)) break;
        uint8_t* dst = ring + static_cast<size_t>(s) * stage_bytes + (warp == 0 ? 0 : wbytes);
        mbar_expect_tx(&full[s], bytes);
        for (int b = 0; b < a.boxes; ++b) {
          const int32_t col = ((s0 + i) * a.boxes + b) * a.box_elems;
          if (warp == 0) tma_load_2d(dst + b * box, map, col, row, &full[s], policy);
          else tma_load_2d_plain(dst + b * box, map, col, row, &full[s]);
        }
      }
      // every copy of this CTA has landed and been read before it may exit
      bool read = true;
      for (int j = i > a.stages ? i - a.stages : 0; j < i; ++j) {
        read = read && wait_phase(&empty[j % a.stages], (j / a.stages) & 1);
        if (!read) wait_phase(&full[j % a.stages], (j / a.stages) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    if (lane == 0) {
      RingPos p;
      for (int i = 0; i < count; ++i, p.next(a.stages)) {
        const int s = p.stage;
        if (!wait_or_abort(&full[s], p.phase, &abort)) break;
        tc_fence_after();
        const uint32_t w = smem_addr(ring + static_cast<size_t>(s) * stage_bytes), x = w + wbytes;
        for (int b = 0; b < a.boxes; ++b)
#pragma unroll
          for (int k = 0; k < kBoxBytes; k += kSliceBytes)
            tc_mma<FP8, 1>(tmem, tile_desc(w + b * kTileRows * kBoxBytes + k), tile_desc(x + b * a.cols * kBoxBytes + k),
                           a.desc, i + b + k > 0);
        tc_commit<1>(&empty[s]);
      }
      tc_commit<1>(&done);
    }
    __syncwarp();
  }
  grid_dep_wait();
  grid_dep_launch();
  const bool ok = __all_sync(0xffffffffu, wait_or_abort(&done, 0, &abort));
  tc_fence_after();
  const int live = static_cast<int>(min(static_cast<int64_t>(a.cols), a.e.m - m0));  // columns in use
  const int r = threadIdx.x & (kTileRows - 1);
  const int64_t n = n0 + r;
  const bool row_ok = n < a.e.n;
  const float ws = FP8 && row_ok ? a.e.ws[n] : 1.f;
  const float bias = a.e.bias && row_ok ? load_as_f32(a.e.bias, a.e.bias_dtype, n * a.e.sbias) : 0.f;
  auto store = [&](int64_t m, float v) {
    if (FP8) v = v * a.e.xs[m] * ws;
    v = activate(v + bias, a.e.act);
    if (a.e.ra) v += load_as_f32(a.e.ra, a.e.ra_dtype, m * a.e.srm + n * a.e.srn);
    static_cast<T*>(a.e.y)[m * a.e.sym + n * a.e.syn] = from_f32<T>(v);
  };
  if (a.split == 1) {
    if (warp >= 4 && ok) {
      const uint32_t mine = tmem + (static_cast<uint32_t>(r & ~31) << 16);
      for (int c = 0; c < live; c += 16) {
        uint32_t v[16];
        tc_load16(mine + c, v);
        if (row_ok) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < live) store(m0 + c + j, __uint_as_float(v[j]));
        }
      }
    }
  } else {
    // partial tiles in the ring's memory, a column of 128 floats after another
    float* part = reinterpret_cast<float*>(ring);
    if (warp >= 4 && ok) {
      const uint32_t mine = tmem + (static_cast<uint32_t>(r & ~31) << 16);
      for (int c = 0; c < live; c += 16) {
        uint32_t v[16];
        tc_load16(mine + c, v);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c + j < live) part[(c + j) * kTileRows + r] = __uint_as_float(v[j]);
      }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (row_ok) {
      for (int c = static_cast<int>(rank) + a.split * (threadIdx.x / kTileRows); c < live;
           c += a.split * (kSplitThreads / kTileRows)) {
        float v = 0.f;
        for (int p = 0; p < a.split; ++p) v += ld_cluster_f32(cluster_map(part + c * kTileRows + r, p));
        store(m0 + c, v);
      }
    }
    __syncwarp();
    cluster_arrive();  // the other CTAs may still be reading this one's partial
    cluster_wait();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    tc_fence_after();
    tmem_free<1>(tmem, a.tmem_cols);
  }
}

// ============================================================== many rows
// Pairs of CTAs (cta_group::2) on tiles of 256 rows of x by up to 256 rows of
// w: each CTA holds 128 rows of the x tile and half of the w tile, so a pair
// reads every operand byte from shared memory half as often as two single
// CTAs would.  Persistent: a pair walks over its tiles with two accumulators
// in tensor memory, the epilogue of one tile under the MMAs of the next.
constexpr int kPairRows = 256;
constexpr int kPairCols = 256;  // at most; a multiple of 32
constexpr int kPairThreads = 256;
constexpr int kChunk = 32;      // accumulator columns an epilogue warp handles at once
constexpr int kStagePitch = kChunk + 1;

struct PairArgs {
  Epilogue e;
  int32_t steps;  // 128-byte boxes along K
  int32_t cols;   // rows of w per tile
  int32_t stages;
  int32_t box_elems;
  uint32_t desc;
  int64_t mt, nt;  // tiles along m and n
  int32_t group;   // m tiles walked together
  int32_t vec;     // y and row_add rows are vectors of 8
};

// Tile t of the walk: `group` m tiles side by side for every n tile, so that
// the pairs at work share both operands' tiles in L2.
FD_DEV void pair_tile(const PairArgs& a, int64_t t, int64_t* mi, int64_t* ni) {
  const int64_t per = static_cast<int64_t>(a.group) * a.nt;
  const int64_t g = t / per, in = t % per;
  const int64_t rows = min(static_cast<int64_t>(a.group), a.mt - g * a.group);
  *mi = g * a.group + in % rows;
  *ni = in / rows;
}

FD_DEV void tma_load_pair(void* dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(fd_stream::smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
FD_DEV void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <typename T, bool FP8>
__global__ void __launch_bounds__(kPairThreads, 1)
    product_pair_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                        const __grid_constant__ PairArgs a) {
  using namespace fd_stream;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kMaxRing], empty[kMaxRing], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort;
  __shared__ __align__(16) float s_bias[2][kPairCols], s_ws[2][kPairCols];
  __shared__ float s_stage[4][32 * kStagePitch];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int half_cols = a.cols / 2;
  const uint32_t xbytes = 128 * kBoxBytes, wbytes = half_cols * kBoxBytes, stage_bytes = xbytes + wbytes;
  const int64_t tiles = a.mt * a.nt, pairs = gridDim.x / 2, first = blockIdx.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);  // four epilogue warps of each CTA
    }
    abort = 0;
    bar_init_fence();
  }
  if (warp == 2) tmem_alloc<2>(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_arrive();  // both CTAs' barriers exist before either is signalled
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  grid_dep_wait();
  grid_dep_launch();

  if (warp == 0) {
    if (lane == 0) {
      prefetch_map(&xmap);
      prefetch_map(&wmap);
      const uint32_t bars = cluster_map(full, 0);
      RingPos p;
      int64_t i = 0;
      bool ok = true;
      for (int64_t t = first; t < tiles && ok; t += pairs) {
        int64_t mi, ni;
        pair_tile(a, t, &mi, &ni);
        const int32_t xr = static_cast<int32_t>(mi * kPairRows + rank * 128);
        const int32_t wr = static_cast<int32_t>(ni * a.cols + rank * half_cols);
        for (int k = 0; k < a.steps; ++k, ++i, p.next(a.stages)) {
          const int s = p.stage;
          if (i >= a.stages && !wait_or_abort(&empty[s], p.phase ^ 1, &abort)) {
            ok = false;
            break;
          }
          // the first CTA's barrier counts the bytes of both
          if (rank == 0) mbar_expect_tx(&full[s], 2 * stage_bytes);
          const uint32_t bar = bars + s * 8;
          uint8_t* dst = ring + static_cast<size_t>(s) * stage_bytes;
          tma_load_pair(dst, &xmap, k * a.box_elems, xr, bar);
          tma_load_pair(dst + xbytes, &wmap, k * a.box_elems, wr, bar);
        }
      }
      // every stage has landed and been read, and its barrier signalled, before the pair may exit
      bool read = true;
      for (int64_t j = i > a.stages ? i - a.stages : 0; j < i; ++j) {
        read = read && wait_phase(&empty[j % a.stages], (j / a.stages) & 1);
        if (!read && rank == 0) wait_phase(&full[j % a.stages], (j / a.stages) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      RingPos p;
      int it = 0;
      bool ok = true;
      for (int64_t t = first; t < tiles && ok; t += pairs, ++it) {
        const int b = it & 1;
        if (!wait_or_abort(&acc_empty[b], ((it >> 1) & 1) ^ 1, &abort)) break;
        tc_fence_after();
        const uint32_t d = tmem + b * kPairCols;
        for (int k = 0; k < a.steps; ++k, p.next(a.stages)) {
          const int s = p.stage;
          if (!wait_or_abort(&full[s], p.phase, &abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t x = smem_addr(ring + static_cast<size_t>(s) * stage_bytes), w = x + xbytes;
#pragma unroll
          for (int kk = 0; kk < kBoxBytes; kk += kSliceBytes)
            tc_mma<FP8, 2>(d, tile_desc(x + kk), tile_desc(w + kk), a.desc, k + kk > 0);
          tc_commit<2>(&empty[s]);
        }
        if (ok) tc_commit<2>(&acc_full[b]);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int q = warp - 4, et = threadIdx.x - 128;
    float* stage = s_stage[q];
    int it = 0;
    bool ok = true;
    for (int64_t t = first; t < tiles; t += pairs, ++it) {
      const int b = it & 1;
      int64_t mi, ni;
      pair_tile(a, t, &mi, &ni);
      const int64_t n0 = ni * a.cols, m0 = mi * kPairRows + rank * 128 + q * 32, m = m0 + lane;
      // the tile's bias and weight scales, loaded under its MMAs
      for (int c = et; c < a.cols; c += 128) {
        const int64_t n = n0 + c;
        const bool in = n < a.e.n;
        s_bias[b][c] = a.e.bias && in ? load_as_f32(a.e.bias, a.e.bias_dtype, n * a.e.sbias) : 0.f;
        if (FP8) s_ws[b][c] = in ? a.e.ws[n] : 0.f;
      }
      const float xs = FP8 && m < a.e.m ? a.e.xs[m] : 1.f;
      named_sync(1, 128);
      // after an expired wait the four warps still meet at every tile's barrier
      ok = __all_sync(0xffffffffu, ok && wait_or_abort(&acc_full[b], (it >> 1) & 1, &abort));
      if (!ok) continue;
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(q * 32) << 16) + b * kPairCols;
      for (int c = 0; c < a.cols; c += kChunk) {
        float v[kChunk];
        tc_load32(acc + c, reinterpret_cast<uint32_t*>(v));
        if (c + kChunk >= a.cols) {  // the accumulator is free for the tile after next
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(cluster_map(&acc_empty[b], 0));
        }
        if (n0 + c >= a.e.n || m0 >= a.e.m) continue;
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          if (FP8) v[j] = v[j] * xs * s_ws[b][c + j];
          v[j] += s_bias[b][c + j];
        }
        activate_all<kChunk>(v, a.e.act);
        if (a.vec) {
          if (m < a.e.m) {
            T* y = static_cast<T*>(a.e.y) + m * a.e.sym + n0 + c;
            const T* ra = static_cast<const T*>(a.e.ra) + (a.e.ra ? m * a.e.srm + n0 + c : 0);
#pragma unroll
            for (int j = 0; j < kChunk; j += 8) {
              if (n0 + c + j >= a.e.n) break;
              if (a.e.ra) {
                float f[8];
                unpack8<T>(*reinterpret_cast<const uint4*>(ra + j), f);
#pragma unroll
                for (int u = 0; u < 8; ++u) v[j + u] += f[u];
              }
              *reinterpret_cast<uint4*>(y + j) = pack8<T>(v + j);
            }
          }
        } else {
          // any layout of y and row_add: through shared memory, a row of 32
          // consecutive columns at a time
          __syncwarp();
#pragma unroll
          for (int j = 0; j < kChunk; ++j) stage[lane * kStagePitch + j] = v[j];
          __syncwarp();
          const int64_t n = n0 + c + lane;
          if (n < a.e.n) {
            for (int r = 0; r < 32 && m0 + r < a.e.m; ++r) {
              float o = stage[r * kStagePitch + lane];
              if (a.e.ra) o += load_as_f32(a.e.ra, a.e.ra_dtype, (m0 + r) * a.e.srm + n * a.e.srn);
              static_cast<T*>(a.e.y)[(m0 + r) * a.e.sym + n * a.e.syn] = from_f32<T>(o);
            }
          }
        }
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();  // the pair's last signals and MMAs have arrived on both sides
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

constexpr size_t kSmemMax = 227 * 1024;
// Tensor memory has 512 columns an SM and an allocation waits for them.  A
// split CTA takes at most 256 and at least this much shared memory, a pair CTA
// all 512 and more than 228 KB less this: no SM ever holds CTAs of theirs that
// want more than there is, so no allocation waits for a CTA that is itself
// waiting for a peer.
constexpr size_t kSplitSmemMin = 80 * 1024;

template <typename Kern, typename Args>
cudaError_t launch_cluster(Kern kern, dim3 grid, int threads, int cluster, size_t smem, cudaStream_t st,
                           const CUtensorMap& m0, const CUtensorMap& m1, const Args& a) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, m0, m1, a);
}

int mma_format(int in_dtype) { return in_dtype == FD_BF16 ? 1 : 0; }

// Few rows.  FD_ERR_UNSUPPORTED: a layout TMA cannot address.
template <typename T, bool FP8>
int launch_split(const GenericArgs& g, int in_dtype, bool w_early, cudaStream_t st) {
  constexpr int es = FP8 ? 1 : 2;
  const Epilogue& e = g.epi;
  SplitArgs a;
  a.e = e;
  const int64_t mblocks = (e.m + 255) / 256;
  const int64_t per = (e.m + mblocks - 1) / mblocks;
  a.cols = static_cast<int32_t>((per + 15) / 16 * 16);
  a.boxes = a.cols <= 64 ? 2 : 1;
  a.box_elems = kBoxBytes / es;
  const int64_t steps = (g.k + a.boxes * a.box_elems - 1) / (a.boxes * a.box_elems);
  const int64_t nblocks = (e.n + kTileRows - 1) / kTileRows;
  const int64_t tiles = nblocks * mblocks;
  const int sms = fd_host::sm_count();
  int split = 1;
  while (split < kMaxSplit && tiles * split * 2 <= sms && steps >= split * 4) split *= 2;
  if (const char* env = std::getenv("FD_PRODUCT_TUNE")) {
    int b = 0, c = 0;
    if (std::sscanf(env, "%d,%d", &b, &c) == 2) {
      if (b > 0) a.boxes = b;
      if (c > 0) split = c;
    }
  }
  if (steps > 0x7fffffffLL || nblocks * split > 0x7fffffffLL || mblocks > 65535) return FD_ERR_UNSUPPORTED;
  a.steps = static_cast<int32_t>(steps);
  a.split = split;
  a.desc = mma_desc(FP8 ? 0 : mma_format(in_dtype), kTileRows, a.cols);
  a.tmem_cols = 32;
  while (a.tmem_cols < static_cast<uint32_t>(a.cols)) a.tmem_cols *= 2;
  a.w_early = w_early;
  const size_t stage = static_cast<size_t>(a.boxes) * kBoxBytes * (kTileRows + a.cols);
  const size_t part = split > 1 ? static_cast<size_t>(a.cols) * kTileRows * 4 : 0;
  size_t budget = tiles * split > sms ? 110 * 1024 : 220 * 1024;
  a.stages = static_cast<int32_t>(std::min<size_t>(kMaxRing, budget / stage));
  if (a.stages < 2) a.stages = 2;
  const size_t smem = std::max(kSplitSmemMin, std::max(a.stages * stage, part) + 1024);
  if (smem > kSmemMax - 1024) return FD_ERR_UNSUPPORTED;
  CUtensorMap wm, xm;
  if (!operand_map(&wm, g.w, e.n, g.k, g.swn, g.swk, es, kTileRows) ||
      !operand_map(&xm, g.x, e.m, g.k, g.sxm, g.sxk, es, a.cols))
    return FD_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(nblocks * split), static_cast<unsigned>(mblocks));
  return from_cuda(launch_cluster(product_split_kernel<T, FP8>, grid, kSplitThreads, split, smem, st, wm, xm, a));
}

// Rows of y (and of row_add, where there is one) as vectors of 8 of type T.
bool epilogue_vec(const Epilogue& e, int out_dtype) {
  if (e.n % 8 || e.syn != 1 || e.sym % 8 || !fd_host::aligned16(e.y)) return false;
  if (!e.ra) return true;
  return e.ra_dtype == out_dtype && e.srn == 1 && e.srm % 8 == 0 && fd_host::aligned16(e.ra);
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
  a.mt = (e.m + kPairRows - 1) / kPairRows;
  // columns per tile: the widest that wastes least of the last wave
  int64_t best = 0;
  a.cols = 0;
  for (int c = kPairCols; c >= 128; c -= 32) {
    const int64_t tiles = a.mt * ((e.n + c - 1) / c);
    const int64_t cost = (tiles + pairs - 1) / pairs * (c + 16);
    if (a.cols == 0 || cost < best) {
      best = cost;
      a.cols = c;
    }
  }
  a.group = 8;
  int max_stages = kMaxRing;
  if (const char* env = std::getenv("FD_PAIR_TUNE")) {
    int b = 0, c = 0, d = 0;
    if (std::sscanf(env, "%d,%d,%d", &b, &c, &d) == 3) {
      if (b > 0) a.cols = b;
      if (c > 0) a.group = c;
      if (d > 0) max_stages = d;
    }
  }
  a.nt = (e.n + a.cols - 1) / a.cols;
  if (steps > 0x7fffffffLL || e.m > 0x7fffff00LL || e.n > 0x7fffff00LL) return FD_ERR_UNSUPPORTED;
  a.steps = static_cast<int32_t>(steps);
  a.desc = mma_desc(FP8 ? 0 : mma_format(in_dtype), kPairRows, a.cols);
  a.vec = epilogue_vec(e, out_dtype);
  const size_t stage = static_cast<size_t>(kBoxBytes) * (128 + a.cols / 2);
  a.stages = static_cast<int32_t>(std::min<size_t>(max_stages, 192 * 1024 / stage));
  const size_t smem = a.stages * stage + 1024;
  CUtensorMap xm, wm;
  if (!operand_map(&xm, g.x, e.m, g.k, g.sxm, g.sxk, es, 128) ||
      !operand_map(&wm, g.w, e.n, g.k, g.swn, g.swk, es, a.cols / 2))
    return FD_ERR_UNSUPPORTED;
  const int64_t grid = 2 * std::min<int64_t>(pairs, a.mt * a.nt);
  return from_cuda(launch_cluster(product_pair_kernel<T, FP8>, dim3(static_cast<unsigned>(grid)), kPairThreads, 2, smem,
                                  st, xm, wm, a));
}

template <typename TX, typename T, bool FP8>
int launch_product(const GenericArgs& g, int in_dtype, int out_dtype, bool w_early, cudaStream_t st) {
  int r = FD_ERR_UNSUPPORTED;
  if (g.k > 0) {
    if (g.epi.m > 256) r = launch_pair<T, FP8>(g, in_dtype, out_dtype, st);
    else r = launch_split<T, FP8>(g, in_dtype, w_early, st);
  }
  return r == FD_ERR_UNSUPPORTED ? launch_generic<TX, T, FP8>(g, st) : r;
}

bool epilogue_ok(const Epilogue& e) {
  return e.y && fd_host::valid_dtype(e.bias_dtype) && fd_host::valid_dtype(e.ra_dtype) && e.act >= FD_ACT_NONE &&
         e.act <= FD_ACT_GELU_TANH;
}

// in_dtype: f16, bf16 or e4m3 (then e.xs and e.ws are set and out_dtype is the
// output's; for 16-bit operands out_dtype = in_dtype).  w_early: the kernel
// before this one on the stream does not write w, and has itself waited for
// everything before it.
int product(const GenericArgs& a, int in_dtype, int out_dtype, bool w_early, cudaStream_t st) {
  const Epilogue& e = a.epi;
  if (e.m < 0 || e.n < 0 || a.k < 0) return FD_ERR_ARG;
  if (e.m == 0 || e.n == 0) return FD_OK;
  if (!epilogue_ok(e) || !fd_host::half_dtype(out_dtype) || (a.k > 0 && (!a.x || !a.w))) return FD_ERR_ARG;
  const bool bf = out_dtype == FD_BF16;
  if (in_dtype == FD_E4M3)
    return bf ? launch_product<__half, __nv_bfloat16, true>(a, in_dtype, out_dtype, w_early, st)
              : launch_product<__half, __half, true>(a, in_dtype, out_dtype, w_early, st);
  return bf ? launch_product<__nv_bfloat16, __nv_bfloat16, false>(a, in_dtype, out_dtype, w_early, st)
            : launch_product<__half, __half, false>(a, in_dtype, out_dtype, w_early, st);
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
  return product({x, sxm, sxk, w, swn, swk, k, e}, dtype, dtype, false, static_cast<cudaStream_t>(stream));
}

int fd_linear_fp8_out(const void* x, int64_t sxm, int64_t sxk, const float* x_scale, const void* w, int64_t swn,
                      int64_t swk, const float* w_scale, const void* bias, int32_t bias_dtype, int64_t sbias,
                      const void* row_add, int32_t ra_dtype, int64_t srm, int64_t srn, void* y, int64_t sym,
                      int64_t syn, int32_t out_dtype, int32_t act, int64_t m, int64_t n, int64_t k, void* stream) {
  if (m > 0 && n > 0 && (!x_scale || !w_scale)) return FD_ERR_ARG;
  const Epilogue e{x_scale, w_scale, bias, bias_dtype, sbias, row_add, ra_dtype, srm, srn, y, sym, syn, m, n, act};
  return product({x, sxm, sxk, w, swn, swk, k, e}, FD_E4M3, out_dtype, false, static_cast<cudaStream_t>(stream));
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
