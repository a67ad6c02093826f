// Rows of logits through shared memory: the common frame of the kernels that read [rows, vocab] once.
//
// A persistent CTA (one per SM) takes every n-th row.  One warp keeps a ring of stages filled with bulk
// asynchronous copies of whole rows; G groups of GT threads take the rows in turn and walk over them in shared
// memory as often as they need.  The memory stays busy while the groups sit at their reductions, and a group's loops
// are a few instructions long.  A row that is too long for a third of the shared memory is split over the CTAs of a
// cluster.
//
// A row may start at any element: the copies take the 16-byte vectors that lie in it, the one or two vectors at
// its ends are read and written element by element.
#pragma once
#include <algorithm>

#include "common.cuh"
#include "errors.h"
#include "ptx.cuh"

namespace eisen {

constexpr int RP_MAX_STAGES = 32;

template <typename T>
__device__ __forceinline__ void unpack_vec(const uint4& r, float (&v)[VecOf<T>::N]) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);  // low half = even element
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  }
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The part [lo, hi) of a row's vectors that one CTA holds.
template <typename T>
struct RowSlice {
  static constexpr int V = VecOf<T>::N;
  const T* base;  // the row's first element, moved down to a 16-byte boundary
  int lead;       // elements of the first vector in front of the row
  int n;          // elements of the row
  int lo, hi;     // vectors of this CTA
  int w0, w1;     // those of them that lie in the row
  // the rank-th of 2^parts_log2 slices
  __device__ __forceinline__ RowSlice(const T* row, int len, int rank, int parts_log2) {
    lead = (int)(((uint32_t)reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - lead;
    n = len;
    const int all = (lead + n + V - 1) / V, per = (all + (1 << parts_log2) - 1) >> parts_log2;
    lo = min(rank * per, all);
    hi = min(lo + per, all);
    w0 = max(lo, lead ? 1 : 0);
    w1 = max(min(hi, (lead + n) / V), w0);
  }
  __device__ __forceinline__ int first(int vec) const { return vec * V - lead; }  // row index of its first element
  // a vector that reaches beyond an end of the row, -inf in the places outside
  __device__ __noinline__ uint4 load_edge(int vec) const {
    uint32_t u[4];
    const int e0 = first(vec);
    if constexpr (sizeof(T) == 2) {
      const uint16_t* b = reinterpret_cast<const uint16_t*>(base) + (long long)vec * V;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t l = (e0 + 2 * i >= 0 && e0 + 2 * i < n) ? b[2 * i] : 0xff80u;
        const uint32_t h = (e0 + 2 * i + 1 >= 0 && e0 + 2 * i + 1 < n) ? b[2 * i + 1] : 0xff80u;
        u[i] = l | (h << 16);
      }
    } else {
      const uint32_t* b = reinterpret_cast<const uint32_t*>(base) + (long long)vec * V;
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = (e0 + i >= 0 && e0 + i < n) ? b[i] : 0xff800000u;
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// N vectors of a row, `step` apart, all in flight together; -inf in the places that are not in the slice.  Past the L1
// cache: a row does not fit there.
template <typename T, int N>
__device__ __forceinline__ void load_vectors(const RowSlice<T>& s, int v0, int step, uint4 (&raw)[N]) {
  if (v0 >= s.w0 && v0 + (N - 1) * step < s.w1) {
    const T* at = s.base + (long long)v0 * RowSlice<T>::V;
#pragma unroll
    for (int q = 0; q < N; ++q)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(raw[q].x), "=r"(raw[q].y), "=r"(raw[q].z), "=r"(raw[q].w)
                   : "l"(at + (long long)q * step * RowSlice<T>::V));
    return;
  }
  constexpr uint32_t low = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const int v = v0 + q * step;
    raw[q] = make_uint4(low, low, low, low);
    if (v >= s.w0 && v < s.w1) {
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(raw[q].x), "=r"(raw[q].y), "=r"(raw[q].z), "=r"(raw[q].w)
                   : "l"(s.base + (long long)v * RowSlice<T>::V));
    } else if (v < s.hi) {
      raw[q] = s.load_edge(v);
    }
  }
}

// ---- clusters of CTAs that share a row
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
// arrival that publishes this thread's earlier writes to the peer that waits on the barrier
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      "selp.b32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void mbar_wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait_cluster(bar, parity) || *abort_flag) return;
  const long long t0 = clock64();
  while (!mbar_try_wait_cluster(bar, parity)) {
    if (*abort_flag) return;
    if (clock64() - t0 > EISEN_WAIT_CYCLES) { *abort_flag = 1; return; }
  }
}

// ---- one group of GT threads
template <int GT>
__device__ __forceinline__ void group_sync(int g) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + g), "n"(GT) : "memory");
}
// sum / maximum over W consecutive lanes
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int W>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// barriers of a CTA's ring
struct RowRing {
  uint64_t full[RP_MAX_STAGES];   // 1 arrival and the bytes of the copy
  uint64_t empty[RP_MAX_STAGES];  // the warps of the group that read the stage
  volatile int issued;            // rows the loading warp has sent for
  int abort_flag;
};

__device__ __forceinline__ void ring_init(RowRing& r, int stages, int group_warps) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&r.full[i], 1);
      mbar_init(&r.empty[i], group_warps);
    }
    r.abort_flag = 0;
    r.issued = 0;
    fence_mbar_init();
  }
}

// Waits until the copy of this CTA's i-th row has landed.  Successive rows of a stage may belong to different groups, and
// a group that runs ahead (over rows that are skipped) must not take the end of the stage's row before for its own: a
// row is sent for only after that one was used up, so once it is, the phase of its own copy is the current one.
__device__ __forceinline__ void ring_wait_row(RowRing& r, int i, int stage, uint32_t phase, long long budget = EISEN_WAIT_CYCLES) {
  if (r.issued <= i) {
    const long long t0 = clock64();
    while (r.issued <= i) {
      if (*(volatile int*)&r.abort_flag) return;
      if (clock64() - t0 > budget) { *(volatile int*)&r.abort_flag = 1; return; }
    }
  }
  __threadfence_block();
  mbar_wait(&r.full[stage], phase, &r.abort_flag, nullptr, FAULT_WAIT_FULL, budget);
}

// The end of a kernel, for all of its threads: true where a wait of this CTA ran out, so that the rows it shares in cannot be
// relied on and are to be marked.  Groups go on after such a wait, so every warp of the CTA, and of the cluster's other CTAs, has to be
// through before anything is marked, or a row would be written over its mark.  (A cluster's CTAs do not leave before that
// anyway: a peer may still write to them or read their lists.)  The copies in flight end before the CTA does.
__device__ __forceinline__ bool ring_gave_up(RowRing& r, int cluster, int* fault_word) {
  __syncthreads();
  if (cluster > 1) cluster_sync_all();
  if (!*(volatile int*)&r.abort_flag) return false;
  if (threadIdx.x == 0 && fault_word) atomicCAS(fault_word, 0, FAULT_WAIT_ROWS);
  for (int i = 0; i < 64; ++i) __nanosleep(1000);
  return true;
}

// The loading warp.  slice(row) -> RowSlice; skip(row): the row's logits are not looked at (its stage passes
// through the ring empty).  skip is asked for 32 rows at a time, one per lane.
template <typename T, typename Slice, typename Skip>
__device__ __forceinline__ void ring_load(RowRing& r, uint8_t* smem, int stages, int stage_bytes, int n_mine, long long row0,
                                          long long stride, Slice slice, Skip skip) {
  const int lane = threadIdx.x & 31;
  int st = 0;
  uint32_t phase = 1;
  for (int i0 = 0; i0 < n_mine; i0 += 32) {
    const bool mine = i0 + lane < n_mine && skip(row0 + (long long)(i0 + lane) * stride);
    const uint32_t skips = __ballot_sync(0xffffffffu, mine);
    bool given_up = false;
    if (lane == 0) {
      const int m = min(32, n_mine - i0);
      for (int i = 0; i < m; ++i) {
        given_up = !mbar_wait(&r.empty[st], phase, &r.abort_flag, nullptr, FAULT_WAIT_EMPTY);
        if (given_up) break;
        const RowSlice<T> s = slice(row0 + (long long)(i0 + i) * stride);
        const uint32_t bytes = (uint32_t)(s.w1 - s.w0) * 16;
        if (((skips >> i) & 1) || bytes == 0) {
          mbar_arrive(&r.full[st]);
        } else {
          mbar_arrive_expect_tx(&r.full[st], bytes);
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                           smem_u32(smem + (size_t)st * stage_bytes + (size_t)(s.w0 - s.lo) * 16)),
                       "l"(s.base + (long long)s.w0 * RowSlice<T>::V), "r"(bytes), "r"(smem_u32(&r.full[st]))
                       : "memory");
        }
        __threadfence_block();
        r.issued = i0 + i + 1;
        if (++st == stages) { st = 0; phase ^= 1; }
      }
    }
    if (__any_sync(0xffffffffu, given_up)) return;  // nothing more is sent for
  }
}

// ---- host: shape of a launch
struct RowShape {
  int cluster, cluster_log2, stages, stage_bytes, smem;
};

// Shared memory a CTA may use, less a little for its static part.
constexpr int RP_SMEM = 216 * 1024;

// `extra`: dynamic shared memory beside the stages.  A row of up to a third of the stage memory stays whole (three
// stages keep the memory busy while two groups work); longer rows are split over 2, 4 or 8 CTAs, but for those
// that would take 4 and fit one CTA whole (1024 x 100003 bf16, loss and gradient: 107 us whole, 128 in four slices that meet
// for every row), and so are rows that alone leave SMs idle, down to slices of `least` bytes.  stages == 0: no split fits.
inline RowShape row_shape(long long rows, long long vocab, int elem, int extra, int want_stages, int least) {
  RowShape s = {};
  const long long row_bytes = (vocab * elem + 31) / 16 * 16;
  const long long room = RP_SMEM - extra;
  int c = 1;
  auto slice = [&](int cl) { return ((row_bytes / 16 + cl - 1) / cl * 16 + 127) / 128 * 128; };
  while (c < 8 && slice(c) * 3 > room) c *= 2;
  if (c >= 4 && slice(1) <= room) c = 1;
  while (c < 8 && rows * c * 2 <= sm_count() && row_bytes / (2 * c) >= least) c *= 2;
  if (slice(c) > room || slice(c) > (1 << 20)) return s;
  s.cluster = c;
  s.cluster_log2 = c == 1 ? 0 : c == 2 ? 1 : c == 4 ? 2 : 3;
  s.stage_bytes = (int)slice(c);
  s.stages = (int)std::min<long long>(std::min<long long>(want_stages, RP_MAX_STAGES), room / s.stage_bytes);
  s.smem = s.stages * s.stage_bytes + extra;
  return s;
}

template <auto KERNEL, typename P>
int launch_pipe(const char* what, const RowShape& s, long long rows, int threads, cudaStream_t stream, const P& p) {
  static bool attr_set[MAX_DEVICE_SLOTS] = {false};  // one per kernel
  static int resident[MAX_DEVICE_SLOTS][4] = {{0}};  // clusters of 1, 2, 4, 8 CTAs that run at the same time
  const int slot = device_slot();
  if (!attr_set[slot]) {
    const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, RP_SMEM);
    if (e != cudaSuccess) return fail(EISEN_ERR_CUDA, cudaGetErrorString(e));
    attr_set[slot] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sm_count() / s.cluster * s.cluster), 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = RP_SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)s.cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.cluster > 1 ? 1 : 0;
  // the rows are dealt out over clusters that are all resident (a cluster's CTAs share a group of SMs, and the groups
  // do not divide evenly): one more would start when another ends, and take as long again
  int& n = resident[slot][s.cluster_log2];
  if (!n) {
    int most = sm_count();
    if (s.cluster > 1 && (cudaOccupancyMaxActiveClusters(&most, KERNEL, &cfg) != cudaSuccess || most <= 0)) {
      cudaGetLastError();
      most = std::max(sm_count() / s.cluster / 2, 1);
    }
    n = most;
  }
  cfg.gridDim = dim3((unsigned)(std::min<long long>(rows, n) * s.cluster), 1, 1);
  cfg.dynamicSmemBytes = (size_t)s.smem;
  cudaLaunchKernelEx(&cfg, KERNEL, p);  // its status is read by check_launch
  return check_launch(what);
}

}  // namespace eisen
