// A row of logits held in registers by one CTA, or slice by slice by the CTAs of a cluster.  The row may start at
// any element: it is read as the 16-byte vectors that cover it, the one or two vectors that reach beyond it
// element by element, with -inf in the places outside.
#pragma once
#include "common.cuh"
#include "errors.h"
#include "ptx.cuh"

namespace eisen {

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

template <typename T>
struct RowView {
  static constexpr int V = VecOf<T>::N;
  const T* base;  // the row's first element, moved down to a 16-byte boundary
  int lead;       // elements of the first vector in front of the row
  int n;          // elements of the row
  __device__ __forceinline__ RowView(const T* row, int len) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - lead;
    n = len;
  }
  __device__ __forceinline__ int vectors() const { return (lead + n + V - 1) / V; }
  __device__ __forceinline__ int first(int vec) const { return vec * V - lead; }  // row index of its first element
  // vectors inside the row: [whole_lo, whole_hi)
  __device__ __forceinline__ int whole_lo() const { return lead ? 1 : 0; }
  __device__ __forceinline__ int whole_hi() const { return (lead + n) / V; }
  // a vector that lies in the row; used once, kept out of L1
  __device__ __forceinline__ static uint4 load_whole(const T* at) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(at));
    return r;
  }
  // one that reaches beyond an end of it
  __device__ __noinline__ uint4 load_edge(int vec) const {
    uint32_t u[4];
    const int e0 = first(vec);
    if constexpr (sizeof(T) == 2) {
      const uint16_t* b = reinterpret_cast<const uint16_t*>(base) + (long long)vec * V;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (e0 + 2 * i >= 0 && e0 + 2 * i < n) ? b[2 * i] : 0xff80u;
        const uint32_t hi = (e0 + 2 * i + 1 >= 0 && e0 + 2 * i + 1 < n) ? b[2 * i + 1] : 0xff80u;
        u[i] = lo | (hi << 16);
      }
    } else {
      const uint32_t* b = reinterpret_cast<const uint32_t*>(base) + (long long)vec * V;
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = (e0 + i >= 0 && e0 + i < n) ? b[i] : 0xff800000u;
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// -inf in every place of a vector
template <typename T>
__device__ __forceinline__ uint4 minus_inf_vec() {
  constexpr uint32_t w = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  return make_uint4(w, w, w, w);
}

// This thread's vectors lo + tid, lo + tid + THREADS, ... < hi of a row; -inf beyond
template <typename T, int THREADS, int NV>
__device__ __forceinline__ void load_slice(const RowView<T>& view, int lo, int hi, uint4 (&raw)[NV]) {
  const int w0 = max(lo, view.whole_lo()), w1 = min(hi, view.whole_hi());
  const int v0 = lo + (int)threadIdx.x;
  const T* at = view.base + (long long)v0 * VecOf<T>::N;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int v = v0 + j * THREADS;
    if (v >= w0 && v < w1) raw[j] = RowView<T>::load_whole(at + j * (THREADS * VecOf<T>::N));
    else raw[j] = minus_inf_vec<T>();
  }
  // the one or two vectors at the row's ends, by the threads that own them
  if (v0 < w0 || hi > w1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = v0 + j * THREADS;
      if (v < hi && (v < w0 || v >= w1)) raw[j] = view.load_edge(v);
    }
  }
}

// largest element of NV vectors; NaN where one of them is NaN
template <typename T, int NV>
__device__ __forceinline__ float max_of(const uint4 (&raw)[NV]) {
  if constexpr (sizeof(T) == 2) {
    auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    __nv_bfloat162 m = pair(raw[0].x);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      m = __hmax2_nan(m, pair(raw[j].x));
      m = __hmax2_nan(m, pair(raw[j].y));
      m = __hmax2_nan(m, pair(raw[j].z));
      m = __hmax2_nan(m, pair(raw[j].w));
    }
    const float a = __low2float(m), b = __high2float(m);
    return a != a ? a : (b != b ? b : fmaxf(a, b));
  } else {
    float m = __uint_as_float(raw[0].x);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t u[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float d;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(m), "f"(__uint_as_float(u[i])));
        m = d;
      }
    }
    return m;
  }
}

// ---- clusters of CTAs that share a row (cluster size 1: everything below is skipped by the callers)
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t addr) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// CTAs per row: enough that a slice of the row fits the registers of a CTA (`most` vectors), and, where the rows
// alone leave SMs idle, more of them down to `least` vectors a slice.  0: the row is too long.
inline int cluster_for_row(long long rows, long long vectors, int most, int least) {
  int c = 1;
  while (c <= 8 && (vectors + c - 1) / c > most) c *= 2;
  if (c > 8) return 0;
  while (c < 8 && rows * c * 2 <= sm_count() && vectors / (2 * c) >= least) c *= 2;
  return c;
}

template <typename K, typename... A>
int launch_rows(K kernel, const char* what, long long rows, int cluster, int threads, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster), 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return check_launch(what);
}

}  // namespace eisen
