// The k largest logits of every row in descending order (equal values: the lowest index first), and the row's
// log-sum-exp at a temperature: what a teacher hands to a student (distill.cu).
//
// The threads of a CTA
//   1. take the largest element of every thread's share: the k-th largest of these is a threshold that at least k
//      elements of the row reach and, on rows in no special order, few more do;
//   2. list the elements that reach it;
//   3. rank the listed ones against each other.
// Few rows (two per SM at most) are read once, into shared memory (row_pipe.cuh, split over a cluster's CTAs where they alone
// leave SMs idle), and the exponentials are added up in the second pass.  Rows in numbers stay where they are: many small CTAs read
// them once for the maxima and the sum, and note which vectors to look into again (top_stream_kernel).
// Keys are 64 bits, value above complemented index, so every two differ and nothing depends on the order of arrival.
// Rows whose large values sit in a few threads' shares (or are equal in thousands) overflow the list; for them the
// exact threshold is found digit by digit over all elements, first of the value, then of the index.
#include <algorithm>
#include <cfloat>
#include <cstdio>

#include "common.cuh"
#include "errors.h"
#include "row_pipe.cuh"
#include "../../include/eisen_b200.h"

namespace eisen {
namespace {

constexpr int TOP_MAX_K = 256;

struct TopParams {
  const void* logits;
  long long ld;
  float* values;
  int* ids;
  float* lse;
  long long rows;
  int vocab, k;
  float inv_t;
  int* fault_word;
  int keyed;  // top_stream_kernel: there is room for the vectors' keys
  RowShape shape;
};

// order of the values as unsigned integers: -0 equals +0, NaN comes first
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// largest element of a vector; NaN where one of them is NaN
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& r) {
  if constexpr (sizeof(T) == 2) {
    auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(pair(r.x), pair(r.y)), __hmax2_nan(pair(r.z), pair(r.w)));
    return max_nan(__low2float(m), __high2float(m));
  } else {
    return max_nan(max_nan(__uint_as_float(r.x), __uint_as_float(r.y)), max_nan(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
}

// whether an element of a vector is not below `floor` (its upper 16 bits are the threshold's: for bf16 they are all that
// counts)
template <typename T>
__device__ __forceinline__ bool reaches(const uint4& r, float floor) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t f = __float_as_uint(floor) >> 16, ff = f | (f << 16);
    auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const uint32_t below = __hlt2_mask(pair(r.x), pair(ff)) & __hlt2_mask(pair(r.y), pair(ff)) & __hlt2_mask(pair(r.z), pair(ff)) &
                           __hlt2_mask(pair(r.w), pair(ff));
    return below != 0xffffffffu;
  } else {
    return !(__uint_as_float(r.x) < floor) || !(__uint_as_float(r.y) < floor) || !(__uint_as_float(r.z) < floor) ||
           !(__uint_as_float(r.w) < floor);
  }
}

// Upper 16 bits of the key of a vector's largest element; `most` takes that element into a maximum without NaN.  bf16: the key
// from the element's own 16 bits (adding 0 makes one zero of the two; a NaN of the packed maximum is 0x7fff).
template <typename T>
__device__ __forceinline__ uint32_t vec_key(const uint4& r, float& most) {
  if constexpr (sizeof(T) == 2) {
    auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(pair(r.x), pair(r.y)), __hmax2_nan(pair(r.z), pair(r.w)));
    m = __hadd2(__hmax2_nan(m, __lowhigh2highlow(m)), pair(0u));
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&m) & 0xffffu;
    most = fmaxf(most, __uint_as_float(u << 16));
    return (u & 0x8000u) ? u ^ 0xffffu : u | 0x8000u;
  } else {
    const float x = vec_max<T>(r);
    most = fmaxf(most, x);
    return order_key(x) >> 16;
  }
}

// f(rank, key) for the listed keys, at least for the `most` largest of them.  Up to 96 keys by counting those that are larger
// (2 or 4 threads share a key's comparisons where there are threads enough); more are sorted in place, which takes
// log^2 steps instead of `listed`: 8192 x 16000 bf16, k 128: 162 us by counting, 140 sorted.  The list has room up to the next
// power of two.  sync(): a barrier of the THREADS threads.
template <int THREADS, typename Sync, typename F>
__device__ __forceinline__ void each_rank(uint64_t* list, int listed, int most, int tid, Sync sync, F f) {
  if (listed <= 96) {
    const int share = 4 * listed <= THREADS ? 2 : 2 * listed <= THREADS ? 1 : 0;  // log2
    const int part = tid & ((1 << share) - 1);
    for (int j0 = 0; j0 < listed; j0 += THREADS >> share) {
      const int j = j0 + (tid >> share);
      const uint64_t c = j < listed ? list[j] : ~0ull;
      int r = 0;
      const ulonglong2* two = reinterpret_cast<const ulonglong2*>(list);
#pragma unroll 4
      for (int o = part; o < listed / 2; o += 1 << share) {
        const ulonglong2 l = two[o];
        r += (l.x > c) + (l.y > c);
      }
      if ((listed & 1) && part == 0) r += list[listed - 1] > c;
      if (share > 0) r += __shfl_xor_sync(0xffffffffu, r, 1);
      if (share > 1) r += __shfl_xor_sync(0xffffffffu, r, 2);
      if (j < listed && part == 0) f(r, c);
    }
    return;
  }
  int all = 128;
  while (all < listed) all *= 2;
  for (int j = listed + tid; j < all; j += THREADS) list[j] = 0;  // below every key
  for (int size = 2; size <= all; size *= 2)
    for (int stride = size / 2; stride > 0; stride /= 2) {
      sync();
      for (int i = tid; i < all / 2; i += THREADS) {
        const int lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const uint64_t a = list[lo], b = list[hi];
        if ((a < b) == ((lo & size) == 0)) {  // runs of `size` fall and rise in turn; the last one falls
          list[lo] = b;
          list[hi] = a;
        }
      }
    }
  sync();
  for (int j = tid; j < min(listed, most); j += THREADS) f(j, list[j]);
}

// how many of a group's threads say so (a barrier of the group)
template <int GT>
__device__ __forceinline__ int group_count(int g, bool yes) {
  int n;
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.u32 p, %1, 0;\nbar.red.popc.u32 %0, %2, %3, p;\n}"
      : "=r"(n)
      : "r"((uint32_t)yes), "r"(1 + g), "n"(GT)
      : "memory");
  return n;
}

// One warp: the bin of 256 at which the count from the top reaches `want`.  out = bin, count above it, count in it.
__device__ __forceinline__ void pick_bin(const int* hist, int want, int* out) {
  const int lane = threadIdx.x & 31;
  int c[8], total = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) { c[i] = hist[255 - lane * 8 - i]; total += c[i]; }
  int before = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  before -= total;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (before < want && before + c[i] >= want) { out[0] = 255 - lane * 8 - i; out[1] = before; out[2] = c[i]; }
    before += c[i];
  }
}

struct TopSelect {
  int hist[256];
  int pick[3];
};

// The k-th largest key of a set by digits of eight bits, first of the value, then (where the last bin holds more than are
// wanted) of the complemented index.  each(f): f(index, value) for every element that the calling thread owns; sync(): a
// barrier of the threads that share the set; tid: this thread's number among them (at least 32 of them).
template <int THREADS, typename Each, typename Sync>
__device__ void exact_threshold(TopSelect& s, int tid, int k, int all, uint32_t& value, uint32_t& last, Each each, Sync sync) {
  uint32_t prefix = 0, mask = 0;
  int want = k, in_bin = all;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) s.hist[i] = 0;
    sync();
    each([&](int, float x) {
      const uint32_t key = order_key(x);
      if ((key & mask) == prefix) atomicAdd(&s.hist[(key >> shift) & 255], 1);
    });
    sync();
    if (tid < 32) pick_bin(s.hist, want, s.pick);
    sync();
    prefix |= (uint32_t)s.pick[0] << shift;
    mask |= 255u << shift;
    want -= s.pick[1];
    in_bin = s.pick[2];
    sync();
  }
  value = prefix;
  last = 0xffffffffu;  // highest index taken among the elements equal to the threshold
  if (in_bin > want) {
    uint32_t ip = 0, im = 0;  // the largest complements are the lowest indices
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += THREADS) s.hist[i] = 0;
      sync();
      each([&](int i, float x) {
        const uint32_t c = ~(uint32_t)i;
        if (order_key(x) == prefix && (c & im) == ip) atomicAdd(&s.hist[(c >> shift) & 255], 1);
      });
      sync();
      if (tid < 32) pick_bin(s.hist, want, s.pick);
      sync();
      ip |= (uint32_t)s.pick[0] << shift;
      im |= 255u << shift;
      want -= s.pick[1];
      sync();
    }
    last = ~ip;
  }
}

// f(index, value) for the vectors of a slice in shared memory that belong to thread gt of GT; places outside the row
// are left out
template <typename T, int GT, typename F>
__device__ __forceinline__ void each_element(const RowSlice<T>& s, const uint4* vec, int gt, F f) {
  constexpr int V = RowSlice<T>::V;
  const int cnt = s.hi - s.lo;
#pragma unroll 1
  for (int v = gt; v < cnt; v += GT) {
    float x[V];
    unpack_vec<T>(vec[v], x);
    const int e = s.first(s.lo + v);
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (e + c >= 0 && e + c < s.n) f(e + c, x[c]);
  }
}

__host__ __device__ constexpr int top_list(int k) { return k <= 64 ? 256 : 1024; }  // entries of a group's list

template <typename T, int GT>
__global__ void __launch_bounds__(GT + 32, 1)
top_pipe_kernel(const TopParams p) {
  constexpr int V = VecOf<T>::N, GW = GT / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ RowRing ring;
  __shared__ uint64_t xbar, xdone;  // all slices' lists are there; the first CTA has read them
  __shared__ float s_max[GW], s_sum[GW];
  __shared__ uint32_t s_range[GW];
  __shared__ int s_count, s_hits;
  __shared__ __align__(8) float s_slice[2];  // a slice's maximum and sum
  __shared__ TopSelect s_sel;
  const int tid = threadIdx.x, lane = tid & 31;
  const int C = p.shape.cluster, k = p.k, n = p.vocab, cap = top_list(k);
  const int rank = C > 1 ? (int)cluster_ctarank() : 0;
  const long long row0 = blockIdx.x >> p.shape.cluster_log2, stride = gridDim.x >> p.shape.cluster_log2;
  const int n_mine = row0 < p.rows ? (int)((p.rows - row0 + stride - 1) / stride) : 0;
  ring_init(ring, p.shape.stages, GW);
  if (tid == 0) {
    mbar_init(&xbar, C);
    mbar_init(&xdone, 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (C > 1) cluster_sync_all();
  const T* logits = reinterpret_cast<const T*>(p.logits);
  auto slice_of = [&](long long row) { return RowSlice<T>(logits + row * p.ld, n, rank, p.shape.cluster_log2); };
  if (tid >= GT) {
    ring_load<T>(ring, smem, p.shape.stages, p.shape.stage_bytes, n_mine, row0, stride, slice_of, [](long long) { return false; });
  } else {
    const int gt = tid, warp = gt >> 5;
    uint64_t* list = reinterpret_cast<uint64_t*>(smem + (size_t)p.shape.stages * p.shape.stage_bytes);
    int* hits = reinterpret_cast<int*>(list + cap);  // vectors with an element that reaches the threshold
    uint64_t* best = list + cap + cap / 2;  // this slice's k largest in descending order (clusters)
    uint64_t* all = best + TOP_MAX_K;       // every slice's, in the first CTA
    int stage = -1;  // the stage of row i, and its phase
    uint32_t phase = 0, turn = 0;
    for (int i = 0; i < n_mine; ++i, ++turn) {
      if (++stage == p.shape.stages) { stage = 0; phase ^= 1; }
      const long long row = row0 + (long long)i * stride;
      const RowSlice<T> s = slice_of(row);
      // the vectors at the row's ends, by the threads that walk over them
      uint4 edge0 = make_uint4(0, 0, 0, 0), edge1 = edge0;
      const bool own0 = s.w0 > s.lo && gt == 0, own1 = s.w1 < s.hi && s.hi - 1 >= s.w0 && gt == (s.hi - 1 - s.lo) % GT;
      if (own0) edge0 = s.load_edge(s.lo);
      if (own1) edge1 = s.load_edge(s.hi - 1);
      uint4* vec = reinterpret_cast<uint4*>(smem + (size_t)stage * p.shape.stage_bytes);
      const int cnt = s.hi - s.lo;
      const int e_lo = max(s.first(s.lo), 0), here = max(min(s.first(s.hi), n) - e_lo, 0);  // elements of this slice
      const int kk = min(k, here);
      ring_wait_row(ring, i, stage, phase);
      if (own0) vec[0] = edge0;
      if (own1) vec[cnt - 1] = edge1;

      // ---- largest elements of this thread's four shares; NaN counts as the largest
      float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
      for (int v = gt; v < cnt; v += 4 * GT) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (v + q * GT < cnt) m[q] = max_nan(m[q], vec_max<T>(vec[v + q * GT]));
      }
      const float most = max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
      if (gt == 0) { s_count = 0; s_hits = 0; }
      const uint32_t top_key = gt < cnt ? order_key(most) >> 16 : 0;
      const float wm = warp_max(most);  // drops NaN, which the sum brings back
      const uint32_t k_hi = __reduce_max_sync(0xffffffffu, top_key);
      const uint32_t k_lo = __reduce_min_sync(0xffffffffu, gt < cnt ? top_key : 0xffffu);
      if (lane == 0) { s_max[warp] = wm; s_range[warp] = (k_hi << 16) | k_lo; }
      group_sync<GT>(0);
      // the bits in which the threads' maxima agree are the threshold's too
      uint32_t hi16 = 0, lo16 = 0xffffu;
#pragma unroll
      for (int w = 0; w < GW; ++w) {
        hi16 = max(hi16, s_range[w] >> 16);
        lo16 = min(lo16, s_range[w] & 0xffffu);
      }
      const int bits = 32 - __clz(hi16 ^ lo16);
      // ---- threshold: the kk-th largest of the threads' maxima in their upper 16 bits, by bisection.  Where kk is more than
      // half of the threads, the lesser of so many maxima would let too much through: then of the four shares' maxima
      uint32_t tau = 0;
      if (2 * kk <= min(cnt, GT)) {
        tau = (hi16 >> bits) << bits;
#pragma unroll 1
        for (int bit = bits - 1; bit >= 0; --bit) {
          const uint32_t trial = tau | (1u << bit);
          if (group_count<GT>(0, top_key >= trial) >= kk) tau = trial;  // trial is not 0: threads without a share do not count
        }
      } else if (kk <= min(cnt, 4 * GT)) {
        uint32_t key[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) key[q] = gt + q * GT < cnt ? order_key(m[q]) >> 16 : 0;
#pragma unroll 1
        for (int bit = 15; bit >= 0; --bit) {
          const uint32_t trial = tau | (1u << bit);  // never 0: places without a share do not count
          int total = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) total += group_count<GT>(0, key[q] >= trial);
          if (total >= kk) tau = trial;
        }
      }
      group_sync<GT>(0);
      float ref = lanes_max<GW>(s_max[lane % GW]);
      if (ref == -INFINITY) ref = 0.0f;
      // every element whose key reaches tau; NaN does, and so does everything where tau is 0
      const float floor_value = key_value(tau << 16);
      const float c2 = 1.4426950408889634f * p.inv_t, off = -ref * c2;
      const bool far = sizeof(T) == 4 || fabsf(ref) * p.inv_t > 1e4f;
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint4 next = gt < cnt ? vec[gt] : make_uint4(0, 0, 0, 0);
      // a thread notes which of its vectors hold such an element (32 at a time); looking into them here would hold up
      // the other 31 lanes of the warp
#pragma unroll 1
      for (int v0 = gt; v0 - gt < cnt; v0 += 32 * GT) {
        uint32_t noted = 0;
#pragma unroll 1
        for (int j = 0; j < 32; ++j) {
          const int v = v0 + j * GT;
          if (v >= cnt) break;
          const uint4 r = next;
          if (v + GT < cnt) next = vec[v + GT];  // on its way while this one is worked on
          noted |= (uint32_t)reaches<T>(r, floor_value) << j;
          if (p.lse) {
            float x[V];
            unpack_vec<T>(r, x);
            if (far) {
#pragma unroll
              for (int c = 0; c < V; ++c) acc[c & 3] += expf((x[c] - ref) * p.inv_t);
            } else {
#pragma unroll
              for (int c = 0; c < V; ++c) acc[c & 3] += exp2_approx(fmaf(x[c], c2, off));
            }
          }
        }
        // the notes of a warp, one after the other, into the group's list of vectors
        int mine = __popc(noted), before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += up;
        }
        int at = 0;
        if (lane == 31 && before) at = atomicAdd(&s_hits, before);
        at = __shfl_sync(0xffffffffu, at, 31) + before - mine;
        for (; noted; noted &= noted - 1, ++at)
          if (at < cap) hits[at] = v0 + (__ffs(noted) - 1) * GT;
      }
      float sum = (acc[0] + acc[1]) + (acc[2] + acc[3]);
      sum = warp_sum(sum);
      if (lane == 0) s_sum[warp] = sum;
      group_sync<GT>(0);
      sum = lanes_sum<GW>(s_sum[lane % GW]);
      const int noted = s_hits;
      if (noted <= cap) {
        for (int j = gt; j < noted; j += GT) {
          float x[V];
          const int v = hits[j], e = s.first(s.lo + v);
          unpack_vec<T>(vec[v], x);
          uint32_t in = 0;
#pragma unroll
          for (int c = 0; c < V; ++c) in |= (uint32_t)(!(x[c] < floor_value) && e + c >= 0 && e + c < n) << c;
          int at = atomicAdd(&s_count, __popc(in));
#pragma unroll
          for (int c = 0; c < V; ++c)
            if ((in >> c) & 1) {
              if (at < cap) list[at] = ((uint64_t)order_key(x[c]) << 32) | (uint32_t)~(e + c);
              ++at;
            }
        }
      }
      group_sync<GT>(0);
      int listed = noted <= cap ? s_count : cap + 1;
      if (listed > cap) {
        uint32_t value, last;
        exact_threshold<GT>(s_sel, gt, kk, here, value, last, [&](auto f) { each_element<T, GT>(s, vec, gt, f); },
                            [&]() { group_sync<GT>(0); });
        if (gt == 0) s_count = 0;
        group_sync<GT>(0);
        each_element<T, GT>(s, vec, gt, [&](int e, float x) {
          const uint32_t q = order_key(x);
          if (q > value || (q == value && (uint32_t)e <= last)) {
            const int at = atomicAdd(&s_count, 1);
            if (at < cap) list[at] = ((uint64_t)q << 32) | (uint32_t)~e;
          }
        });
        group_sync<GT>(0);
        listed = min(s_count, cap);
      }
      fence_proxy_async_smem();  // the vectors at the ends, before a copy takes their place
      mbar_arrive_warp(&ring.empty[stage]);

      // ---- ranks.  Places of a slice's list that no element takes hold 0, below every key
      float top = ref;  // the row's largest
      auto put = [&](int r, uint64_t c) {
        const float v = key_value((uint32_t)(c >> 32));
        p.values[row * k + r] = v;
        p.ids[row * k + r] = (int)~(uint32_t)c;
        if (r == 0 && p.lse && top == INFINITY) p.lse[row] = v;  // inf or NaN, where the sum ran into inf - inf
      };
      if (C == 1) {
        if (gt == 0 && p.lse && top != INFINITY) p.lse[row] = ref * p.inv_t + logf(sum);
        each_rank<GT>(list, listed, k, gt, [&]() { group_sync<GT>(0); }, [&](int r, uint64_t c) { if (r < k) put(r, c); });
        group_sync<GT>(0);  // the list is read before the next row's takes its place
      } else {
        if (gt == 0) { s_slice[0] = sum == 0.0f ? -INFINITY : ref; s_slice[1] = sum; }
        for (int j = gt + kk; j < k; j += GT) best[j] = 0;
        each_rank<GT>(list, listed, k, gt, [&]() { group_sync<GT>(0); }, [&](int r, uint64_t c) { if (r < k) best[r] = c; });
        group_sync<GT>(0);
        if (gt == 0) mbar_arrive_release_cluster(mapa_cluster(smem_u32(&xbar), 0));
        if (rank == 0) {
          mbar_wait_cluster(&xbar, turn & 1, &ring.abort_flag);
          const uint32_t b0 = smem_u32(best), s0 = smem_u32(&s_slice[0]);
          top = -INFINITY;
          for (int o = 0; o < C; ++o) top = fmaxf(top, __uint_as_float((uint32_t)ld_cluster_u64(mapa_cluster(s0, o))));
          // the slices' lists into this CTA's memory: a search over there costs its latency step by step
          for (int j = gt; j < C * k; j += GT) {
            const int from = j / k;
            all[j] = ld_cluster_u64(mapa_cluster(b0 + 8 * (j - from * k), from));
          }
          group_sync<GT>(0);
          for (int j = gt; j < C * k; j += GT) {
            const int from = j / k, at = j - from * k;
            const uint64_t c = all[j];
            if (c == 0) continue;
            int r = at;  // before it in its own list, and in every other one
            for (int o = 0; o < C && r < k; ++o) {
              if (o == from) continue;
              const uint64_t* other = all + o * k;
              int lo = 0, hi = k;
              while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (other[mid] > c) lo = mid + 1;
                else hi = mid;
              }
              r += lo;
            }
            if (r < k) put(r, c);
          }
          if (gt == 0 && p.lse && top != INFINITY) {
            const float r0 = top == -INFINITY ? 0.0f : top;
            float gs = 0.0f;
            for (int o = 0; o < C; ++o) {
              const uint64_t ms = ld_cluster_u64(mapa_cluster(s0, o));
              gs += __uint_as_float((uint32_t)(ms >> 32)) * expf((__uint_as_float((uint32_t)ms) - r0) * p.inv_t);
            }
            p.lse[row] = r0 * p.inv_t + logf(gs);
          }
          group_sync<GT>(0);
          if (gt < C) mbar_arrive_release_cluster(mapa_cluster(smem_u32(&xdone), gt));
        }
        mbar_wait_cluster(&xdone, turn & 1, &ring.abort_flag);  // `best` may be written again
      }
    }
  }
  if (ring_gave_up(ring, C, p.fault_word)) {
    for (int i = 0; i < n_mine; ++i) {
      const long long row = row0 + (long long)i * stride;
      for (int j = tid; j < k; j += blockDim.x) {
        p.values[row * k + j] = NAN;
        p.ids[row * k + j] = -1;  // an absent entry to whoever reads on
      }
      if (tid == 0 && p.lse) p.lse[row] = NAN;
    }
  }
}

// Rows in numbers, or rows that no cluster holds: nothing is staged.  A CTA reads its row once for the threads' maxima and
// the sum (a running maximum, brought up to date four vectors at a time), and notes the key of every vector's largest
// element, so that it knows where to look for the elements that reach the threshold; rows of more than TS_KEYS vectors
// are read again for that, out of the L2 cache for the most part.  Ten CTAs of 128 threads per SM (32 of
// one warp for short rows: 16384 x 1000 bf16 31 us, 54 with two) cover each other's latencies, where the staged form above has three rows at work on an SM; and a thread's
// work beside its elements, some 500 instructions, is shared by more of them than in larger CTAs (4096 x 32000 bf16, k 64:
// 92 us with 256 threads, 79 with 128).
constexpr int TS_FLIGHT = 4, TS_KEYS = 16384;

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 32 ? 32 : 1280 / THREADS)
top_stream_kernel(const TopParams p) {
  constexpr int V = VecOf<T>::N, WARPS = THREADS / 32;
  extern __shared__ __align__(16) uint64_t list[];
  __shared__ float s_max[WARPS], s_sum[WARPS];
  __shared__ uint32_t s_range[WARPS];
  __shared__ int s_count, s_hits, s_cnt[2][WARPS];
  __shared__ TopSelect s_sel;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int k = p.k, n = p.vocab, cap = top_list(k);
  int* hits = reinterpret_cast<int*>(list + cap);
  uint16_t* keys = reinterpret_cast<uint16_t*>(list + cap + cap / 2);
  const long long row = blockIdx.x;
  const RowSlice<T> s(reinterpret_cast<const T*>(p.logits) + row * p.ld, n, 0, 0);
  const float scale = 1.4426950408889634f * p.inv_t;
  const bool keyed = p.keyed;
  uint32_t m[TS_FLIGHT];  // keys of the shares' maxima, upper 16 bits; 0: no share
  float ref = -INFINITY, sum = 0.0f;  // the running maximum without NaN, the sum
#pragma unroll
  for (int q = 0; q < TS_FLIGHT; ++q) m[q] = 0;
#pragma unroll 1
  for (int v0 = tid; v0 < s.hi; v0 += TS_FLIGHT * THREADS) {
    uint4 raw[TS_FLIGHT];
    load_vectors<T>(s, v0, THREADS, raw);
    float bm = ref;
#pragma unroll
    for (int q = 0; q < TS_FLIGHT; ++q) {
      const int v = v0 + q * THREADS;
      const uint32_t key = vec_key<T>(raw[q], bm);
      if (v < s.hi) {
        m[q] = max(m[q], key);
        if (keyed) keys[v] = (uint16_t)key;
      }
    }
    if (p.lse) {
      const float r0 = bm == -INFINITY ? 0.0f : bm;
      if (bm > ref) {
        sum *= ref == -INFINITY ? 0.0f : expf((ref - r0) * p.inv_t);
        ref = bm;
      }
      const float off = -r0 * scale;
      const bool far = sizeof(T) == 4 || fabsf(r0) * p.inv_t > 1e4f;
      float acc[2] = {0.0f, 0.0f};
#pragma unroll
      for (int q = 0; q < TS_FLIGHT; ++q) {
        float x[V];
        unpack_vec<T>(raw[q], x);
        if (far) {
#pragma unroll
          for (int c = 0; c < V; ++c) acc[c & 1] += expf((x[c] - r0) * p.inv_t);
        } else {
#pragma unroll
          for (int c = 0; c < V; c += 2) {
            float h0, h1;
            ffma2(h0, h1, x[c], x[c + 1], scale, scale, off, off);
            fadd2(acc[0], acc[1], acc[0], acc[1], exp2_approx(h0), exp2_approx(h1));
          }
        }
      }
      sum += acc[0] + acc[1];
    } else {
      ref = bm;
    }
  }
  // ---- threshold, as above
  const uint32_t top_key = max(max(m[0], m[1]), max(m[2], m[3]));
  const float wm = warp_max(ref);
  const uint32_t k_hi = __reduce_max_sync(0xffffffffu, top_key);
  const bool by_thread = (THREADS == 32 ? 2 : 4) * k <= min(s.hi, THREADS);  // the threshold goes by the threads' maxima, else by the shares'
  uint32_t least = 0xffffu;
#pragma unroll
  for (int q = 0; q < TS_FLIGHT; ++q)
    if (m[q]) least = min(least, m[q]);
  const uint32_t k_lo = __reduce_min_sync(0xffffffffu, by_thread && top_key ? top_key : least);
  if (lane == 0) { s_max[warp] = wm; s_range[warp] = (k_hi << 16) | k_lo; }
  if (tid == 0) { s_count = 0; s_hits = 0; }
  __syncthreads();
  const float top = lanes_max<WARPS>(s_max[lane % WARPS]), base = top == -INFINITY ? 0.0f : top;
  sum = warp_sum(sum * (ref == -INFINITY ? 1.0f : expf((ref - base) * p.inv_t)));
  if (lane == 0) s_sum[warp] = sum;
  uint32_t hi16 = 0, lo16 = 0xffffu;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    hi16 = max(hi16, s_range[w] >> 16);
    lo16 = min(lo16, s_range[w] & 0xffffu);
  }
  const int bits = 32 - __clz(hi16 ^ lo16);
  uint32_t tau = 0;
  if (by_thread) {
    tau = (hi16 >> bits) << bits;
#pragma unroll 1
    for (int bit = bits - 1; bit >= 0; --bit) {
      const uint32_t trial = tau | (1u << bit);
      if (__syncthreads_count(top_key >= trial) >= k) tau = trial;
    }
  } else if (k <= min(s.hi, TS_FLIGHT * THREADS)) {
    tau = (hi16 >> bits) << bits;
#pragma unroll 1
    for (int bit = bits - 1; bit >= 0; --bit) {
      const uint32_t trial = tau | (1u << bit);  // not 0: places without a share do not count
      int c = 0;
#pragma unroll
      for (int q = 0; q < TS_FLIGHT; ++q) c += m[q] >= trial;
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) s_cnt[bit & 1][warp] = c;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) total += s_cnt[bit & 1][w];
      if (total >= k) tau = trial;
    }
  }
  __syncthreads();  // s_sum, the counters
  if (tid == 0 && p.lse && top != INFINITY) {
    float all = 0.0f;
    for (int w = 0; w < WARPS; ++w) all += s_sum[w];
    p.lse[row] = base * p.inv_t + logf(all);
  }
  // ---- the vectors that hold an element at or above it
  const float floor_value = key_value(tau << 16);
#pragma unroll 1
  for (int v0 = tid; v0 - tid < s.hi; v0 += 8 * TS_FLIGHT * THREADS) {
    uint32_t noted = 0;
    if (keyed) {
#pragma unroll 4
      for (int b = 0; b < 8 * TS_FLIGHT; ++b) {
        const int v = v0 + b * THREADS;
        if (v < s.hi) noted |= (uint32_t)(keys[v] >= tau) << b;  // this thread's own notes
      }
    } else {
#pragma unroll 1
      for (int b = 0; b < 8; ++b) {
        uint4 raw[TS_FLIGHT];
        const int v = v0 + b * TS_FLIGHT * THREADS;
        if (v >= s.hi) break;
        load_vectors<T>(s, v, THREADS, raw);
#pragma unroll
        for (int q = 0; q < TS_FLIGHT; ++q) noted |= (uint32_t)(v + q * THREADS < s.hi && reaches<T>(raw[q], floor_value)) << (b * TS_FLIGHT + q);
      }
    }
    int mine = __popc(noted), before = mine;
    if (__any_sync(0xffffffffu, mine)) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      int at = 0;
      if (lane == 31) at = atomicAdd(&s_hits, before);
      at = __shfl_sync(0xffffffffu, at, 31) + before - mine;
      for (; noted; noted &= noted - 1, ++at)
        if (at < cap) hits[at] = v0 + (__ffs(noted) - 1) * THREADS;
    }
  }
  __syncthreads();
  const int noted = s_hits;
  if (noted <= cap) {
    for (int j = tid; j < noted; j += THREADS) {
      uint4 raw[1];
      float x[V];
      const int v = hits[j], e = s.first(v);
      load_vectors<T>(s, v, 0, raw);
      unpack_vec<T>(raw[0], x);
      uint32_t in = 0;
#pragma unroll
      for (int c = 0; c < V; ++c) in |= (uint32_t)(!(x[c] < floor_value) && e + c >= 0 && e + c < n) << c;
      int at = atomicAdd(&s_count, __popc(in));
#pragma unroll
      for (int c = 0; c < V; ++c)
        if ((in >> c) & 1) {
          if (at < cap) list[at] = ((uint64_t)order_key(x[c]) << 32) | (uint32_t)~(e + c);
          ++at;
        }
    }
  }
  __syncthreads();
  int listed = noted <= cap ? s_count : cap + 1;
  if (listed > cap) {
    auto each = [&](auto f) {
#pragma unroll 1
      for (int v = tid; v < s.hi; v += THREADS) {
        uint4 raw[1];
        float x[V];
        load_vectors<T>(s, v, 0, raw);
        unpack_vec<T>(raw[0], x);
        const int e = s.first(v);
#pragma unroll
        for (int c = 0; c < V; ++c)
          if (e + c >= 0 && e + c < n) f(e + c, x[c]);
      }
    };
    uint32_t value, last;
    exact_threshold<THREADS>(s_sel, tid, k, n, value, last, each, []() { __syncthreads(); });
    if (tid == 0) s_count = 0;
    __syncthreads();
    each([&](int e, float x) {
      const uint32_t q = order_key(x);
      if (q > value || (q == value && (uint32_t)e <= last)) {
        const int at = atomicAdd(&s_count, 1);
        if (at < cap) list[at] = ((uint64_t)q << 32) | (uint32_t)~e;
      }
    });
    __syncthreads();
    listed = min(s_count, cap);
  }
  each_rank<THREADS>(list, listed, k, tid, []() { __syncthreads(); }, [&](int r, uint64_t c) {
    if (r >= k) return;
    const float v = key_value((uint32_t)(c >> 32));
    p.values[row * k + r] = v;
    p.ids[row * k + r] = (int)~(uint32_t)c;
    if (r == 0 && p.lse && top == INFINITY) p.lse[row] = v;  // inf or NaN, where the sum ran into inf - inf
  });
}

template <typename T>
int top_launch(TopParams& p, cudaStream_t s) {
  const long long bytes = (long long)p.vocab * sizeof(T);
  const int lists = 8 * (top_list(p.k) * 3 / 2);
  // few rows: all of a CTA's threads, and up to eight CTAs, for each of them
  if (p.rows <= 2LL * sm_count()) {
    p.shape = row_shape(p.rows, p.vocab, sizeof(T), lists + 9 * 8 * TOP_MAX_K, 3, 8192);
    if (p.shape.stages) return launch_pipe<top_pipe_kernel<T, 512>>("top_logits", p.shape, p.rows, 512 + 32, s, p);
  }
  const long long vectors = bytes / 16 + 2;  // a row that starts inside a vector touches one more
  p.keyed = vectors <= TS_KEYS;
  const int smem = lists + (p.keyed ? (int)vectors * 2 : 0);
  // a warp's four shares per lane are too few for a threshold near the k-th largest where k is more than half of them
  if (bytes <= 8192 && p.k <= 64) top_stream_kernel<T, 32><<<(unsigned)p.rows, 32, smem, s>>>(p);
  else top_stream_kernel<T, 128><<<(unsigned)p.rows, 128, smem, s>>>(p);
  return check_launch("top_logits");
}

}  // namespace
}  // namespace eisen

extern "C" int eisen_top_logits(void* stream, const void* logits, long long ld, float* values, int* ids, float* lse, long long rows,
                                long long vocab, long long k, float temperature, int dtype) {
  using namespace eisen;
  if (rows < 0 || rows > 0x7fffffffLL || vocab <= 0 || vocab > 0x7fffff00LL)
    return fail(EISEN_ERR_LIMIT, "top_logits: rows must be in [0, 2^31), vocab in [1, 2^31 - 256]");
  if (dtype != DT_F32 && dtype != DT_BF16) return fail(EISEN_ERR_INVALID, "top_logits: logits must be f32 or bf16");
  if (k < 1 || k > TOP_MAX_K || k > vocab) return fail(EISEN_ERR_LIMIT, "top_logits: k must be in [1, min(vocab, 256)]");
  if (ld < vocab) return fail(EISEN_ERR_INVALID, "top_logits: the row stride is shorter than a row");
  if (!(temperature > 0.0f) || !(temperature <= FLT_MAX) || !(1.0f / temperature <= FLT_MAX))
    return fail(EISEN_ERR_INVALID, "top_logits: the temperature must be positive and finite");
  if (rows == 0) return 0;
  if (!logits || !values || !ids) return fail(EISEN_ERR_INVALID, "top_logits: logits, values and ids must not be null");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DT_F32 ? 4 : 2)) return fail(EISEN_ERR_INVALID, "top_logits: unaligned pointer");
  TopParams p = {logits, ld, values, ids, lse, rows, (int)vocab, (int)k, 1.0f / temperature, fault_word(), 0, {}};
  EISEN_DISPATCH_DTYPE(dtype, T, { return top_launch<T>(p, (cudaStream_t)stream); });
}
