// A teacher's top logits and the loss of a student against them.
//
//   eisen_top_logits     the k largest entries of every row in descending order (equal values: the lowest index
//                        first), and the row's log-sum-exp at a temperature
//   eisen_distill_*      kd T^2 sum_j q_j (ln q_j - ln p_j) - ce ln(softmax(x)_y + 1e-8) with p = softmax(x / T) and q
//                        the teacher's distribution over the entries it gives; gradient
//                        kd T (Q p_i - sum_{id_j = i} q_j) + ce (softmax(x)_i - [i = y]),  Q = sum_j q_j
//
// All of them read a row of `vocab` logits once or twice and are bound by that traffic.  Maxima, sums and
// probabilities are f32; only dlogits of bf16 logits is rounded, once.
#include <algorithm>
#include <cfloat>
#include <cstdio>

#include "common.cuh"
#include "errors.h"
#include "row_slice.cuh"
#include "../../include/eisen_b200.h"

namespace eisen {
namespace {

constexpr int TOP_THREADS = 512;
constexpr int TOP_MAX_K = 256;
constexpr int DS_THREADS = 512;
constexpr int DS_MAX_K = 1024;

template <typename T>
__device__ __forceinline__ float exp_row(float x) {
  if constexpr (sizeof(T) == 2) return __expf(x);
  else return expf(x);
}

// f(index, value) for every element of a row that may start at any element boundary: 16-byte reads between a
// scalar head and a scalar tail
template <typename T, typename F>
__device__ __forceinline__ void for_row(const T* __restrict__ xr, int n, int tid, int threads, F f) {
  constexpr int V = VecOf<T>::N;
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) & 15) / sizeof(T)));
  if (tid < head) f(tid, to_f32(xr[tid]));
  const int nvec = (n - head) / V;
  for (int i = tid; i < nvec; i += threads) {
    float v[V];
    ld16(xr + head + i * V, v);
#pragma unroll
    for (int e = 0; e < V; ++e) f(head + i * V + e, v[e]);
  }
  const int at = head + nvec * V + tid;
  if (at < n) f(at, to_f32(xr[at]));
}

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

// running maximum and sum of exp((x - m) * inv_t)
struct OnlineSum {
  float m = -INFINITY, s = 0.0f;
  template <typename T>
  __device__ __forceinline__ void add(float x, float inv_t) {
    if (x > m) {
      s *= m == -INFINITY ? 0.0f : exp_row<T>((m - x) * inv_t);
      m = x;
    }
    s += exp_row<T>((x - (m == -INFINITY ? 0.0f : m)) * inv_t);
  }
};

// The digit (of 256) of the threshold: the highest bin at which the count from the top reaches `want`.
// Returns the count above that bin and leaves the bin in sh[0].
__device__ __forceinline__ void pick_bin(const int* hist, int want, int* out) {
  // one warp: lane l owns bins 255 - 8 l ... 255 - 8 l - 7
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

template <typename T>
__global__ void __launch_bounds__(TOP_THREADS)
top_logits_kernel(const T* __restrict__ logits, long long ld, float* __restrict__ values, int* __restrict__ ids,
                  float* __restrict__ lse, int vocab, int k, float inv_t) {
  __shared__ int hist[256];
  __shared__ int pick[3];
  __shared__ int count;
  __shared__ float sh[32];
  __shared__ uint64_t cand[TOP_MAX_K];
  const long long row = blockIdx.x;
  const T* xr = logits + row * ld;
  const int tid = threadIdx.x;
  // threshold by digits of eight bits, first of the value, then (where the last bin holds more than are
  // wanted) of the index from the low end
  uint32_t prefix = 0, mask = 0;
  int want = k, in_bin = vocab;
  OnlineSum os;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const bool first = shift == 24;
    for_row(xr, vocab, tid, TOP_THREADS, [&](int, float x) {
      if (first && lse) os.add<T>(x, inv_t);
      const uint32_t key = order_key(x);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
    });
    __syncthreads();
    if (tid < 32) pick_bin(hist, want, pick);
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    mask |= 255u << shift;
    want -= pick[1];
    in_bin = pick[2];
    __syncthreads();
  }
  if (lse) {
    const float gm = block_max(os.m, sh);
    const float ref = gm == -INFINITY ? 0.0f : gm;
    const float s = block_sum(os.s * (os.m == -INFINITY && os.s == 0.0f ? 0.0f : exp_row<T>((os.m == -INFINITY ? 0.0f : os.m - ref) * inv_t)), sh);
    if (tid == 0) lse[row] = ref * inv_t + logf(s);
    __syncthreads();
  }
  uint32_t last = 0xffffffffu;  // highest index taken among the entries equal to the threshold
  if (in_bin > want) {
    uint32_t ip = 0, im = 0;  // on the complement of the index: the largest complements are the lowest indices
    int iw = want;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for_row(xr, vocab, tid, TOP_THREADS, [&](int i, float x) {
        const uint32_t c = ~(uint32_t)i;
        if (order_key(x) == prefix && (c & im) == ip) atomicAdd(&hist[(c >> shift) & 255], 1);
      });
      __syncthreads();
      if (tid < 32) pick_bin(hist, iw, pick);
      __syncthreads();
      ip |= (uint32_t)pick[0] << shift;
      im |= 255u << shift;
      iw -= pick[1];
      __syncthreads();
    }
    last = ~ip;
  }
  if (tid == 0) count = 0;
  __syncthreads();
  for_row(xr, vocab, tid, TOP_THREADS, [&](int i, float x) {
    const uint32_t key = order_key(x);
    if (key > prefix || (key == prefix && (uint32_t)i <= last)) {
      const int at = atomicAdd(&count, 1);
      if (at < TOP_MAX_K) cand[at] = ((uint64_t)key << 32) | (uint32_t)~i;
    }
  });
  __syncthreads();
  // rank by counting: the composites are distinct, so the result does not depend on the order of arrival
  if (tid < k) {
    const uint64_t c = cand[tid];
    int r = 0;
    for (int j = 0; j < k; ++j) r += cand[j] > c;
    const float v = key_value((uint32_t)(c >> 32));
    if (r == 0 && lse && v == INFINITY) lse[row] = v;  // where the sum ran into inf - inf
    values[row * k + r] = v;
    ids[row * k + r] = (int)~(uint32_t)c;
  }
}

struct DistillParams {
  const void* logits;
  long long ld;
  const int* t_ids;
  const float* t_logits;
  const float* t_lse;
  const int* targets;
  void* dlogits;
  long long ldd;
  float* row_loss;
  float* lse;             // [2][rows]: at the temperature, at 1
  const float* grad_out;
  long long rows;
  int vocab, k, ignore_index;
  float temperature, inv_t, kd_weight, ce_weight, grad_scale;
  int accumulate;
  int* bad_id_flag;
  int sum_kind, grad_kind, cluster;  // distill_row_kernel: see RowExp
};

constexpr int DS_FWD = 1, DS_BWD = 2;

// The entries of one row that need more than p_i: the teacher's ids and the target (entry k).
struct RowEntries {
  int id[DS_MAX_K + 1];    // -1: absent
  float q[DS_MAX_K + 1];
  float x[DS_MAX_K + 1];   // the student's logits there
  float old[DS_MAX_K + 1]; // accumulate: what dlogits holds there
};

template <typename T, int MODE>
__global__ void __launch_bounds__(DS_THREADS)
distill_kernel(const DistillParams p) {
  __shared__ RowEntries en;
  __shared__ float sh[32];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, V_ = p.vocab, k = p.k;
  const T* xr = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  T* dr = (MODE & DS_BWD) ? reinterpret_cast<T*>(p.dlogits) + row * p.ldd : nullptr;
  const int y = p.targets ? p.targets[row] : -1;
  const bool ignored = p.targets && y == p.ignore_index;
  const bool out = p.targets && !ignored && (y < 0 || y >= V_);
  if (ignored || out) {
    if constexpr (MODE & DS_FWD) {
      if (tid == 0) {
        p.row_loss[row] = 0.0f;
        if (p.lse) { p.lse[row] = 0.0f; p.lse[p.rows + row] = 0.0f; }
        if (out && p.bad_id_flag) *p.bad_id_flag = 1;
      }
    }
    if constexpr (MODE & DS_BWD) {
      if (!p.accumulate)
        for (int i = tid; i < V_; i += DS_THREADS) dr[i] = from_f32<T>(0.0f);
    }
    return;
  }
  // ---- the teacher's distribution
  const float inv_t = p.inv_t;
  float tm = -INFINITY;
  for (int j = tid; j <= k; j += DS_THREADS) {
    int id = j < k ? p.t_ids[row * k + j] : y;
    if (j < k && id >= V_) {
      if ((MODE & DS_FWD) && p.bad_id_flag) *p.bad_id_flag = 1;
      id = -1;
    }
    id = id < 0 ? -1 : id;
    float t = -INFINITY;
    if (j < k && id >= 0) t = p.t_logits[row * k + j] * inv_t;
    en.id[j] = id;
    en.q[j] = t;
    en.x[j] = id >= 0 ? to_f32(xr[id]) : 0.0f;
    if ((MODE & DS_BWD) && p.accumulate) en.old[j] = id >= 0 ? to_f32(dr[id]) : 0.0f;
    tm = t != t ? t : fmaxf(tm, t);
  }
  float tl;
  if (p.t_lse) {
    tl = p.t_lse[row];
    __syncthreads();
  } else {
    tm = block_max(tm, sh);
    const float ref = tm == -INFINITY ? 0.0f : tm;
    float s = 0.0f;
    for (int j = tid; j < k; j += DS_THREADS) s += expf(en.q[j] - ref);
    s = block_sum(s, sh);
    tl = s > 0.0f || s != s ? ref + logf(s) : 0.0f;  // no entry: every q is 0
  }
  float Q = 0.0f;
  for (int j = tid; j <= k; j += DS_THREADS) Q += (en.q[j] = expf(en.q[j] - tl));
  Q = block_sum(Q, sh);

  const bool two = p.ce_weight != 0.0f && p.temperature != 1.0f;
  float lt, l1;
  if constexpr (MODE & DS_FWD) {
    OnlineSum os, o1;
    for_row(xr, V_, tid, DS_THREADS, [&](int, float x) {
      os.add<T>(x, inv_t);
      if (two || p.lse) o1.add<T>(x, 1.0f);
    });
    const float gm = block_max(os.m, sh), ref = gm == -INFINITY ? 0.0f : gm;
    const float mine = os.m == -INFINITY ? 0.0f : os.m - ref;
    const float st = block_sum(os.s * exp_row<T>(mine * inv_t), sh);
    const float s1 = block_sum(o1.s * exp_row<T>(mine), sh);
    lt = ref * inv_t + logf(st);
    l1 = ref + logf(two || p.lse ? s1 : st);
    float kl = 0.0f;
    for (int j = tid; j < k; j += DS_THREADS) {
      const float q = en.q[j];
      if (q > 0.0f || q != q) kl += q * (p.t_logits[row * k + j] * inv_t - tl - (en.x[j] * inv_t - lt));
    }
    kl = block_sum(kl, sh);
    if (tid == 0) {
      float l = 0.0f;
      if (p.kd_weight != 0.0f) l = p.kd_weight * p.temperature * p.temperature * kl;
      if (p.ce_weight != 0.0f) l -= p.ce_weight * logf(expf(en.x[k] - l1) + 1e-8f);
      p.row_loss[row] = l;
      if (p.lse) { p.lse[row] = lt; p.lse[p.rows + row] = l1; }
    }
  } else {
    lt = p.lse[row];
    l1 = p.lse[p.rows + row];
  }
  if constexpr (MODE & DS_BWD) {
    const float g = p.grad_scale * (p.grad_out ? *p.grad_out : 1.0f);
    const float kq = p.kd_weight * p.temperature * g, kp = kq * Q, c1 = p.ce_weight * g;
    auto grad = [&](float x) {
      float d = kp * exp_row<T>(x * inv_t - lt);
      if (p.ce_weight != 0.0f) d += c1 * exp_row<T>(x - l1);
      return d;
    };
    for (int i = tid; i < V_; i += DS_THREADS) {
      float d = grad(to_f32(xr[i]));
      if (p.accumulate) d += to_f32(dr[i]);
      dr[i] = from_f32<T>(d);
    }
    __syncthreads();
    // entries with a term of their own: the first of equal ids collects them all and writes last
    for (int j = tid; j <= k; j += DS_THREADS) {
      const int id = en.id[j];
      if (id < 0) continue;
      float q = 0.0f;
      bool first = true;
      for (int i = 0; i <= k; ++i) {
        if (en.id[i] == id) {
          if (i < j) first = false;
          if (i < k) q += en.q[i];
        }
      }
      if (!first) continue;
      float d = grad(en.x[j]) - kq * q;
      if (id == y && p.ce_weight != 0.0f) d -= c1;
      if (p.accumulate) d += en.old[j];
      dr[id] = from_f32<T>(d);
    }
  }
}

// A row's exponentials exp((x - ref) / T) and exp(x - ref).  KIND says how they are formed:
//   ONE   the first alone (temperature 1, or no cross-entropy term)
//   TWO   both, each by itself
//   PLAIN the f32 form, (x - ref) first and expf: rows of f32 logits, and rows whose largest entry is near the end of
//         the type's range (all of it masked by the lowest value), where the products with ref would overflow
//   10 a + b   bf16 rows whose temperature is b / a: h = exp((x - ref) / b), the exponentials are h^a and h^b.  The
//         special-function unit gives 16 results per clock and SM: two exponentials in both passes over a row are 8000
//         clocks per 32000 entries where the memory needs 5600, one is 4000.  A power multiplies the relative error of
//         h (2^-22) by at most 7, far below the 2^-8 of the bf16 result.
constexpr int ONE = 0, TWO = 1, PLAIN = 2;

template <typename T, int KIND>
struct RowExp {
  float ref, inv_t, c, off, off1;
  bool two;
  __device__ __forceinline__ RowExp(float r, float it, bool both) : ref(r), inv_t(it), two(both) {
    c = 1.4426950408889634f * (KIND < 10 ? it : 1.0f / (float)(KIND % 10));
    off = -r * c;
    off1 = -r * 1.4426950408889634f;
  }
  // the exponentials of two elements, in packed arithmetic: et = exp((x - ref) / T), e1 = exp(x - ref)
  __device__ __forceinline__ void operator()(float x, float y, float (&et)[2], float (&e1)[2]) const {
    if constexpr (KIND == PLAIN) {
      et[0] = expf((x - ref) * inv_t);
      et[1] = expf((y - ref) * inv_t);
      e1[0] = two ? expf(x - ref) : 0.0f;
      e1[1] = two ? expf(y - ref) : 0.0f;
    } else {
      float h0, h1;
      ffma2(h0, h1, x, y, c, c, off, off);
      h0 = exp2_approx(h0);
      h1 = exp2_approx(h1);
      if constexpr (KIND == ONE) {
        et[0] = h0; et[1] = h1;
        e1[0] = e1[1] = 0.0f;
      } else if constexpr (KIND == TWO) {
        et[0] = h0; et[1] = h1;
        ffma2(h0, h1, x, y, 1.4426950408889634f, 1.4426950408889634f, off1, off1);
        e1[0] = exp2_approx(h0);
        e1[1] = exp2_approx(h1);
      } else {
        constexpr int A = KIND / 10, B = KIND % 10;
        float s0, s1, f0, f1;  // h^2, h^4
        fmul2(s0, s1, h0, h1, h0, h1);
        if constexpr (B >= 4) fmul2(f0, f1, s0, s1, s0, s1);
        et[0] = A == 1 ? h0 : s0;
        et[1] = A == 1 ? h1 : s1;
        if constexpr (B == 1) { e1[0] = h0; e1[1] = h1; }
        else if constexpr (B == 2) { e1[0] = s0; e1[1] = s1; }
        else if constexpr (B == 3) fmul2(e1[0], e1[1], s0, s1, h0, h1);
        else if constexpr (B == 4) { e1[0] = f0; e1[1] = f1; }
        else if constexpr (B == 5) fmul2(e1[0], e1[1], f0, f1, h0, h1);
        else {
          fmul2(f0, f1, f0, f1, s0, s1);
          fmul2(e1[0], e1[1], f0, f1, h0, h1);
        }
      }
    }
  }
};

// f(RowExp) for the kind that the row takes: one branch per pass, the same for the whole CTA
template <typename T, typename F>
__device__ __forceinline__ void with_exp(int kind, float ref, float inv_t, F f) {
  if constexpr (sizeof(T) == 4) {
    f(RowExp<T, PLAIN>(ref, inv_t, kind != ONE));
  } else {
    if (fabsf(ref) > 1e30f) return f(RowExp<T, PLAIN>(ref, inv_t, kind != ONE));
    switch (kind) {
      case ONE: return f(RowExp<T, ONE>(ref, inv_t, false));
      case TWO: return f(RowExp<T, TWO>(ref, inv_t, true));
      case 12: return f(RowExp<T, 12>(ref, inv_t, true));
      case 13: return f(RowExp<T, 13>(ref, inv_t, true));
      case 14: return f(RowExp<T, 14>(ref, inv_t, true));
      case 21: return f(RowExp<T, 21>(ref, inv_t, true));
      case 23: return f(RowExp<T, 23>(ref, inv_t, true));
      case 25: return f(RowExp<T, 25>(ref, inv_t, true));
      default: return f(RowExp<T, 27>(ref, inv_t, true));
    }
  }
}

// the kind for both exponentials at a temperature
int exp_kind(float temperature, int dtype) {
  if (dtype == DT_BF16)
    for (int a = 1; a <= 2; ++a)
      for (int b = 1; b <= (a == 1 ? 4 : 7); ++b)
        if ((a == 1 || b % 2) && temperature * (float)a == (float)b && temperature != 1.0f) return 10 * a + b;
  return TWO;
}

// the elements of a vector that reaches beyond an end of its row, or whose place in dlogits is not aligned
template <typename T>
__device__ __noinline__ void store_edge(T* dr, int e, int n, const float (&d)[VecOf<T>::N], bool accumulate) {
#pragma unroll
  for (int i = 0; i < VecOf<T>::N; ++i)
    if (e + i >= 0 && e + i < n) dr[e + i] = from_f32<T>(accumulate ? d[i] + to_f32(dr[e + i]) : d[i]);
}

// A row in the registers of one CTA, or of a cluster of p.cluster CTAs with a slice of the vectors each: the
// logits are read once, by loads that are all in flight together, and two CTAs per SM (more of shorter rows) work
// while the other one's loads are on their way.  The gradient pass takes the exponentials again from the registers.
// The teacher's entries go through shared memory beside the row's own maximum and sums; entries with a term of
// their own are written after the dense pass, by the first thread among equal ids.  Few threads with many vectors
// each: what a thread does beside its elements (addresses, three reductions, the row's scalars) is several hundred
// instructions, as many as 60 elements take.
constexpr int row_ctas(int threads, int nv) { return nv >= 16 ? 512 / threads : 1024 / threads; }
template <typename T, int THREADS, int NV, int MODE>
__global__ void __launch_bounds__(THREADS, row_ctas(THREADS, NV))
distill_row_kernel(const DistillParams p) {
  constexpr int V = VecOf<T>::N, WARPS = THREADS / 32;
  constexpr int PAD = DS_MAX_K + 4;
  constexpr bool FWD = (MODE & DS_FWD) != 0, BWD = (MODE & DS_BWD) != 0, ACC = BWD && !FWD;
  __shared__ __align__(16) int s_id[PAD];  // the teacher's ids, -1: absent; entry k: the target
  __shared__ float s_t[PAD];               // its logits / T
  __shared__ float s_x[PAD];               // the student's logits there
  __shared__ float s_old[ACC ? PAD : 1];   // what dlogits held there
  __shared__ float s_max[2][WARPS], s_sum[4][WARPS];
  __shared__ float s_xch[8][3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = p.cluster, k = p.k, n = p.vocab;
  const int rank = C > 1 ? (int)cluster_ctarank() : 0;
  const long long row = C > 1 ? blockIdx.x / C : blockIdx.x;
  if (FWD && C > 1) cluster_arrive();  // matched before the first access to a peer's shared memory
  const T* xr = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  T* dr = BWD ? reinterpret_cast<T*>(p.dlogits) + row * p.ldd : nullptr;
  const int y = p.targets ? p.targets[row] : -1;
  // requested in front of the row, whose loads take their place behind them
  const bool entries = BWD || rank == 0;
  int id0 = -1;
  float t0 = 0.0f;
  if (entries && tid < k) {
    id0 = p.t_ids[row * k + tid];
    t0 = p.t_logits[row * k + tid];
  }
  const RowView<T> view(xr, n);
  const int nvec = view.vectors(), per = (nvec + C - 1) / C;
  const int lo = min(rank * per, nvec), hi = min(lo + per, nvec);
  uint4 raw[NV];
  load_slice<T, THREADS, NV>(view, lo, hi, raw);
  const bool aligned = BWD && ((reinterpret_cast<uintptr_t>(dr) ^ reinterpret_cast<uintptr_t>(xr)) & 15) == 0;
  const bool ignored = p.targets && y == p.ignore_index;
  const bool out = p.targets && !ignored && (y < 0 || y >= n);
  if (ignored || out) {
    if (FWD && tid == 0 && rank == 0) {
      p.row_loss[row] = 0.0f;
      if (p.lse) { p.lse[row] = 0.0f; p.lse[p.rows + row] = 0.0f; }
      if (out && p.bad_id_flag) *p.bad_id_flag = 1;
    }
    if (BWD && !p.accumulate) {
      for (int v = lo + tid; v < hi; v += THREADS) {
        const int e = view.first(v);
        if (aligned && e >= 0 && e + V <= n) *reinterpret_cast<uint4*>(dr + e) = make_uint4(0, 0, 0, 0);
        else
          for (int i = max(e, 0); i < min(e + V, n); ++i) dr[i] = from_f32<T>(0.0f);
      }
    }
    if (FWD && C > 1) cluster_wait();
    return;
  }
  float tm = -INFINITY;
  if (entries) {
    for (int j = tid; j < ((k + 4) & ~3); j += THREADS) {
      int id = j == k ? y : -1;
      float t = -INFINITY;
      if (j < k) {
        id = j < THREADS ? id0 : p.t_ids[row * k + j];
        if (id >= n) {
          if (FWD && p.bad_id_flag) *p.bad_id_flag = 1;
          id = -1;
        }
        if (id >= 0) t = (j < THREADS ? t0 : p.t_logits[row * k + j]) * p.inv_t;
      }
      id = max(id, -1);
      s_id[j] = id;
      s_t[j] = t;
      s_x[j] = id >= 0 ? to_f32(xr[id]) : 0.0f;
      if (ACC && p.accumulate) s_old[j] = id >= 0 ? to_f32(dr[id]) : 0.0f;
      tm = fmaxf(tm, t);
    }
  }
  // the row's maximum and the teacher's
  float ref = 0.0f;
  if constexpr (FWD) {
    const float m = warp_max(max_of<T, NV>(raw));
    if (lane == 0) s_max[0][warp] = m;
  }
  tm = warp_max(tm);
  if (lane == 0) s_max[1][warp] = tm;
  __syncthreads();
  if constexpr (FWD) {
    ref = warp_max(s_max[0][lane % WARPS]);
    if (ref == -INFINITY) ref = 0.0f;
  }
  // the teacher's sum: of exp(t - tref) = q_j S, where tref is its given log-sum-exp (S = 1) or its maximum
  float tref;
  if (p.t_lse) {
    tref = p.t_lse[row];
  } else {
    tref = warp_max(s_max[1][lane % WARPS]);
    if (tref == -INFINITY) tref = 0.0f;
  }
  float S = 0.0f;
  if (entries)
    for (int j = tid; j < k; j += THREADS) S += expf(s_t[j] - tref);
  float st = 0.0f, s1 = 0.0f;
  if constexpr (FWD) {
    float sa[2] = {0.0f, 0.0f}, sb[2] = {0.0f, 0.0f};
    with_exp<T>(p.sum_kind, ref, p.inv_t, [&](const auto& ex) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float x[V];
        unpack_vec<T>(raw[j], x);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          float et[2], e1[2];
          ex(x[i], x[i + 1], et, e1);
          fadd2(sa[0], sa[1], sa[0], sa[1], et[0], et[1]);
          if (ex.two) fadd2(sb[0], sb[1], sb[0], sb[1], e1[0], e1[1]);
        }
      }
    });
    st = warp_sum(sa[0] + sa[1]);
    s1 = warp_sum(sb[0] + sb[1]);
    if (lane == 0) { s_sum[0][warp] = st; s_sum[1][warp] = s1; }
  }
  S = warp_sum(S);
  if (lane == 0) s_sum[2][warp] = S;
  __syncthreads();
  auto total = [&](int which) { return warp_sum(lane < WARPS ? s_sum[which][lane] : 0.0f); };
  S = total(2);
  // q_j = exp(t_j - tref) * inv_s,  Q = sum of them
  const float inv_s = p.t_lse || S == 0.0f ? 1.0f : __fdividef(1.0f, S), Q = S * inv_s;
  const bool has_kd = p.kd_weight != 0.0f, has_ce = p.ce_weight != 0.0f;
  if constexpr (FWD) {
    st = total(0);
    s1 = total(1);
    if (C > 1) {
      cluster_wait();
      if (tid < C) {
        const uint32_t to = mapa_cluster(smem_u32(&s_xch[rank][0]), tid);
        st_cluster_f32(to, st == 0.0f ? -INFINITY : ref);  // a slice without a finite entry has no say in the maximum
        st_cluster_f32(to + 4, st);
        st_cluster_f32(to + 8, s1);
      }
      cluster_arrive();
      cluster_wait();
      float gm = -INFINITY;
      for (int r = 0; r < C; ++r) gm = fmaxf(gm, s_xch[r][0]);
      ref = gm == -INFINITY ? 0.0f : gm;
      st = s1 = 0.0f;
      for (int r = 0; r < C; ++r) {
        const float d = s_xch[r][0] - ref;
        st += s_xch[r][1] * expf(d * p.inv_t);
        s1 += s_xch[r][2] * expf(d);
      }
    }
    if (warp == 0 && rank == 0) {
      const float lt = ref * p.inv_t + logf(st);
      const float l1 = p.sum_kind == ONE ? (p.temperature == 1.0f ? lt : 0.0f) : ref + logf(s1);
      const float tl = p.t_lse || S == 0.0f ? tref : tref + logf(S);  // ln q_j = t_j - tl
      float kl = 0.0f;
      for (int j = lane; j < k; j += 32) {
        const float t = s_t[j], q = expf(t - tl);
        if (q > 0.0f || q != q) kl += q * (t - tl - (s_x[j] * p.inv_t - lt));
      }
      kl = warp_sum(kl);
      if (lane == 0) {
        float l = 0.0f;
        if (has_kd) l = p.kd_weight * p.temperature * p.temperature * kl;
        if (has_ce) l -= p.ce_weight * logf(expf(s_x[k] - l1) + 1e-8f);
        p.row_loss[row] = l;
        if (p.lse) { p.lse[row] = lt; p.lse[p.rows + row] = l1; }
      }
    }
  } else {
    ref = p.lse[p.rows + row];
  }
  if constexpr (BWD) {
    // d = kt exp((x - ref) / T) + k1 exp(x - ref): kt, k1 turn the exponentials into weighted probabilities
    const float g = p.grad_scale * (p.grad_out ? *p.grad_out : 1.0f);
    const float kq = has_kd ? p.kd_weight * p.temperature * g : 0.0f, c1 = has_ce ? p.ce_weight * g : 0.0f;
    float kt = 0.0f, k1 = 0.0f;
    if (has_kd) kt = FWD ? __fdividef(kq * Q, st) : kq * Q * expf(ref * p.inv_t - p.lse[row]);
    if (has_ce) k1 = FWD ? __fdividef(c1, p.grad_kind == ONE ? st : s1) : c1;
    if (p.grad_kind == ONE) { kt += k1; k1 = 0.0f; }  // temperature 1: one exponential for both terms
    const int w0 = aligned ? max(lo, view.whole_lo()) : hi, w1 = aligned ? min(hi, view.whole_hi()) : hi;
    const int v0 = lo + tid;
    T* to = dr + view.first(v0);
    with_exp<T>(p.grad_kind, ref, p.inv_t, [&](const auto& ex) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = v0 + j * THREADS;
        if (v < hi) {
          float d[V];
          unpack_vec<T>(raw[j], d);
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            float et[2], e1[2];
            ex(d[i], d[i + 1], et, e1);
            fmul2(d[i], d[i + 1], et[0], et[1], kt, kt);
            if (ex.two) ffma2(d[i], d[i + 1], e1[0], e1[1], k1, k1, d[i], d[i + 1]);
          }
          T* at = to + j * (THREADS * V);
          if (v >= w0 && v < w1) {
            if (ACC && p.accumulate) {
              float o[V];
              ld16(at, o);
#pragma unroll
              for (int i = 0; i < V; ++i) d[i] += o[i];
            }
            st16(at, d);
          } else {
            store_edge<T>(dr, view.first(v), n, d, ACC && p.accumulate);
          }
        }
      }
    });
    __syncthreads();
    // entries of this slice with a term of their own: the first of equal ids collects the probabilities of all
    const int e_lo = max(view.first(lo), 0), e_hi = min(view.first(hi), n);
    for (int j = tid; j <= k; j += THREADS) {
      const int id = s_id[j];
      if (id < e_lo || id >= e_hi) continue;
      int same = 0;
      for (int i = 0; i <= k; i += 4) {
        const int4 o = *reinterpret_cast<const int4*>(s_id + i);
        same += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
      }
      float w = j < k ? expf(s_t[j] - tref) : 0.0f;
      if (same > 1) {
        int i = 0;
        while (s_id[i] != id) ++i;
        if (i < j) continue;
        w = 0.0f;
        for (; i < k; ++i)
          if (s_id[i] == id) w += expf(s_t[i] - tref);
      }
      float d = 0.0f;
      with_exp<T>(p.grad_kind, ref, p.inv_t, [&](const auto& ex) {
        float et[2], e1[2];
        ex(s_x[j], s_x[j], et, e1);
        d = kt * et[0] + k1 * e1[0];
      });
      if (has_kd) d -= kq * w * inv_s;
      if (id == y) d -= c1;
      if (ACC && p.accumulate) d += s_old[j];
      dr[id] = from_f32<T>(d);
    }
  }
}

int distill_check(const char* what, const DistillParams& p, int dtype, bool bwd) {
  static thread_local char msg[160];
  auto bad = [&](int code, const char* why) {
    snprintf(msg, sizeof(msg), "%s: %s", what, why);
    return fail(code, msg);
  };
  const size_t es = dtype == DT_F32 ? 4 : 2;
  if (dtype != DT_F32 && dtype != DT_BF16) return bad(EISEN_ERR_INVALID, "logits must be f32 or bf16");
  if (!p.logits || !p.t_ids || !p.t_logits) return bad(EISEN_ERR_INVALID, "logits and the teacher's ids and logits must not be null");
  if (p.ld < p.vocab || (bwd && p.ldd < p.vocab)) return bad(EISEN_ERR_INVALID, "a row stride is shorter than a row");
  if ((reinterpret_cast<uintptr_t>(p.logits) % es) || (bwd && (reinterpret_cast<uintptr_t>(p.dlogits) % es)))
    return bad(EISEN_ERR_INVALID, "unaligned pointer");
  if (bwd && !p.dlogits) return bad(EISEN_ERR_INVALID, "dlogits must not be null");
  if (p.k < 1 || p.k > DS_MAX_K) return bad(EISEN_ERR_LIMIT, "k must be in [1, 1024]");
  if (!(p.temperature > 0.0f) || !(p.temperature <= FLT_MAX) || !(1.0f / p.temperature <= FLT_MAX))
    return bad(EISEN_ERR_INVALID, "the temperature must be positive and finite");
  if (!p.targets && p.ce_weight != 0.0f) return bad(EISEN_ERR_INVALID, "a cross-entropy weight needs targets");
  return 0;
}

int distill_sizes(const char* what, long long rows, long long vocab, long long k) {
  static thread_local char msg[160];
  if (rows >= 0 && rows <= 0x7fffffffLL && vocab > 0 && vocab <= 0x7fffff00LL && k >= 0 && k <= 0x7fffffffLL) return 0;
  snprintf(msg, sizeof(msg), "%s: rows must be in [0, 2^31), vocab in [1, 2^31 - 256]", what);
  return fail(EISEN_ERR_LIMIT, msg);
}

// Rows of up to 8 slices of 4096 vectors (262144 bf16 or 131072 f32 entries) stay in registers; longer ones take
// distill_kernel, which reads them a second time.  Short rows in numbers get CTAs of 128 threads, whose barriers are
// cheaper; few rows get more threads and CTAs each.
template <typename T, int MODE>
int distill_launch(const char* what, DistillParams& p, cudaStream_t s) {
  const long long vectors = (p.vocab + VecOf<T>::N - 1) / VecOf<T>::N + 1;  // one more for a row that starts inside one
  const bool few = p.rows < 2LL * sm_count();
  p.cluster = cluster_for_row(p.rows, vectors, 4096, 512);
  if (!p.cluster) {
    distill_kernel<T, MODE><<<(unsigned)p.rows, DS_THREADS, 0, s>>>(p);
    return check_launch(what);
  }
  const long long per = (vectors + p.cluster - 1) / p.cluster;
  if (!few && per <= 256) return launch_rows(distill_row_kernel<T, 128, 2, MODE>, what, p.rows, p.cluster, 128, s, p);
  if (!few && per <= 1024) return launch_rows(distill_row_kernel<T, 128, 8, MODE>, what, p.rows, p.cluster, 128, s, p);
  if (per <= 1024) return launch_rows(distill_row_kernel<T, 256, 4, MODE>, what, p.rows, p.cluster, 256, s, p);
  if (per <= 2048) return launch_rows(distill_row_kernel<T, 256, 8, MODE>, what, p.rows, p.cluster, 256, s, p);
  return launch_rows(distill_row_kernel<T, 256, 16, MODE>, what, p.rows, p.cluster, 256, s, p);
}

int distill_run(const char* what, int mode, DistillParams& p, int dtype, cudaStream_t s) {
  // both exponentials are summed where the caller takes both log-sum-exps or the cross-entropy needs its own
  const bool one = p.temperature == 1.0f;
  p.sum_kind = one || (!p.lse && p.ce_weight == 0.0f) ? ONE : exp_kind(p.temperature, dtype);
  p.grad_kind = one || p.ce_weight == 0.0f ? ONE : exp_kind(p.temperature, dtype);
  EISEN_DISPATCH_DTYPE(dtype, T, {
    if (mode == DS_FWD) return distill_launch<T, DS_FWD>(what, p, s);
    if (mode == DS_BWD) return distill_launch<T, DS_BWD>(what, p, s);
    return distill_launch<T, DS_FWD | DS_BWD>(what, p, s);
  });
}

}  // namespace
}  // namespace eisen

extern "C" {

int eisen_top_logits(void* stream, const void* logits, long long ld, float* values, int* ids, float* lse, long long rows,
                     long long vocab, long long k, float temperature, int dtype) {
  using namespace eisen;
  if (int rc = distill_sizes("top_logits", rows, vocab, k)) return rc;
  if (dtype != DT_F32 && dtype != DT_BF16) return fail(EISEN_ERR_INVALID, "top_logits: logits must be f32 or bf16");
  if (k < 1 || k > TOP_MAX_K || k > vocab) return fail(EISEN_ERR_LIMIT, "top_logits: k must be in [1, min(vocab, 256)]");
  if (ld < vocab) return fail(EISEN_ERR_INVALID, "top_logits: the row stride is shorter than a row");
  if (!(temperature > 0.0f) || !(temperature <= FLT_MAX) || !(1.0f / temperature <= FLT_MAX))
    return fail(EISEN_ERR_INVALID, "top_logits: the temperature must be positive and finite");
  if (rows == 0) return 0;
  if (!logits || !values || !ids) return fail(EISEN_ERR_INVALID, "top_logits: logits, values and ids must not be null");
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DT_F32 ? 4 : 2)) return fail(EISEN_ERR_INVALID, "top_logits: unaligned pointer");
  EISEN_DISPATCH_DTYPE(dtype, T, {
    top_logits_kernel<T><<<(unsigned)rows, TOP_THREADS, 0, (cudaStream_t)stream>>>((const T*)logits, ld, values, ids, lse, (int)vocab,
                                                                                  (int)k, 1.0f / temperature);
    return check_launch("top_logits");
  });
}

int eisen_distill_fwd(void* stream, const void* logits, long long ld, const int* teacher_ids, const float* teacher_logits,
                      const float* teacher_lse, const int* targets, float* loss, float* row_loss, float* lse, long long rows,
                      long long vocab, long long k, int ignore_index, float temperature, float kd_weight, float ce_weight, int dtype,
                      int* bad_id_flag) {
  using namespace eisen;
  if (int rc = distill_sizes("distill_fwd", rows, vocab, k)) return rc;
  DistillParams p = {logits, ld, teacher_ids, teacher_logits, teacher_lse, targets, nullptr, 0, row_loss, lse, nullptr, rows, (int)vocab,
                     (int)k, ignore_index, temperature, 1.0f / temperature, kd_weight, ce_weight, 1.0f, 0, bad_id_flag};
  if (rows == 0) {
    if (loss && cudaMemsetAsync(loss, 0, 4, (cudaStream_t)stream) != cudaSuccess) return fail(EISEN_ERR_CUDA, "distill_fwd: memset");
    return 0;
  }
  if (int rc = distill_check("distill_fwd", p, dtype, false)) return rc;
  if (!row_loss) return fail(EISEN_ERR_INVALID, "distill_fwd: row_loss must not be null");
  const int rc = distill_run("distill_fwd", DS_FWD, p, dtype, (cudaStream_t)stream);
  if (rc || !loss) return rc;
  return eisen_ce_loss_reduce(stream, row_loss, loss, rows);
}

int eisen_distill_bwd(void* stream, const void* logits, long long ld, const int* teacher_ids, const float* teacher_logits,
                      const float* teacher_lse, const int* targets, const float* lse, void* dlogits, long long ld_d,
                      const float* grad_out, long long rows, long long vocab, long long k, int ignore_index, float temperature,
                      float kd_weight, float ce_weight, int dtype, int accumulate) {
  using namespace eisen;
  if (int rc = distill_sizes("distill_bwd", rows, vocab, k)) return rc;
  DistillParams p = {logits, ld, teacher_ids, teacher_logits, teacher_lse, targets, dlogits, ld_d, nullptr, const_cast<float*>(lse),
                     grad_out, rows, (int)vocab, (int)k, ignore_index, temperature, 1.0f / temperature, kd_weight, ce_weight, 1.0f,
                     accumulate, nullptr};
  if (rows == 0) return 0;
  if (int rc = distill_check("distill_bwd", p, dtype, true)) return rc;
  if (!lse) return fail(EISEN_ERR_INVALID, "distill_bwd: lse must not be null");
  return distill_run("distill_bwd", DS_BWD, p, dtype, (cudaStream_t)stream);
}

int eisen_distill_fused(void* stream, const void* logits, long long ld, const int* teacher_ids, const float* teacher_logits,
                        const float* teacher_lse, const int* targets, void* dlogits, long long ld_d, float* loss, float* row_loss,
                        float* lse, long long rows, long long vocab, long long k, int ignore_index, float temperature, float kd_weight,
                        float ce_weight, float grad_scale, int dtype, int* bad_id_flag) {
  using namespace eisen;
  if (int rc = distill_sizes("distill_fused", rows, vocab, k)) return rc;
  DistillParams p = {logits, ld, teacher_ids, teacher_logits, teacher_lse, targets, dlogits, ld_d, row_loss, lse, nullptr, rows,
                     (int)vocab, (int)k, ignore_index, temperature, 1.0f / temperature, kd_weight, ce_weight, grad_scale, 0, bad_id_flag};
  if (rows == 0) {
    if (loss && cudaMemsetAsync(loss, 0, 4, (cudaStream_t)stream) != cudaSuccess) return fail(EISEN_ERR_CUDA, "distill_fused: memset");
    return 0;
  }
  if (int rc = distill_check("distill_fused", p, dtype, true)) return rc;
  if (!row_loss) return fail(EISEN_ERR_INVALID, "distill_fused: row_loss must not be null");
  const int rc = distill_run("distill_fused", DS_FWD | DS_BWD, p, dtype, (cudaStream_t)stream);
  if (rc || !loss) return rc;
  return eisen_ce_loss_reduce(stream, row_loss, loss, rows);
}

}  // extern "C"
