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
#include "row_pipe.cuh"
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
  int sum_kind, grad_kind;  // distill_pipe_kernel: see RowExp
  RowShape shape;
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

// The frame of row_pipe.cuh with a row's work in one group of GT threads:
//   maximum -> sums of the exponentials -> gradient over the logits in shared memory -> the entries with a term of
//   their own (the teacher's ids and the target; the first of equal ids collects the probabilities of all).
// The exponentials are taken again for the gradient.  A row's ids, teacher logits and target are requested while the
// row before it is worked on.
constexpr int pipe_threads(int gt, int groups) { return gt * groups + RP_EXTRA; }
__host__ __device__ constexpr int entry_pad(int k) { return (k + 4) & ~3; }
constexpr int entry_bytes(int k, int groups) { return groups * 2 * 3 * entry_pad(k) * 4; }

template <typename T, int GT, int G, int MODE>
__global__ void __launch_bounds__(GT * G + RP_EXTRA, 1)
distill_pipe_kernel(const DistillParams p) {
  constexpr int V = VecOf<T>::N, GW = GT / 32;
  constexpr int PRE = GT >= 128 ? 1 : 4;  // entries per thread requested a row ahead
  constexpr bool FWD = (MODE & DS_FWD) != 0, BWD = (MODE & DS_BWD) != 0, ACC = BWD && !FWD;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ RowRing ring;
  __shared__ uint64_t xbar[G];
  __shared__ float s_max[G][2][GW], s_sum[G][3][GW];
  __shared__ float s_xch[G][2][8][3];
  const int tid = threadIdx.x, lane = tid & 31;
  const int C = p.shape.cluster, k = p.k, n = p.vocab, KP = entry_pad(k);
  const int rank = C > 1 ? (int)cluster_ctarank() : 0;
  const long long row0 = blockIdx.x / C, stride = gridDim.x / C;
  const int n_mine = row0 < p.rows ? (int)((p.rows - row0 + stride - 1) / stride) : 0;
  ring_init(ring, p.shape.stages, BWD ? 1 : GW, GW);
  if (tid == 0) {
    for (int g = 0; g < G; ++g) mbar_init(&xbar[g], C);
    fence_mbar_init();
  }
  __syncthreads();
  if (C > 1) cluster_sync_all();
  const T* logits = reinterpret_cast<const T*>(p.logits);
  T* dlogits = reinterpret_cast<T*>(p.dlogits);
  auto slice_of = [&](long long row) { return RowSlice<T>(logits + row * p.ld, n, rank, C); };
  auto skipped = [&](int y) { return p.targets && (y == p.ignore_index || y < 0 || y >= n); };
  auto skip_row = [&](long long row) { return p.targets && skipped(p.targets[row]); };

  if (tid >= GT * G + 32) {
    if constexpr (BWD)
      ring_store<T>(ring, smem, p.shape.stages, p.shape.stage_bytes, n_mine, row0, stride, slice_of, skip_row,
                    [&](long long row) { return dlogits + row * p.ldd; });
  } else if (tid >= GT * G) {
    ring_load<T>(ring, smem, p.shape.stages, p.shape.stage_bytes, n_mine, row0, stride, slice_of, skip_row);
  } else {
    const int g = tid / GT, gt = tid % GT, warp = gt >> 5;
    uint8_t* entries = smem + (size_t)p.shape.stages * p.shape.stage_bytes + (size_t)g * (2 * 3 * 4) * KP;
    const bool has_kd = p.kd_weight != 0.0f, has_ce = p.ce_weight != 0.0f;
    const float g_out = p.grad_scale * (BWD && p.grad_out ? *p.grad_out : 1.0f);
    const bool want = BWD || rank == 0;  // this CTA looks at the teacher's entries
    int y_next = -1, id_next[PRE];
    float t_next[PRE], tl_next = 0.0f, lt_next = 0.0f, l1_next = 0.0f;
    auto request = [&](int i) {
      if (i >= n_mine) return;
      const long long row = row0 + i * stride;
      y_next = p.targets ? p.targets[row] : -1;
      if (p.t_lse) tl_next = p.t_lse[row];
      if constexpr (!FWD) { lt_next = p.lse[row]; l1_next = p.lse[p.rows + row]; }
#pragma unroll
      for (int c = 0; c < PRE; ++c) {
        const int j = gt + c * GT;
        id_next[c] = -1;
        t_next[c] = 0.0f;
        if (want && j < k) {
          id_next[c] = p.t_ids[row * k + j];
          t_next[c] = p.t_logits[row * k + j];
        }
      }
    };
    request(g);
    int turn = -1;  // rows this group has worked on (skipped ones do not count): its entries and slots alternate
    for (int i = g; i < n_mine; i += G) {
      const long long row = row0 + i * stride;
      const int st_i = i % p.shape.stages;
      const uint32_t ring_phase = (uint32_t)(i / p.shape.stages) & 1;
      const int y = y_next;
      const float tl_given = tl_next, lt_given = lt_next, l1_given = l1_next;
      T* dr = BWD ? dlogits + row * p.ldd : nullptr;
      const RowSlice<T> s = slice_of(row);
      const bool aligned = BWD && (int)((reinterpret_cast<uintptr_t>(dr) & 15) / sizeof(T)) == s.lead;
      if (skipped(y)) {
        request(i + G);
        if (FWD && gt == 0 && rank == 0) {
          p.row_loss[row] = 0.0f;
          if (p.lse) { p.lse[row] = 0.0f; p.lse[p.rows + row] = 0.0f; }
          if (y != p.ignore_index && p.bad_id_flag) *p.bad_id_flag = 1;
        }
        if (BWD && !(ACC && p.accumulate)) {
          for (int v = s.lo + gt; v < s.hi; v += GT) {
            const int e = s.first(v);
            if (aligned && v >= s.w0 && v < s.w1) *reinterpret_cast<uint4*>(dr + e) = make_uint4(0, 0, 0, 0);
            else
              for (int c = max(e, 0); c < min(e + V, n); ++c) dr[c] = from_f32<T>(0.0f);
          }
        }
        ring_wait_row(ring, i, st_i, ring_phase);
        mbar_arrive_warp(BWD ? &ring.done[st_i] : &ring.empty[st_i]);
        continue;
      }
      ++turn;
      int* s_id = reinterpret_cast<int*>(entries) + (turn & 1) * 3 * KP;
      float* s_t = reinterpret_cast<float*>(s_id + KP);
      float* s_x = s_t + KP;
      float tm = -INFINITY;
      if (want) {
        auto entry = [&](int j, int id, float t) {
          if (id >= n) {
            if (FWD && p.bad_id_flag) *p.bad_id_flag = 1;
            id = -1;
          }
          t = id >= 0 && j < k ? t * p.inv_t : -INFINITY;
          s_id[j] = max(id, -1);
          s_t[j] = t;
          tm = fmaxf(tm, t);
        };
#pragma unroll
        for (int c = 0; c < PRE; ++c) {
          const int j = gt + c * GT;
          if (j < KP) entry(j, j < k ? id_next[c] : (j == k ? y : -1), t_next[c]);
        }
        for (int j = gt + PRE * GT; j < KP; j += GT)
          entry(j, j < k ? p.t_ids[row * k + j] : (j == k ? y : -1), j < k ? p.t_logits[row * k + j] : 0.0f);
      }
      request(i + G);
      // the vectors at the row's ends, by the threads that walk over them
      uint4 edge0 = make_uint4(0, 0, 0, 0), edge1 = edge0;
      const bool own0 = s.w0 > s.lo && gt == 0, own1 = s.w1 < s.hi && s.hi - 1 >= s.w0 && gt == (s.hi - 1 - s.lo) % GT;
      if (own0) edge0 = s.load_edge(s.lo);
      if (own1) edge1 = s.load_edge(s.hi - 1);
      uint4* vec = reinterpret_cast<uint4*>(smem + (size_t)st_i * p.shape.stage_bytes);
      const int cnt = s.hi - s.lo;
      ring_wait_row(ring, i, st_i, ring_phase);
      if (own0) vec[0] = edge0;
      if (own1) vec[cnt - 1] = edge1;

      float ref = 0.0f;
      if constexpr (FWD) {
        float m = -INFINITY;
        if constexpr (sizeof(T) == 2) {
          const uint32_t lowest = 0xff80ff80u;
          __nv_bfloat162 m2 = *reinterpret_cast<const __nv_bfloat162*>(&lowest), m3 = m2;
#pragma unroll 4
          for (int v = gt; v < cnt; v += GT) {
            const uint4 r = vec[v];
            m2 = __hmax2(m2, __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&r.x), *reinterpret_cast<const __nv_bfloat162*>(&r.y)));
            m3 = __hmax2(m3, __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&r.z), *reinterpret_cast<const __nv_bfloat162*>(&r.w)));
          }
          m2 = __hmax2(m2, m3);
          m = fmaxf(__low2float(m2), __high2float(m2));
        } else {
#pragma unroll 4
          for (int v = gt; v < cnt; v += GT) {
            const uint4 r = vec[v];
            m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(r.x), __uint_as_float(r.y))), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
          }
        }
        m = warp_max(m);
        if (lane == 0) s_max[g][0][warp] = m;
      }
      tm = warp_max(tm);
      if (lane == 0) s_max[g][1][warp] = tm;
      group_sync<GT>(g);
      if constexpr (FWD) {
        ref = lanes_max<GW>(s_max[g][0][lane % GW]);
        if (ref == -INFINITY) ref = 0.0f;
      }
      // the teacher's sum: of exp(t - tref) = q_j S, where tref is its given log-sum-exp (S = 1) or its maximum
      float tref = tl_given;
      if (!p.t_lse) {
        tref = lanes_max<GW>(s_max[g][1][lane % GW]);
        if (tref == -INFINITY) tref = 0.0f;
      }
      float S = 0.0f;
      const int e_lo = max(s.first(s.lo), 0), e_hi = min(s.first(s.hi), n);
      if (want)
        for (int j = gt; j <= k; j += GT) {
          const int id = s_id[j];
          float x = 0.0f;
          if (id >= e_lo && id < e_hi) x = to_f32(reinterpret_cast<const T*>(vec)[id - s.first(s.lo)]);
          else if (FWD && C > 1 && rank == 0 && id >= 0) x = to_f32(logits[row * p.ld + id]);
          s_x[j] = x;
          S += expf(s_t[j] - tref);
        }
      float st = 0.0f, s1 = 0.0f;
      if constexpr (FWD) {
        float sa[2] = {0.0f, 0.0f}, sb[2] = {0.0f, 0.0f};
        with_exp<T>(p.sum_kind, ref, p.inv_t, [&](const auto& ex) {
#pragma unroll 2
          for (int v = gt; v < cnt; v += GT) {
            float x[V];
            unpack_vec<T>(vec[v], x);
#pragma unroll
            for (int c = 0; c < V; c += 2) {
              float et[2], e1[2];
              ex(x[c], x[c + 1], et, e1);
              fadd2(sa[0], sa[1], sa[0], sa[1], et[0], et[1]);
              if (ex.two) fadd2(sb[0], sb[1], sb[0], sb[1], e1[0], e1[1]);
            }
          }
        });
        st = warp_sum(sa[0] + sa[1]);
        s1 = warp_sum(sb[0] + sb[1]);
        if (lane == 0) { s_sum[g][0][warp] = st; s_sum[g][1][warp] = s1; }
      }
      S = warp_sum(S);
      if (lane == 0) s_sum[g][2][warp] = S;
      group_sync<GT>(g);
      S = lanes_sum<GW>(s_sum[g][2][lane % GW]);
      // q_j = exp(t_j - tref) * inv_s,  Q = sum of them
      const float inv_s = p.t_lse || S == 0.0f ? 1.0f : __fdividef(1.0f, S), Q = S * inv_s;
      if constexpr (FWD) {
        st = lanes_sum<GW>(s_sum[g][0][lane % GW]);
        s1 = lanes_sum<GW>(s_sum[g][1][lane % GW]);
        if (C > 1) {
          float(*mine)[3] = s_xch[g][turn & 1];
          if (gt < C) {
            const uint32_t to = mapa_cluster(smem_u32(&mine[rank][0]), gt);
            st_cluster_f32(to, st == 0.0f ? -INFINITY : ref);  // a slice without a finite entry has no say in the maximum
            st_cluster_f32(to + 4, st);
            st_cluster_f32(to + 8, s1);
            mbar_arrive_release_cluster(mapa_cluster(smem_u32(&xbar[g]), gt));
          }
          mbar_wait_cluster(&xbar[g], (uint32_t)(turn & 1), &ring.abort_flag);
          float gm = -INFINITY;
          for (int r = 0; r < C; ++r) gm = fmaxf(gm, mine[r][0]);
          ref = gm == -INFINITY ? 0.0f : gm;
          st = s1 = 0.0f;
          for (int r = 0; r < C; ++r) {
            const float d = mine[r][0] - ref;
            st += mine[r][1] * expf(d * p.inv_t);
            s1 += mine[r][2] * expf(d);
          }
        }
        if (warp == GW - 1 && rank == 0) {
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
        ref = l1_given;
      }
      if constexpr (!BWD) {
        fence_proxy_async_smem();  // the vectors at the ends, before a copy takes their place
        mbar_arrive_warp(&ring.empty[st_i]);
      } else {
        // d = kt exp((x - ref) / T) + k1 exp(x - ref): kt, k1 turn the exponentials into weighted probabilities
        const float kq = has_kd ? p.kd_weight * p.temperature * g_out : 0.0f, c1 = has_ce ? p.ce_weight * g_out : 0.0f;
        float kt = 0.0f, k1 = 0.0f;
        if (has_kd) kt = FWD ? __fdividef(kq * Q, st) : kq * Q * expf(ref * p.inv_t - lt_given);
        if (has_ce) k1 = FWD ? __fdividef(c1, p.grad_kind == ONE ? st : s1) : c1;
        if (p.grad_kind == ONE) { kt += k1; k1 = 0.0f; }  // temperature 1: one exponential for both terms
        const bool acc = ACC && p.accumulate;
        with_exp<T>(p.grad_kind, ref, p.inv_t, [&](const auto& ex) {
#pragma unroll 2
          for (int v = gt; v < cnt; v += GT) {
            float d[V];
            unpack_vec<T>(vec[v], d);
#pragma unroll
            for (int c = 0; c < V; c += 2) {
              float et[2], e1[2];
              ex(d[c], d[c + 1], et, e1);
              fmul2(d[c], d[c + 1], et[0], et[1], kt, kt);
              if (ex.two) ffma2(d[c], d[c + 1], e1[0], e1[1], k1, k1, d[c], d[c + 1]);
            }
            if (acc) {
              const int e = s.first(s.lo + v);
              if (aligned && s.lo + v >= s.w0 && s.lo + v < s.w1) {
                float o[V];
                ld16(dr + e, o);
#pragma unroll
                for (int c = 0; c < V; ++c) d[c] += o[c];
              } else {
#pragma unroll
                for (int c = 0; c < V; ++c)
                  if (e + c >= 0 && e + c < n) d[c] += to_f32(dr[e + c]);
              }
            }
            st16(reinterpret_cast<T*>(vec + v), d);
          }
        });
        group_sync<GT>(g);
        T* out = reinterpret_cast<T*>(vec) - s.first(s.lo);  // out[id]: the entry of this slice
        for (int j = gt; j <= k; j += GT) {
          const int id = s_id[j];
          if (id < e_lo || id >= e_hi) continue;
          int same = 0;
          for (int c = 0; c <= k; c += 4) {
            const int4 o = *reinterpret_cast<const int4*>(s_id + c);
            same += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
          }
          float w = j < k ? expf(s_t[j] - tref) : 0.0f;
          if (same > 1) {
            int c = 0;
            while (s_id[c] != id) ++c;
            if (c < j) continue;
            w = 0.0f;
            for (; c < k; ++c)
              if (s_id[c] == id) w += expf(s_t[c] - tref);
          }
          float d = 0.0f;
          with_exp<T>(p.grad_kind, ref, p.inv_t, [&](const auto& ex) {
            float et[2], e1[2];
            ex(s_x[j], s_x[j], et, e1);
            d = kt * et[0] + k1 * e1[0];
          });
          if (has_kd) d -= kq * w * inv_s;
          if (id == y) d -= c1;
          if (acc) d += to_f32(dr[id]);
          out[id] = from_f32<T>(d);
        }
        if (!aligned || s.edges()) {
          group_sync<GT>(g);
          if (!aligned) {
            for (int e = e_lo + gt; e < e_hi; e += GT) dr[e] = out[e];
          } else {
            const int a = min(s.first(s.w0), e_hi), b = max(s.first(s.w1), a);
            for (int e = e_lo + gt; e < a; e += GT) dr[e] = out[e];
            for (int e = b + gt; e < e_hi; e += GT) dr[e] = out[e];
          }
        }
        fence_proxy_async_smem();
        mbar_arrive_warp(&ring.done[st_i]);
      }
    }
  }
  if (ring.abort_flag)
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight end before the CTA does
  if (C > 1) {
    __syncwarp();
    cluster_sync_all();  // nobody leaves while a peer may still write to it
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

// One warp per row for short rows in numbers, groups of 128 or 256 threads for longer ones (a group's reductions cost
// the same whatever its row), all of a CTA's threads where there is at most one row per CTA.  Rows that do not fit the
// shared memory of eight CTAs take distill_kernel, which reads them a second time.
template <typename T, int MODE>
int distill_launch(const char* what, DistillParams& p, cudaStream_t s) {
  const long long bytes = (long long)p.vocab * sizeof(T);
  auto shape = [&](int groups, int least) {
    p.shape = row_shape(p.rows, p.vocab, sizeof(T), entry_bytes(p.k, groups), std::max(2 * groups, 3), least);
    return p.shape.stages >= groups;
  };
  if (p.rows > 2LL * sm_count()) {
    if (bytes <= 4096 && p.k <= 128 && shape(16, 1 << 30))
      return launch_pipe<distill_pipe_kernel<T, 32, 16, MODE>>(what, p.shape, p.rows, pipe_threads(32, 16), s, p);
    if (bytes <= 24 * 1024 && shape(4, 1 << 30))
      return launch_pipe<distill_pipe_kernel<T, 128, 4, MODE>>(what, p.shape, p.rows, pipe_threads(128, 4), s, p);
    if (shape(2, 1 << 30)) return launch_pipe<distill_pipe_kernel<T, 256, 2, MODE>>(what, p.shape, p.rows, pipe_threads(256, 2), s, p);
  }
  if (shape(1, 8192)) return launch_pipe<distill_pipe_kernel<T, 512, 1, MODE>>(what, p.shape, p.rows, pipe_threads(512, 1), s, p);
  distill_kernel<T, MODE><<<(unsigned)p.rows, DS_THREADS, 0, s>>>(p);
  return check_launch(what);
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
