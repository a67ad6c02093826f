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
  EISEN_DISPATCH_DTYPE(dtype, T, {
    distill_kernel<T, DS_FWD><<<(unsigned)rows, DS_THREADS, 0, (cudaStream_t)stream>>>(p);
    int rc = check_launch("distill_fwd");
    if (rc || !loss) return rc;
    return eisen_ce_loss_reduce(stream, row_loss, loss, rows);
  });
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
  EISEN_DISPATCH_DTYPE(dtype, T, {
    distill_kernel<T, DS_BWD><<<(unsigned)rows, DS_THREADS, 0, (cudaStream_t)stream>>>(p);
    return check_launch("distill_bwd");
  });
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
  EISEN_DISPATCH_DTYPE(dtype, T, {
    distill_kernel<T, DS_FWD | DS_BWD><<<(unsigned)rows, DS_THREADS, 0, (cudaStream_t)stream>>>(p);
    int rc = check_launch("distill_fused");
    if (rc || !loss) return rc;
    return eisen_ce_loss_reduce(stream, row_loss, loss, rows);
  });
}

}  // extern "C"
