// The loss of a student against a teacher's top logits (top_logits.cu), and its gradient:
//   kd T^2 sum_j q_j (ln q_j - ln p_j) - ce ln(softmax(x)_y + 1e-8)  with p = softmax(x / T) and q the teacher's
//   distribution over the entries it gives; gradient
//   kd T (Q p_i - sum_{id_j = i} q_j) + ce (softmax(x)_i - [i = y]),  Q = sum_j q_j
//
// Bound by the traffic of the rows of `vocab` logits.  Few rows, and loss and gradient together over rows of more than 16 KB, are read
// once into shared memory and written once (distill_pipe_kernel); all else is read from global memory, and for a gradient beside
// the loss a second time out of the L2 cache (distill_stream_kernel); distill_launch has the rule.  Maxima, sums and statistics are f32.
#include <algorithm>
#include <cfloat>
#include <cstdio>
#include <type_traits>

#include <cuda_fp16.h>

#include "common.cuh"
#include "errors.h"
#include "row_pipe.cuh"
#include "../../include/eisen_b200.h"

namespace eisen {
namespace {

constexpr int DS_MAX_K = 1024;

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
  int sum_kind, grad_kind;  // see RowExp
  int* fault_word;
  RowShape shape;
};

constexpr int DS_FWD = 1, DS_BWD = 2;

// A row's exponentials et = exp((x - ref) / T) and e1 = exp(x - ref).  KIND says how they are formed:
//   ONE     et alone (temperature 1, or no cross-entropy term and one log-sum-exp), as h^2 with h = exp((x - ref) / 2T)
//   3 .. 8  bf16 rows, 2T = 3, 4 .. 8 (T = 1.5, 2 .. 4): et = h^2, e1 = h^2T with the same h
//   TWO     both, each by itself
//   PLAIN1, PLAIN2   (x - ref) first and expf, et alone or both: rows of f32 logits, and bf16 rows whose largest entry is
//           beyond 1e4 (all of it masked by the type's lowest value, say): there the rounding of ref / T is felt
// The special-function unit gives 16 results per clock and SM, 2000 clocks for 32000 entries.  Two exponentials in both
// passes over a row would take 8000 where the memory needs 5600.  So the first pass of the staged form leaves h in the
// row's place in shared memory for the second: f32 rows keep et itself, bf16 rows h in fp16 (half a step is 2^-11 of h;
// et has twice that, a quarter of bf16's own half step, e1 2T <= 8 times, at most as much as bf16's half step).  h, not
// its square, so that fp16's range covers et down to 2^-38 (2T = 8) or 2^-54 (2T <= 3) of the row's largest; smaller
// ones fade to 0.
constexpr int ONE = 2, TWO = 1, PLAIN1 = 10, PLAIN2 = 11;

template <typename T, int KIND>
struct RowExp {
  static constexpr bool ROOT = KIND >= ONE && KIND <= 8;
  static constexpr bool BOTH = KIND != ONE && KIND != PLAIN1;
  static constexpr bool KEEPS = sizeof(T) == 4 ? KIND == PLAIN1 : ROOT;  // what the first pass leaves serves the second
  // h is held times 2^Z: et comes out times 2^2Z, e1 times 2^(KIND Z) (at most 2^40, so that a row's sum and its
  // reciprocal stay in range)
  static constexpr int Z = !ROOT ? 0 : 40 / KIND < 13 ? 40 / KIND : 13;
  static constexpr float scale_t = 1.0f / (float)(1ll << (2 * Z)), scale_1 = 1.0f / (float)(1ll << (ROOT ? KIND * Z : 0));
  float ref, inv_t, c, off, off1;
  __device__ __forceinline__ RowExp(float r, float it) : ref(r), inv_t(it) {
    c = 1.4426950408889634f * (ROOT ? 0.5f * it : it);
    off = (float)Z - r * c;
    off1 = -r * 1.4426950408889634f;
  }
  // h of two elements, or et itself where there is no root
  __device__ __forceinline__ void root(float x, float y, float& h0, float& h1) const {
    if constexpr (KIND >= PLAIN1) {
      h0 = expf((x - ref) * inv_t);
      h1 = expf((y - ref) * inv_t);
    } else {
      ffma2(h0, h1, x, y, c, c, off, off);
      h0 = exp2_approx(h0);
      h1 = exp2_approx(h1);
    }
  }
  __device__ __forceinline__ void powers(float h0, float h1, float (&et)[2], float (&e1)[2]) const {
    if constexpr (!ROOT) {
      et[0] = h0; et[1] = h1;
    } else {
      fmul2(et[0], et[1], h0, h1, h0, h1);
      float f0, f1;  // h^4
      if constexpr (KIND >= 4) fmul2(f0, f1, et[0], et[1], et[0], et[1]);
      if constexpr (KIND == 3) fmul2(e1[0], e1[1], et[0], et[1], h0, h1);
      else if constexpr (KIND == 4) { e1[0] = f0; e1[1] = f1; }
      else if constexpr (KIND == 5) fmul2(e1[0], e1[1], f0, f1, h0, h1);
      else if constexpr (KIND == 6) fmul2(e1[0], e1[1], f0, f1, et[0], et[1]);
      else if constexpr (KIND == 7) {
        fmul2(f0, f1, f0, f1, et[0], et[1]);
        fmul2(e1[0], e1[1], f0, f1, h0, h1);
      } else if constexpr (KIND == 8) fmul2(e1[0], e1[1], f0, f1, f0, f1);
    }
  }
  __device__ __forceinline__ void both(float x, float y, float (&et)[2], float (&e1)[2]) const {
    float h0, h1;
    root(x, y, h0, h1);
    powers(h0, h1, et, e1);
    apart(x, y, e1);
  }
  // e1 where it does not come from h
  __device__ __forceinline__ void apart(float x, float y, float (&e1)[2]) const {
    if constexpr (KIND == TWO) {
      ffma2(e1[0], e1[1], x, y, 1.4426950408889634f, 1.4426950408889634f, off1, off1);
      e1[0] = exp2_approx(e1[0]);
      e1[1] = exp2_approx(e1[1]);
    } else if constexpr (KIND == PLAIN2) {
      e1[0] = expf(x - ref);
      e1[1] = expf(y - ref);
    }
  }
};

// f(RowExp) for the kind that the row takes: one branch per pass, the same for all of its threads
template <typename T, typename F>
__device__ __forceinline__ void with_exp(int kind, float ref, float inv_t, F f) {
  if constexpr (sizeof(T) == 4) {
    if (kind == ONE) f(RowExp<T, PLAIN1>(ref, inv_t));
    else f(RowExp<T, PLAIN2>(ref, inv_t));
  } else {
    if (fabsf(ref) * fmaxf(inv_t, 1.0f) > 1e4f) {
      if (kind == ONE) f(RowExp<T, PLAIN1>(ref, inv_t));
      else f(RowExp<T, PLAIN2>(ref, inv_t));
      return;
    }
    switch (kind) {
      case ONE: return f(RowExp<T, ONE>(ref, inv_t));
      case 3: return f(RowExp<T, 3>(ref, inv_t));
      case 4: return f(RowExp<T, 4>(ref, inv_t));
      case 5: return f(RowExp<T, 5>(ref, inv_t));
      case 6: return f(RowExp<T, 6>(ref, inv_t));
      case 7: return f(RowExp<T, 7>(ref, inv_t));
      case 8: return f(RowExp<T, 8>(ref, inv_t));
      default: return f(RowExp<T, TWO>(ref, inv_t));
    }
  }
}

// What a gradient alone takes its exponentials relative to, given the row's two log-sum-exps: at least its largest entry, and
// not so far above it that exp((ref - x) / T) or exp(ref - x) of that entry leaves the range (T lse(x / T) and lse(x) are
// at most T ln n and ln n above it; divided by a small T the latter may be thousands).
__device__ __forceinline__ float grad_ref(const DistillParams& p, float lt, float l1) {
  return p.temperature < 1.0f ? fminf(l1, lt * p.temperature) : l1;
}

// Rows whose log-sum-exps are no use to a gradient alone: a 32-bit number beyond 512 is off by 2^-16 and more, and so would every
// probability be by that of itself (a row that is masked all over by its type's lowest value has them at 1 instead of
// 1 / n).  Their sums are formed again, relative to the row's largest entry.
__device__ __forceinline__ bool sums_again(float lt, float l1) { return !(fabsf(lt) <= 512.0f && fabsf(l1) <= 512.0f); }

// the kind for both exponentials at a temperature other than 1
int exp_kind(float temperature, int dtype) {
  if (dtype == DT_BF16)
    for (int b = 3; b <= 8; ++b)
      if (temperature * 2.0f == (float)b) return b;
  return TWO;
}

// what the first pass leaves for the second: fp16 in the place of bf16, f32 in that of f32
template <typename T>
__device__ __forceinline__ uint4 keep_vec(const float (&x)[VecOf<T>::N]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      u[i] = __float_as_uint(x[i]);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <typename T>
__device__ __forceinline__ void kept_vec(const uint4& r, float (&x)[VecOf<T>::N]) {
  const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[i] = __uint_as_float(u[i]);
    }
  }
}

// The frame of row_pipe.cuh.  A group of GT threads walks over its row three times: maximum, sums of the exponentials,
// gradient, which goes from registers to global memory: a row of 64 KB sent off from shared memory holds its stage,
// one of three, until it has been read (16384 x 32000 bf16: 454 us, 417 from registers).  Beside it two warps see to what the row has of single entries: one reads, a
// row ahead, the teacher's ids and logits and forms their distribution; the other one, when the group has been through
// the row, forms the loss and rewrites the entries that have a term of their own, the ids and the target.  In the
// group's hands these took a quarter of a row's time (4200 of 17000 clocks), latency after latency with most threads idle.
constexpr int pipe_threads(int gt, int groups) { return (gt + 64) * groups + 32; }
__host__ __device__ constexpr int entry_pad(int k) { return (k + 4) & ~3; }
// slots of the table that finds equal ids: at least four times the entries
__host__ __device__ constexpr int entry_slots(int k) {
  int n = 64;
  while (n < 4 * k) n *= 2;
  return n;
}
__host__ __device__ constexpr int entry_bytes(int k) { return 2 * 5 * 4 * entry_pad(k) + 2 * entry_slots(k); }

// A row's entries in shared memory (two sets per group: one in use, one being read).
struct Entries {
  int* id;   // the teacher's ids, -1: absent or beyond the vocabulary
  float* t;  // its logits / T
  float* x;  // the student's logits there
  float* w;  // exp(t - tref), of all equal ids in one of them; -1 in the others
  float* o;  // what dlogits held there (accumulate)
  __device__ __forceinline__ Entries(uint8_t* p, int set, int pad) {
    id = reinterpret_cast<int*>(p) + set * 5 * pad;
    t = reinterpret_cast<float*>(id + pad);
    x = t + pad;
    w = x + pad;
    o = w + pad;
  }
};
struct RowTeacher {  // exp(t - tref) = q_j S;  Q = sum of the q_j
  float tref, S, Q;
};
struct RowStats {  // what the group found; nt, n1: logarithms of the two sums relative to ref
  float ref, kt, k1, nt, n1;
};

template <typename T, int GT, int G, int MODE>
__global__ void __launch_bounds__((GT + 64) * G + 32, 1)
distill_pipe_kernel(const DistillParams p) {
  constexpr int V = VecOf<T>::N, GW = GT / 32;
  constexpr bool FWD = (MODE & DS_FWD) != 0, BWD = (MODE & DS_BWD) != 0, ACC = BWD && !FWD;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ RowRing ring;
  // a row's entries, its statistics and the barriers around them alternate between two sets
  __shared__ uint64_t ready[G][2];     // the entries are prepared
  __shared__ uint64_t through[G][2];   // the group is through the row (its warps)
  __shared__ uint64_t finished[G][2];  // its entries are rewritten, the loss is formed: the set is free
  __shared__ uint64_t xbar[G];         // the slices of a row have met (C arrivals)
  __shared__ float s_red[G][3][GW];
  __shared__ RowTeacher s_teacher[G][2];
  __shared__ RowStats s_stats[G][2];
  __shared__ float s_xch[G][2][8][3];
  const int tid = threadIdx.x, lane = tid & 31;
  const int C = p.shape.cluster, k = p.k, n = p.vocab;
  const int rank = C > 1 ? (int)cluster_ctarank() : 0;
  const long long row0 = blockIdx.x >> p.shape.cluster_log2, stride = gridDim.x >> p.shape.cluster_log2;
  const int n_mine = row0 < p.rows ? (int)((p.rows - row0 + stride - 1) / stride) : 0;
  ring_init(ring, p.shape.stages, GW);
  if (tid == 0) {
    for (int g = 0; g < G; ++g) {
      mbar_init(&xbar[g], C);
      for (int set = 0; set < 2; ++set) {
        mbar_init(&ready[g][set], 1);
        mbar_init(&through[g][set], GW);
        mbar_init(&finished[g][set], 1);
      }
    }
    fence_mbar_init();
  }
  __syncthreads();
  if (C > 1) cluster_sync_all();
  const T* logits = reinterpret_cast<const T*>(p.logits);
  T* dlogits = reinterpret_cast<T*>(p.dlogits);
  const bool has_kd = p.kd_weight != 0.0f, has_ce = p.ce_weight != 0.0f;
  const float g_out = p.grad_scale * (BWD && p.grad_out ? *p.grad_out : 1.0f);
  const float kq = has_kd ? p.kd_weight * p.temperature * g_out : 0.0f, c1 = has_ce ? p.ce_weight * g_out : 0.0f;
  const bool acc = ACC && p.accumulate;
  auto slice_of = [&](long long row) { return RowSlice<T>(logits + row * p.ld, n, rank, p.shape.cluster_log2); };
  auto skipped = [&](int y) { return p.targets && (y == p.ignore_index || y < 0 || y >= n); };
  auto skip_row = [&](long long row) { return p.targets && skipped(p.targets[row]); };
  // dlogits' row starts like the logits' row: whole vectors go there as they are
  auto like = [&](const RowSlice<T>& s, const T* dr) { return (int)(((uint32_t)reinterpret_cast<uintptr_t>(dr) & 15) / sizeof(T)) == s.lead; };
  constexpr int ENTRY0 = GT * G, LOAD0 = ENTRY0 + 64 * G;

  if (tid >= LOAD0) {
    ring_load<T>(ring, smem, p.shape.stages, p.shape.stage_bytes, n_mine, row0, stride, slice_of, skip_row);
  } else if (tid >= ENTRY0) {
    // ---------------- the two entry warps of group g ----------------
    const int g = (tid - ENTRY0) / 64;
    const bool preparing = ((tid - ENTRY0) & 32) == 0;
    const int KP = entry_pad(k), slots = entry_slots(k);
    uint8_t* mine = smem + (size_t)p.shape.stages * p.shape.stage_bytes + (size_t)g * entry_bytes(k);
    uint16_t* table = reinterpret_cast<uint16_t*>(mine + 2 * 5 * 4 * KP);
    const bool want = BWD || rank == 0;  // this CTA has use for the entries
    // the next row of this group that counts (n_mine or more: none) and its target; the targets are requested one ahead
    int cand = g, y_cand = p.targets && g < n_mine ? p.targets[row0 + (long long)g * stride] : -1;
    auto next_row = [&](int& y) {
      while (cand < n_mine) {
        const int i = cand;
        y = y_cand;
        cand += G;
        if (p.targets && cand < n_mine) y_cand = p.targets[row0 + (long long)cand * stride];
        if (!skipped(y)) return i;
      }
      return n_mine;
    };
    // The first 64 entries of a row (two per lane) are requested while the row before it is prepared, and the student's
    // logits there at the end of that.
    int id_next[2], id[2];
    float t_next[2], x_next[2], t[2], x[2], tl_next = 0.0f, xy_next = 0.0f;
    auto clean = [&](int v) {
      if (v >= n) {
        if (FWD && p.bad_id_flag) *p.bad_id_flag = 1;
        return -1;
      }
      return max(v, -1);
    };
    auto request = [&](int i) {
      if (i >= n_mine) return;
      const long long row = row0 + (long long)i * stride;
      const int* ids = p.t_ids + row * k + lane;
      const float* tv = p.t_logits + row * k + lane;
      if (p.t_lse) tl_next = p.t_lse[row];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool in = lane + 32 * c < k;
        id_next[c] = in ? ids[32 * c] : -1;
        t_next[c] = in ? tv[32 * c] : 0.0f;
      }
    };
    auto gather = [&](int i, int y) {
      if (i >= n_mine) return;
      const T* xr = logits + (row0 + (long long)i * stride) * p.ld;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        id_next[c] = clean(id_next[c]);
        x_next[c] = id_next[c] >= 0 ? to_f32(xr[id_next[c]]) : 0.0f;
      }
      xy_next = y >= 0 ? to_f32(xr[y]) : 0.0f;
    };
    auto prepare = [&](int i, int y, int set, int after, int y_after) {
      const long long row = row0 + (long long)i * stride;
      const T* xr = logits + row * p.ld;
      const T* dr = dlogits + row * p.ldd;
      const Entries e(mine, set, KP);
      float ref = -INFINITY;
      const float tl_given = tl_next, xy = xy_next;
#pragma unroll
      for (int c = 0; c < 2; ++c) { id[c] = id_next[c]; t[c] = t_next[c]; x[c] = x_next[c]; }
      request(after);
      if (lane == 0) {
        e.x[k] = xy;
        if (ACC && acc) e.o[k] = y >= 0 ? to_f32(dr[y]) : 0.0f;
      }
      for (int j0 = lane; j0 - lane < k; j0 += 64) {
        if (j0 >= 64) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int j = j0 + 32 * c;
            id[c] = j < k ? clean(p.t_ids[row * k + j]) : -1;
            t[c] = j < k ? p.t_logits[row * k + j] : 0.0f;
            x[c] = id[c] >= 0 ? to_f32(xr[id[c]]) : 0.0f;
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int j = j0 + 32 * c;
          if (j < k) {
            t[c] = id[c] >= 0 ? t[c] * p.inv_t : -INFINITY;
            e.id[j] = id[c];
            e.t[j] = t[c];
            e.x[j] = x[c];
            if (ACC && acc) e.o[j] = id[c] >= 0 ? to_f32(dr[id[c]]) : 0.0f;
            ref = fmaxf(ref, t[c]);
          }
        }
      }
      // exp(t - ref) = q_j S, where ref is the teacher's given log-sum-exp (S = 1) or its maximum.  A row without an entry
      // above -inf has no weight whatever was given for it: the log-sum-exp of a teacher that masks everything is -inf too
      const float most = warp_max(ref);
      ref = most == -INFINITY ? 0.0f : p.t_lse ? tl_given : most;
      if constexpr (BWD)
        for (int c = lane; c < slots / 8; c += 32) reinterpret_cast<uint4*>(table)[c] = make_uint4(~0u, ~0u, ~0u, ~0u);
      __syncwarp();
      float S = 0.0f;
      bool again = false;
      for (int j = lane; j < k; j += 32) {
        const float w = expf(e.t[j] - ref);
        S += w;
        if constexpr (BWD) {
          // equal ids find the same slot: whoever came first there stands for all of them (who it is does not matter)
          const int id = e.id[j];
          bool first = id >= 0;
          if (id >= 0) {
            int h = (int)(((uint32_t)id * 0x9e3779b1u) >> 16) & (slots - 1);
            for (int tries = 0; tries < slots; ++tries) {
              const uint16_t o = atomicCAS(table + h, (uint16_t)0xffff, (uint16_t)j);
              if (o == 0xffff) break;
              if (e.id[o] == id) { first = false; again = true; break; }
              h = (h + 1) & (slots - 1);
            }
          }
          e.w[j] = first ? w : -1.0f;
        }
      }
      if (BWD && __any_sync(0xffffffffu, again)) {
        __syncwarp();
        for (int j = lane; j < k; j += 32)
          if (e.w[j] != -1.0f) {  // in the order of the entries, so that the sum is the same every time
            float w = 0.0f;
            for (int c = 0; c < k; ++c)
              if (e.id[c] == e.id[j]) w += expf(e.t[c] - ref);
            e.w[j] = w;
          }
      }
      S = warp_sum(S);
      if (lane == 0) s_teacher[g][set] = {ref, S, p.t_lse || S == 0.0f ? S : 1.0f};
      gather(after, y_after);
    };
    int y = -1, y_after = -1;
    int i = next_row(y);
    if (preparing && want) {
      request(i);
      gather(i, y);
    }
    for (int turn = 0; i < n_mine; ++turn) {
      const int set = turn & 1;
      const uint32_t phase = (uint32_t)(turn >> 1) & 1;
      const int after = next_row(y_after);
      if (preparing) {
        if (turn >= 2) mbar_wait(&finished[g][set], phase ^ 1, &ring.abort_flag, nullptr, FAULT_WAIT_EMPTY);
        if (want) prepare(i, y, set, after, y_after);
        mbar_arrive_warp(&ready[g][set]);
        i = after;
        y = y_after;
        continue;
      }
      mbar_wait(&ready[g][set], phase, &ring.abort_flag, nullptr, FAULT_WAIT_FULL);
      mbar_wait(&through[g][set], phase, &ring.abort_flag, nullptr, FAULT_WAIT_FULL);
      const long long row = row0 + (long long)i * stride;
      const Entries e(mine, set, KP);
      const RowStats st = s_stats[g][set];
      const RowTeacher te = s_teacher[g][set];
      const float S = te.S, inv_s = p.t_lse || S == 0.0f ? 1.0f : 1.0f / S;
      if constexpr (BWD) {
        const RowSlice<T> s = slice_of(row);
        T* dr = dlogits + row * p.ldd;
        const int e_lo = max(s.first(s.lo), 0), e_hi = min(s.first(s.hi), n);
        auto rewrite = [&](int j, int id, float less) {
          float x = e.x[j];
          x -= st.ref;
          float d = st.kt * expf(x * p.inv_t);
          if (st.k1 != 0.0f) d += st.k1 * expf(x);
          d -= less;
          if (ACC && acc) d += e.o[j];
          dr[id] = from_f32<T>(d);
        };
        bool met = false;  // the target is one of the ids
        for (int j = lane; j < k; j += 32) {
          const int id = e.id[j];
          const float w = e.w[j];
          met |= id >= 0 && id == y;
          if (id >= e_lo && id < e_hi && w != -1.0f) rewrite(j, id, (has_kd ? kq * w * inv_s : 0.0f) + (id == y ? c1 : 0.0f));
        }
        met = __any_sync(0xffffffffu, met);
        if (has_ce && !met && lane == 0 && y >= e_lo && y < e_hi) rewrite(k, y, c1);
      }
      if (FWD && rank == 0) {
        // in differences: far from 0 the log-sum-exps themselves are rounded too coarsely
        const float ns = p.t_lse || S == 0.0f ? 0.0f : logf(S);
        float kl = 0.0f;
        for (int j = lane; j < k; j += 32) {
          const float lq = e.t[j] - te.tref - ns, q = expf(lq);
          if (q > 0.0f || q != q) kl += q * (lq - ((e.x[j] - st.ref) * p.inv_t - st.nt));
        }
        kl = warp_sum(kl);
        if (lane == 0) {
          float l = 0.0f;
          if (has_kd) l = p.kd_weight * p.temperature * p.temperature * kl;
          if (has_ce) l -= p.ce_weight * logf(expf(e.x[k] - st.ref - st.n1) + 1e-8f);
          p.row_loss[row] = l;
          if (p.lse) {
            p.lse[row] = st.ref * p.inv_t + st.nt;
            p.lse[p.rows + row] = st.ref + st.n1;
          }
        }
      }
      mbar_arrive_warp(&finished[g][set]);
      i = after;
      y = y_after;
    }
  } else {
    // ---------------- a group ----------------
    const int g = tid / GT, gt = tid % GT, warp = gt >> 5;
    int y_next = -1;
    float lt_next = 0.0f, l1_next = 0.0f;
    auto request = [&](int i) {
      if (i >= n_mine) return;
      const long long row = row0 + (long long)i * stride;
      y_next = p.targets ? p.targets[row] : -1;
      if constexpr (!FWD) { lt_next = p.lse[row]; l1_next = p.lse[p.rows + row]; }
    };
    request(g);
    int turn = -1;       // rows this group has worked on (skipped ones do not count)
    int met_rows = 0;    // those of them whose slices have met
    int stage = g - G;   // the stage of row i, and its phase; a ring has at least G stages
    uint32_t phase = 0;
    for (int i = g; i < n_mine; i += G) {
      stage += G;
      if (stage >= p.shape.stages) { stage -= p.shape.stages; phase ^= 1; }
      const long long row = row0 + (long long)i * stride;
      const int y = y_next;
      const float lt_given = lt_next, l1_given = l1_next;
      request(i + G);
      T* dr = BWD ? dlogits + row * p.ldd : nullptr;
      const RowSlice<T> s = slice_of(row);
      if (skipped(y)) {
        if (FWD && gt == 0 && rank == 0) {
          p.row_loss[row] = 0.0f;
          if (p.lse) { p.lse[row] = 0.0f; p.lse[p.rows + row] = 0.0f; }
          if (y != p.ignore_index && p.bad_id_flag) *p.bad_id_flag = 1;
        }
        if (BWD && !acc) {
          const bool whole = like(s, dr);
          for (int v = s.lo + gt; v < s.hi; v += GT) {
            const int e = s.first(v);
            if (whole && v >= s.w0 && v < s.w1) *reinterpret_cast<uint4*>(dr + e) = make_uint4(0, 0, 0, 0);
            else
              for (int c = max(e, 0); c < min(e + V, n); ++c) dr[c] = from_f32<T>(0.0f);
          }
        }
        ring_wait_row(ring, i, stage, phase);
        mbar_arrive_warp(&ring.empty[stage]);
        continue;
      }
      ++turn;
      const int set = turn & 1;
      const uint32_t set_phase = (uint32_t)(turn >> 1) & 1;
      // the vectors at the row's ends, by the threads that walk over them
      uint4 edge0 = make_uint4(0, 0, 0, 0), edge1 = edge0;
      const bool own0 = s.w0 > s.lo && gt == 0, own1 = s.w1 < s.hi && s.hi - 1 >= s.w0 && gt == (s.hi - 1 - s.lo) % GT;
      if (own0) edge0 = s.load_edge(s.lo);
      if (own1) edge1 = s.load_edge(s.hi - 1);
      uint4* vec = reinterpret_cast<uint4*>(smem + (size_t)stage * p.shape.stage_bytes);
      const int cnt = s.hi - s.lo;
      ring_wait_row(ring, i, stage, phase);
      if (own0) vec[0] = edge0;
      if (own1) vec[cnt - 1] = edge1;

      const bool sums = FWD || sums_again(lt_given, l1_given);
      float ref = FWD ? 0.0f : grad_ref(p, lt_given, l1_given), own_ref = ref, st = 0.0f, s1 = 0.0f, own_st = 1.0f;
      if (sums) {
        float m = -INFINITY;
        if constexpr (sizeof(T) == 2) {
          auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
          __nv_bfloat162 m2 = pair(0xff80ff80u), m3 = m2;
#pragma unroll 4
          for (int v = gt; v < cnt; v += GT) {
            const uint4 r = vec[v];
            m2 = __hmax2(m2, __hmax2(pair(r.x), pair(r.y)));
            m3 = __hmax2(m3, __hmax2(pair(r.z), pair(r.w)));
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
        if (lane == 0) s_red[g][0][warp] = m;
        group_sync<GT>(g);
        ref = lanes_max<GW>(s_red[g][0][lane % GW]);
        if (ref == -INFINITY) ref = 0.0f;
        own_ref = ref;
        float sa[2] = {0.0f, 0.0f}, sb[2] = {0.0f, 0.0f};
        with_exp<T>(p.sum_kind, ref, p.inv_t, [&](const auto& ex) {
          using Ex = std::remove_cv_t<std::remove_reference_t<decltype(ex)>>;
          uint4 next = gt < cnt ? vec[gt] : make_uint4(0, 0, 0, 0);
#pragma unroll 1
          for (int v = gt; v < cnt; v += GT) {
            float x[V];
            unpack_vec<T>(next, x);
            if (v + GT < cnt) next = vec[v + GT];  // on its way while this one is worked on
#pragma unroll
            for (int c = 0; c < V; c += 2) {
              float h0, h1, et[2], e1[2];
              ex.root(x[c], x[c + 1], h0, h1);
              ex.powers(h0, h1, et, e1);
              ex.apart(x[c], x[c + 1], e1);
              fadd2(sa[0], sa[1], sa[0], sa[1], et[0], et[1]);
              if constexpr (Ex::BOTH) fadd2(sb[0], sb[1], sb[0], sb[1], e1[0], e1[1]);
              x[c] = h0;
              x[c + 1] = h1;
            }
            if constexpr (FWD && BWD && Ex::KEEPS) vec[v] = keep_vec<T>(x);
          }
          st = (sa[0] + sa[1]) * Ex::scale_t;
          s1 = (sb[0] + sb[1]) * Ex::scale_1;
        });
        st = warp_sum(st);
        s1 = warp_sum(s1);
        if (lane == 0) { s_red[g][1][warp] = st; s_red[g][2][warp] = s1; }
        group_sync<GT>(g);
        if constexpr (!BWD) {
          fence_proxy_async_smem();  // the vectors at the ends, before a copy takes their place
          mbar_arrive_warp(&ring.empty[stage]);
        }
        st = lanes_sum<GW>(s_red[g][1][lane % GW]);
        s1 = lanes_sum<GW>(s_red[g][2][lane % GW]);
        if (C > 1) {
          own_st = st;
          // the entry warp has read its logits: after the exchange the other CTAs may write theirs over them
          mbar_wait(&ready[g][set], set_phase, &ring.abort_flag, nullptr, FAULT_WAIT_FULL);
          float(*met)[3] = s_xch[g][met_rows & 1];
          if (gt < C) {
            const uint32_t to = mapa_cluster(smem_u32(&met[rank][0]), gt);
            st_cluster_f32(to, st == 0.0f ? -INFINITY : ref);  // a slice without a finite entry has no say in the maximum
            st_cluster_f32(to + 4, st);
            st_cluster_f32(to + 8, s1);
            mbar_arrive_release_cluster(mapa_cluster(smem_u32(&xbar[g]), gt));
          }
          mbar_wait_cluster(&xbar[g], (uint32_t)(met_rows & 1), &ring.abort_flag);
          ++met_rows;
          float gm = -INFINITY;
          for (int r = 0; r < C; ++r) gm = fmaxf(gm, met[r][0]);
          ref = gm == -INFINITY ? 0.0f : gm;
          st = s1 = 0.0f;
          for (int r = 0; r < C; ++r) {
            const float d = met[r][0] - ref;
            st += met[r][1] * expf(d * p.inv_t);
            s1 += met[r][2] * expf(d);
          }
        }
      }
      if (!(sums && C > 1)) mbar_wait(&ready[g][set], set_phase, &ring.abort_flag, nullptr, FAULT_WAIT_FULL);
      // d = kt exp((x - ref) / T) + k1 exp(x - ref): kt, k1 turn the exponentials into weighted probabilities
      float kt = 0.0f, k1 = 0.0f;
      if constexpr (BWD) {
        const float Q = s_teacher[g][set].Q;
        if (has_kd) kt = sums ? __fdividef(kq * Q, st) : kq * Q * expf(ref * p.inv_t - lt_given);
        if (has_ce) k1 = sums ? __fdividef(c1, p.grad_kind == ONE ? st : s1) : c1 * expf(ref - l1_given);
        if (p.grad_kind == ONE) { kt += k1; k1 = 0.0f; }  // temperature 1: one exponential for both terms
      }
      if (gt == 0) {
        RowStats& o = s_stats[g][set];
        o.ref = ref;
        o.kt = kt;
        o.k1 = k1;
        if constexpr (FWD) {
          o.nt = logf(st);
          o.n1 = p.sum_kind == ONE ? o.nt : logf(s1);  // temperature 1: the same sum; otherwise there is no use for a second one
        }
      }
      if constexpr (!BWD) {
        mbar_arrive_warp(&through[g][set]);
      } else {
        // vectors that go to dlogits as they are
        const int w0 = like(s, dr) ? s.w0 : s.hi, w1 = like(s, dr) ? s.w1 : s.hi;
        // a slice without a finite entry has nothing but zeros
        const float at = C > 1 && sums ? (own_st == 0.0f ? 0.0f : expf((own_ref - ref) * p.inv_t)) : 1.0f;
        const float a1 = C > 1 && sums ? (own_st == 0.0f ? 0.0f : expf(own_ref - ref)) : 1.0f;
        with_exp<T>(FWD ? p.sum_kind : p.grad_kind, own_ref, p.inv_t, [&](const auto& ex) {
          using Ex = std::remove_cv_t<std::remove_reference_t<decltype(ex)>>;
          const float mt = kt * at * Ex::scale_t, m1 = k1 * a1 * Ex::scale_1;
          uint4 next = gt < cnt ? vec[gt] : make_uint4(0, 0, 0, 0);
#pragma unroll 1
          for (int v = gt; v < cnt; v += GT) {
            float d[V];
            if constexpr (FWD && Ex::KEEPS) kept_vec<T>(next, d);
            else unpack_vec<T>(next, d);
            if (v + GT < cnt) next = vec[v + GT];
#pragma unroll
            for (int c = 0; c < V; c += 2) {
              float et[2], e1[2];
              if constexpr (FWD && Ex::KEEPS) ex.powers(d[c], d[c + 1], et, e1);
              else ex.both(d[c], d[c + 1], et, e1);
              fmul2(d[c], d[c + 1], et[0], et[1], mt, mt);
              if constexpr (Ex::BOTH) ffma2(d[c], d[c + 1], e1[0], e1[1], m1, m1, d[c], d[c + 1]);
            }
            const int e = s.first(s.lo + v);
            if (s.lo + v >= w0 && s.lo + v < w1) {
              if (ACC && acc) {
                float o[V];
                ld16(dr + e, o);
#pragma unroll
                for (int c = 0; c < V; ++c) d[c] += o[c];
              }
              st16(dr + e, d);
            } else {
#pragma unroll
              for (int c = 0; c < V; ++c)
                if (e + c >= 0 && e + c < n) {
                  if (ACC && acc) d[c] += to_f32(dr[e + c]);
                  dr[e + c] = from_f32<T>(d[c]);
                }
            }
          }
        });
        fence_proxy_async_smem();  // what was kept in the row's place, before a copy takes it
        mbar_arrive_warp(&ring.empty[stage]);
        mbar_arrive_warp(&through[g][set]);
      }
    }
  }
  if (ring_gave_up(ring, C, p.fault_word)) {
    for (int i = tid; i < n_mine; i += blockDim.x) {
      const long long row = row0 + (long long)i * stride;
      if (FWD) p.row_loss[row] = NAN;
      if (BWD) dlogits[row * p.ldd] = from_f32<T>(NAN);
    }
  }
}

// largest element of a vector
template <typename T>
__device__ __forceinline__ float largest(const uint4& r) {
  if constexpr (sizeof(T) == 2) {
    auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2(__hmax2(pair(r.x), pair(r.y)), __hmax2(pair(r.z), pair(r.w)));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
}

// Rows in numbers: nothing is staged.  A CTA reads its row once for a running maximum and sums (four vectors of every
// thread in flight, brought to a new maximum four vectors at a time), and where there is a gradient once more, out of the
// L2 cache.  Ten CTAs of 128 threads per SM (32 of one warp for short rows, five of 256 for long f32 rows: 600 x 131072, loss and
// then gradient, 181 us against 215) cover each other's latencies: the entries' gathers, the reductions, the entries that
// are written last.  The staged form has two or three rows at work on an SM.
constexpr int DF_FLIGHT = 4;
constexpr int stream_bytes(int k) { return 5 * 4 * entry_pad(k) + 2 * entry_slots(k); }

template <typename T, int DF_THREADS, int MODE, bool AGAIN>
__device__ __forceinline__ void distill_stream_row(const DistillParams& p) {
  constexpr int V = VecOf<T>::N, WARPS = DF_THREADS / 32;
  constexpr bool FWD = (MODE & DS_FWD) != 0, BWD = (MODE & DS_BWD) != 0, ACC = BWD && !FWD;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_red[4][WARPS];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.vocab, k = p.k;
  const Entries e(smem, 0, entry_pad(k));
  uint16_t* table = reinterpret_cast<uint16_t*>(smem + 5 * 4 * entry_pad(k));
  const T* xr = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  T* dr = BWD ? reinterpret_cast<T*>(p.dlogits) + row * p.ldd : nullptr;
  const RowSlice<T> s(xr, n, 0, 0);
  // vectors that go to dlogits as they are
  const bool like = BWD && (int)(((uint32_t)reinterpret_cast<uintptr_t>(dr) & 15) / sizeof(T)) == s.lead;
  const int w0 = like ? s.w0 : s.hi, w1 = like ? s.w1 : s.hi;
  const bool acc = ACC && p.accumulate;
  const int y = p.targets ? p.targets[row] : -1;
  const bool ignored = p.targets && y == p.ignore_index;
  const bool out = p.targets && !ignored && (y < 0 || y >= n);
  if (ignored || out) {
    if (FWD && tid == 0) {
      p.row_loss[row] = 0.0f;
      if (p.lse) { p.lse[row] = 0.0f; p.lse[p.rows + row] = 0.0f; }
      if (out && p.bad_id_flag) *p.bad_id_flag = 1;
    }
    if (BWD && !acc)
      for (int v = tid; v < s.hi; v += DF_THREADS) {
        const int at = s.first(v);
        if (v >= w0 && v < w1) *reinterpret_cast<uint4*>(dr + at) = make_uint4(0, 0, 0, 0);
        else
          for (int c = max(at, 0); c < min(at + V, n); ++c) dr[c] = from_f32<T>(0.0f);
      }
    return;
  }
  // the teacher's entries, absent ones at -inf; entry k is the target
  float tm = -INFINITY;
  for (int j = tid; j <= k; j += DF_THREADS) {
    int id = j < k ? p.t_ids[row * k + j] : y;
    float t = j < k ? p.t_logits[row * k + j] * p.inv_t : -INFINITY;
    if (id >= n) {
      if (FWD && p.bad_id_flag) *p.bad_id_flag = 1;
      id = -1;
    }
    id = max(id, -1);
    if (id < 0) t = -INFINITY;
    e.id[j] = id;
    e.t[j] = t;
    e.x[j] = id >= 0 ? to_f32(xr[id]) : 0.0f;
    if (ACC && acc) e.o[j] = id >= 0 ? to_f32(dr[id]) : 0.0f;
    tm = fmaxf(tm, t);
  }
  if constexpr (BWD)
    for (int c = tid; c < entry_slots(k) / 8; c += DF_THREADS) reinterpret_cast<uint4*>(table)[c] = make_uint4(~0u, ~0u, ~0u, ~0u);
  float m = -INFINITY, st = 0.0f, s1 = 0.0f;
  constexpr bool sums = FWD || AGAIN;
  if constexpr (sums) {
#pragma unroll 1
    for (int v0 = tid; v0 < s.hi; v0 += DF_FLIGHT * DF_THREADS) {
      uint4 raw[DF_FLIGHT];
      load_vectors<T>(s, v0, DF_THREADS, raw);
      float bm = m;
#pragma unroll
      for (int q = 0; q < DF_FLIGHT; ++q) bm = fmaxf(bm, largest<T>(raw[q]));
      const float ref = bm == -INFINITY ? 0.0f : bm;
      if (bm > m) {
        st *= m == -INFINITY ? 0.0f : expf((m - ref) * p.inv_t);  // a NaN of st stays one
        s1 *= m == -INFINITY ? 0.0f : expf(m - ref);
        m = bm;
      }
      with_exp<T>(p.sum_kind, ref, p.inv_t, [&](const auto& ex) {
        using Ex = std::remove_cv_t<std::remove_reference_t<decltype(ex)>>;
        float sa[2] = {0.0f, 0.0f}, sb[2] = {0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < DF_FLIGHT; ++q) {
          float x[V];
          unpack_vec<T>(raw[q], x);
#pragma unroll
          for (int c = 0; c < V; c += 2) {
            float et[2], e1[2];
            ex.both(x[c], x[c + 1], et, e1);
            fadd2(sa[0], sa[1], sa[0], sa[1], et[0], et[1]);
            if constexpr (Ex::BOTH) fadd2(sb[0], sb[1], sb[0], sb[1], e1[0], e1[1]);
          }
        }
        st += (sa[0] + sa[1]) * Ex::scale_t;
        s1 += (sb[0] + sb[1]) * Ex::scale_1;
      });
    }
  }
  // maxima, then the sums relative to them
  if constexpr (sums) {
    const float wm = warp_max(m);
    if (lane == 0) s_red[0][warp] = wm;
  }
  tm = warp_max(tm);
  if (lane == 0) s_red[1][warp] = tm;
  __syncthreads();
  float ref = sums ? lanes_max<WARPS>(s_red[0][lane % WARPS]) : grad_ref(p, p.lse[row], p.lse[p.rows + row]);
  if (ref == -INFINITY) ref = 0.0f;
  // exp(t - tref) = q_j S, where tref is the teacher's given log-sum-exp (S = 1) or its maximum; 0 without an entry above -inf
  float tref = lanes_max<WARPS>(s_red[1][lane % WARPS]);
  if (tref == -INFINITY) tref = 0.0f;
  else if (p.t_lse) tref = p.t_lse[row];
  float S = 0.0f;
  bool again = false;
  for (int j = tid; j < k; j += DF_THREADS) {
    const float w = expf(e.t[j] - tref);
    S += w;
    if constexpr (BWD) {
      // equal ids find the same slot: whoever came first there stands for all of them (who it is does not matter)
      const int id = e.id[j];
      bool first = id >= 0;
      if (id >= 0) {
        const int slots = entry_slots(k);
        int h = (int)(((uint32_t)id * 0x9e3779b1u) >> 16) & (slots - 1);
        for (int tries = 0; tries < slots; ++tries) {
          const uint16_t o = atomicCAS(table + h, (uint16_t)0xffff, (uint16_t)j);
          if (o == 0xffff) break;
          if (e.id[o] == id) { first = false; again = true; break; }
          h = (h + 1) & (slots - 1);
        }
      }
      e.w[j] = first ? w : -1.0f;
    }
  }
  S = warp_sum(S);
  if constexpr (sums) {
    const float mine = m == -INFINITY ? 0.0f : m - ref;
    st = warp_sum(st * expf(mine * p.inv_t));
    s1 = warp_sum(s1 * expf(mine));
  }
  __syncthreads();
  if (lane == 0) { s_red[0][warp] = st; s_red[1][warp] = s1; s_red[2][warp] = S; }
  again = __syncthreads_or(again);
  st = lanes_sum<WARPS>(s_red[0][lane % WARPS]);
  s1 = lanes_sum<WARPS>(s_red[1][lane % WARPS]);
  S = lanes_sum<WARPS>(s_red[2][lane % WARPS]);
  const bool has_kd = p.kd_weight != 0.0f, has_ce = p.ce_weight != 0.0f;
  float kl = 0.0f;
  if constexpr (FWD) {
    if (warp == 0 || !BWD) {  // the loss; beside a gradient in the hands of one warp
      // in differences: far from 0 the log-sum-exps themselves are rounded too coarsely
      const float nt = logf(st), ns = p.t_lse || S == 0.0f ? 0.0f : logf(S);
      for (int j = BWD ? lane : tid; j < k; j += BWD ? 32 : DF_THREADS) {
        const float lq = e.t[j] - tref - ns, q = expf(lq);
        if (q > 0.0f || q != q) kl += q * (lq - ((e.x[j] - ref) * p.inv_t - nt));
      }
      kl = warp_sum(kl);
    }
    if constexpr (!BWD) {
      if (lane == 0) s_red[3][warp] = kl;
      __syncthreads();
      kl = lanes_sum<WARPS>(s_red[3][lane % WARPS]);
    }
    if (tid == 0) {
      const float nt = logf(st), n1 = p.sum_kind == ONE ? nt : logf(s1);
      float l = 0.0f;
      if (has_kd) l = p.kd_weight * p.temperature * p.temperature * kl;
      if (has_ce) l -= p.ce_weight * logf(expf(e.x[k] - ref - n1) + 1e-8f);
      p.row_loss[row] = l;
      if (p.lse) {
        p.lse[row] = ref * p.inv_t + nt;
        p.lse[p.rows + row] = ref + n1;
      }
    }
  }
  if constexpr (BWD) {
    // d = kt exp((x - ref) / T) + k1 exp(x - ref): kt, k1 turn the exponentials into weighted probabilities
    const float g = p.grad_scale * (p.grad_out ? *p.grad_out : 1.0f);
    const float kq = has_kd ? p.kd_weight * p.temperature * g : 0.0f, c1 = has_ce ? p.ce_weight * g : 0.0f;
    const float Q = p.t_lse || S == 0.0f ? S : 1.0f;
    float kt = 0.0f, k1 = 0.0f;
    if (has_kd) kt = sums ? __fdividef(kq * Q, st) : kq * Q * expf(ref * p.inv_t - p.lse[row]);
    if (has_ce) k1 = sums ? __fdividef(c1, p.grad_kind == ONE ? st : s1) : c1 * expf(ref - p.lse[p.rows + row]);
    if (p.grad_kind == ONE) { kt += k1; k1 = 0.0f; }  // temperature 1: one exponential for both terms
#pragma unroll 1
    for (int v0 = tid; v0 < s.hi; v0 += DF_FLIGHT * DF_THREADS) {
      uint4 raw[DF_FLIGHT];
      load_vectors<T>(s, v0, DF_THREADS, raw);
      with_exp<T>(p.grad_kind, ref, p.inv_t, [&](const auto& ex) {
        using Ex = std::remove_cv_t<std::remove_reference_t<decltype(ex)>>;
        const float mt = kt * Ex::scale_t, m1 = k1 * Ex::scale_1;
#pragma unroll
        for (int q = 0; q < DF_FLIGHT; ++q) {
          const int v = v0 + q * DF_THREADS;
          if (v >= s.hi) break;
          float d[V];
          unpack_vec<T>(raw[q], d);
#pragma unroll
          for (int c = 0; c < V; c += 2) {
            float et[2], e1[2];
            ex.both(d[c], d[c + 1], et, e1);
            fmul2(d[c], d[c + 1], et[0], et[1], mt, mt);
            if constexpr (Ex::BOTH) ffma2(d[c], d[c + 1], e1[0], e1[1], m1, m1, d[c], d[c + 1]);
          }
          const int at = s.first(v);
          if (v >= w0 && v < w1) {
            if (ACC && acc) {
              float o[V];
              ld16(dr + at, o);
#pragma unroll
              for (int c = 0; c < V; ++c) d[c] += o[c];
            }
            st16(dr + at, d);
          } else {
#pragma unroll
            for (int c = 0; c < V; ++c)
              if (at + c >= 0 && at + c < n) {
                if (ACC && acc) d[c] += to_f32(dr[at + c]);
                dr[at + c] = from_f32<T>(d[c]);
              }
          }
        }
      });
    }
    if (again) {  // sums over equal ids, in the order of the entries, so that they are the same every time
      for (int j = tid; j < k; j += DF_THREADS)
        if (e.w[j] != -1.0f) {
          float w = 0.0f;
          for (int c = 0; c < k; ++c)
            if (e.id[c] == e.id[j]) w += expf(e.t[c] - tref);
          e.w[j] = w;
        }
    }
    // the target is one of the ids
    bool met = false;
    for (int j = tid; j < k; j += DF_THREADS) met |= y >= 0 && e.id[j] == y;
    met = __syncthreads_or(met);  // and all of the row is written: the entries with a term of their own come last
    const float inv_s = p.t_lse || S == 0.0f ? 1.0f : 1.0f / S;
    for (int j = tid; j <= k; j += DF_THREADS) {
      const int id = e.id[j];
      const float w = j < k ? e.w[j] : 0.0f;
      if (id < 0 || w == -1.0f || (j == k && (met || !has_ce))) continue;
      const float x = e.x[j] - ref;
      float d = kt * expf(x * p.inv_t);
      if (k1 != 0.0f) d += k1 * expf(x);
      if (has_kd) d -= kq * w * inv_s;
      if (id == y) d -= c1;
      if (ACC && acc) d += e.o[j];
      dr[id] = from_f32<T>(d);
    }
  }
}

// Rows that sums_again() names, in a function of their own: inside the gradient's kernel they cost its other rows 2 %
// (16384 x 32000 bf16: 388 us against 381)
template <typename T, int DF_THREADS>
__device__ __noinline__ void distill_stream_row_again(const DistillParams& p) {
  distill_stream_row<T, DF_THREADS, DS_BWD, true>(p);
}

template <typename T, int DF_THREADS, int MODE>
__global__ void __launch_bounds__(DF_THREADS, DF_THREADS == 32 ? 32 : 1280 / DF_THREADS)
distill_stream_kernel(const __grid_constant__ DistillParams p) {
  if constexpr (MODE == DS_BWD) {
    if (sums_again(p.lse[blockIdx.x], p.lse[p.rows + blockIdx.x])) {
      distill_stream_row_again<T, DF_THREADS>(p);
      return;
    }
  }
  distill_stream_row<T, DF_THREADS, MODE, false>(p);
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
  // a row's gradient would go over the logits of another one
  if (bwd && p.dlogits == p.logits && p.ldd != p.ld && p.rows > 1)
    return bad(EISEN_ERR_INVALID, "dlogits over the logits needs their row stride");
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

// Which form.  Few rows (two per SM at most): staged, all of a CTA's threads and up to eight CTAs for each of them.  Loss and
// gradient together over rows of more than 16 KB: staged, so that the row is read once (4096 x 32000 bf16: 111 us against
// 146 read twice; 8192 x 4096: 80 against 54).  All else: not staged (the loss alone, 1023 x 100003 bf16: 57 us against 84).
template <typename T, int MODE>
int distill_launch(const char* what, DistillParams& p, cudaStream_t s) {
  const long long bytes = (long long)p.vocab * sizeof(T);
  auto shape = [&](int groups, int least) {
    p.shape = row_shape(p.rows, p.vocab, sizeof(T), groups * entry_bytes(p.k), std::max(2 * groups, 3), least);
    return p.shape.stages >= groups;
  };
  if (p.rows <= 2LL * sm_count() && shape(1, 8192))
    return launch_pipe<distill_pipe_kernel<T, 512, 1, MODE>>(what, p.shape, p.rows, pipe_threads(512, 1), s, p);
  if constexpr (MODE == (DS_FWD | DS_BWD)) {
    if (bytes > 16384 && shape(2, 1 << 30))
      return launch_pipe<distill_pipe_kernel<T, 256, 2, MODE>>(what, p.shape, p.rows, pipe_threads(256, 2), s, p);
    if (bytes > 16384 && shape(1, 1 << 30))  // one row at a time in a CTA
      return launch_pipe<distill_pipe_kernel<T, 512, 1, MODE>>(what, p.shape, p.rows, pipe_threads(512, 1), s, p);
  }
  const int smem = stream_bytes(p.k);
  if (bytes <= 8192) distill_stream_kernel<T, 32, MODE><<<(unsigned)p.rows, 32, smem, s>>>(p);
  else if (sizeof(T) == 2 || bytes <= 65536) distill_stream_kernel<T, 128, MODE><<<(unsigned)p.rows, 128, smem, s>>>(p);
  else distill_stream_kernel<T, 256, MODE><<<(unsigned)p.rows, 256, smem, s>>>(p);
  return check_launch(what);
}

int distill_run(const char* what, int mode, DistillParams& p, int dtype, cudaStream_t s) {
  p.fault_word = fault_word();
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
