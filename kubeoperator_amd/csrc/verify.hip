// Verification of drafted tokens for gfx950 (speculative decoding), from given uniform numbers.
//
//   target [B, T+1, V], draft [B, T, V] logits (bf16 or fp32, rows of unit stride); tokens [B, T] int64; u [B, T+1] fp32
//   p_t = softmax(target_t / temp), q_t = softmax(draft_t / temp)
//   token x_t is accepted while u_t q_t(x_t) < p_t(x_t). At the first refusal j (or j = n_draft, all accepted) one more
//   token comes from r = max(p_j - q_j, 0) (r = p_j where j = n_draft or where the difference is 0 everywhere): the
//   smallest i with r_i > 0 and r_0 + .. + r_i > u_T (r_0 + .. + r_{V-1}).
//   temp = 0: a token is accepted while it is the row's argmax (lowest index), and the next one is the argmax.
//
// Probabilities and their sums are held in 64 bits: u_T falls between two of up to 128k running sums, and sums in 32 bits
// would move a noticeable share of those borders past it. A logit of -inf or NaN has probability 0; +inf counts as the
// largest finite value. A row without any probability accepts nothing and yields -1.
//
// Three launches: per-chunk maximum and sum of every row (the only pass over all logits); acceptance and the chunk sums of
// r (the two rows of each sequence's refusal, again); the pick inside the one chunk that u_T falls into. Every
// workgroup that needs the acceptance re-derives it from the chunk statistics (a few hundred numbers): no atomics, no
// order-dependent sums.
#include <float.h>

#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kT = 256;       // threads of a workgroup
constexpr int kMaxRows = 2 * kVerifyMaxDraft + 1;

template <typename E>
__device__ __forceinline__ float ld1(const E* p);
template <>
__device__ __forceinline__ float ld1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float ld1<bf16_t>(const bf16_t* p) { return bf2f(*p); }

// NaN -> -inf (no probability), +inf -> the largest finite value
__device__ __forceinline__ float clean(float z) { return z != z ? -INFINITY : fminf(z, FLT_MAX); }

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// e^((z - m) / temp) in 64 bits; 0 for z = -inf
__device__ __forceinline__ double weight(float z, float m, double inv_temp) {
  return z == -INFINITY ? 0.0 : exp(((double)z - (double)m) * inv_temp);
}

struct Args {
  const void* target;
  const void* draft;
  int64_t ts_b, ts_t, ds_b, ds_t;  // strides of the sequence and token axes (elements)
  const int64_t* tokens;
  const float* u;
  const int* n_draft;  // null: T
  int B, T, V, nch, chunk;
  double inv_temp;  // 0: greedy
  float* pm;        // [B, 2T+1, nch] chunk maximum (rows 0..T target, T+1..2T draft)
  double* ps;       // [B, 2T+1, nch] sum of weights relative to the chunk maximum; greedy: the argmax's index
  double* pr;       // [B, nch] chunk sums of r
  int64_t* out;     // [B, T+1]
  int* accepted;    // [B]
};
__device__ __forceinline__ int drafts(const Args& a, int b) {
  return a.n_draft ? min(max(a.n_draft[b], 0), a.T) : a.T;
}
template <typename E>
__device__ __forceinline__ const E* row_ptr(const Args& a, int b, int r) {
  return r <= a.T ? reinterpret_cast<const E*>(a.target) + b * a.ts_b + r * a.ts_t
                  : reinterpret_cast<const E*>(a.draft) + b * a.ds_b + (int64_t)(r - a.T - 1) * a.ds_t;
}

// ---- pass 1: grid (chunks, rows, B); greedy needs the target's T+1 rows only
template <typename E>
__global__ void __launch_bounds__(kT) verify_stats_kernel(Args a) {
  __shared__ float s_m[kT / 64];
  __shared__ int s_i[kT / 64];
  __shared__ double s_s[kT / 64];
  const int c = blockIdx.x, r = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  const int nd = drafts(a, b);
  if (r <= a.T ? r > nd : r - a.T - 1 >= nd) return;  // a row that no drafted token of this sequence needs
  const E* x = row_ptr<E>(a, b, r);
  const int lo = c * a.chunk, hi = min(a.V, lo + a.chunk);
  float m = -INFINITY;
  int at = 0x7fffffff;
  for (int i = lo + t; i < hi; i += kT) {
    const float z = clean(ld1(x + i));
    if (z > m) {
      m = z;
      at = i;
    }
  }
  // the workgroup's maximum, at its lowest index
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float om = __shfl_xor(m, o, 64);
    const int oi = __shfl_xor(at, o, 64);
    if (om > m || (om == m && oi < at)) {
      m = om;
      at = oi;
    }
  }
  if ((t & 63) == 0) {
    s_m[t >> 6] = m;
    s_i[t >> 6] = at;
  }
  __syncthreads();
  m = s_m[0];
  at = s_i[0];
#pragma unroll
  for (int w = 1; w < kT / 64; ++w)
    if (s_m[w] > m || (s_m[w] == m && s_i[w] < at)) {
      m = s_m[w];
      at = s_i[w];
    }
  const int64_t o = ((int64_t)b * (2 * a.T + 1) + r) * a.nch + c;
  if (a.inv_temp == 0.0) {
    if (t == 0) {
      a.pm[o] = m;
      a.ps[o] = m == -INFINITY ? -1.0 : (double)at;
    }
    return;
  }
  double s = 0.0;
  if (m > -INFINITY)
    for (int i = lo + t; i < hi; i += kT) s += weight(clean(ld1(x + i)), m, a.inv_temp);
  s = wave_sum_d(s);
  if ((t & 63) == 0) s_s[t >> 6] = s;
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < kT / 64; ++w) s += s_s[w];
    a.pm[o] = m;
    a.ps[o] = s;
  }
}

// The chunk statistics of sequence b's rows folded to one (maximum, sum) per row -- greedy: (maximum, argmax) -- and the
// number of accepted tokens, in every thread. Called by whole workgroups.
template <typename E>
__device__ int decide(const Args& a, int b, float* s_m, double* s_s) {
  const int t = threadIdx.x, wv = t >> 6, lane = t & 63;
  const int nd = drafts(a, b), rows = 2 * a.T + 1;
  for (int r = wv; r < (a.inv_temp == 0.0 ? a.T + 1 : rows); r += kT / 64) {
    if (r <= a.T ? r > nd : r - a.T - 1 >= nd) continue;
    const int64_t o = ((int64_t)b * rows + r) * a.nch;
    float m = -INFINITY;
    for (int c = lane; c < a.nch; c += 64) m = fmaxf(m, a.pm[o + c]);
    m = wave_max(m);
    double s = 0.0;
    if (a.inv_temp == 0.0) {
      double at = 2147483647.0;  // the lowest index among the chunks that hold the maximum
      for (int c = lane; c < a.nch; c += 64)
        if (m > -INFINITY && a.pm[o + c] == m) at = fmin(at, a.ps[o + c]);
#pragma unroll
      for (int k = 32; k > 0; k >>= 1) at = fmin(at, __shfl_xor(at, k, 64));
      s = m > -INFINITY ? at : -1.0;
    } else {
      for (int c = lane; c < a.nch; c += 64)
        if (a.pm[o + c] > -INFINITY) s += a.ps[o + c] * weight(a.pm[o + c], m, a.inv_temp);
      s = wave_sum_d(s);
    }
    if (lane == 0) {
      s_m[r] = m;
      s_s[r] = s;
    }
  }
  __syncthreads();
  int j = 0;
  for (; j < nd; ++j) {
    const int64_t x = a.tokens[(int64_t)b * a.T + j];
    if (x < 0 || x >= a.V) break;
    if (a.inv_temp == 0.0) {
      if (s_s[j] != (double)x) break;
      continue;
    }
    const double zp = s_s[j], zq = s_s[a.T + 1 + j];
    const double p = zp > 0.0 ? weight(clean(ld1(row_ptr<E>(a, b, j) + x)), s_m[j], a.inv_temp) / zp : 0.0;
    const double q =
        zq > 0.0 ? weight(clean(ld1(row_ptr<E>(a, b, a.T + 1 + j) + x)), s_m[a.T + 1 + j], a.inv_temp) / zq : 0.0;
    if (!((double)a.u[(int64_t)b * (a.T + 1) + j] * q < p)) break;
  }
  return j;
}

// r_i at the refused (or last) position: both rows' normalisers from decide()
template <typename E>
struct Rest {
  const E *x, *y;  // y null: r = p
  float mp, mq;
  double ip, iq, inv_temp;  // 1 / sum, 0 where the row has no probability
  __device__ __forceinline__ double p(int i) const { return weight(clean(ld1(x + i)), mp, inv_temp) * ip; }
  __device__ __forceinline__ double r(int i) const {
    const double v = p(i);
    return y ? fmax(v - weight(clean(ld1(y + i)), mq, inv_temp) * iq, 0.0) : v;
  }
};
template <typename E>
__device__ Rest<E> rest_of(const Args& a, int b, int j, int nd, const float* s_m, const double* s_s) {
  Rest<E> f;
  f.x = row_ptr<E>(a, b, j);
  f.mp = s_m[j];
  f.ip = s_s[j] > 0.0 ? 1.0 / s_s[j] : 0.0;
  f.inv_temp = a.inv_temp;
  const int k = a.T + 1 + j;
  f.y = j < nd && s_s[k] > 0.0 ? row_ptr<E>(a, b, k) : nullptr;
  f.mq = f.y ? s_m[k] : 0.f;
  f.iq = f.y ? 1.0 / s_s[k] : 0.0;
  return f;
}

// ---- pass 2 (not greedy): grid (chunks, B), chunk sums of r
template <typename E>
__global__ void __launch_bounds__(kT) verify_rest_kernel(Args a) {
  __shared__ float s_m[kMaxRows];
  __shared__ double s_s[kMaxRows], s_w[kT / 64];
  const int c = blockIdx.x, b = blockIdx.y, t = threadIdx.x;
  const int j = decide<E>(a, b, s_m, s_s);
  const Rest<E> f = rest_of<E>(a, b, j, drafts(a, b), s_m, s_s);
  const int lo = c * a.chunk, hi = min(a.V, lo + a.chunk);
  double s = 0.0;
  for (int i = lo + t; i < hi; i += kT) s += f.r(i);
  s = wave_sum_d(s);
  if ((t & 63) == 0) s_w[t >> 6] = s;
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < kT / 64; ++w) s += s_w[w];
    a.pr[(int64_t)b * a.nch + c] = s;
  }
}

// the first index of [lo, hi) whose running sum (from `before`) passes `want`, else the last one with r > 0, else -1;
// in every thread. Thread t owns a run of consecutive indexes, so the order is that of the indexes.
template <typename F>
__device__ int pick(F r, int lo, int hi, double before, double want, double* s_w, int* s_i) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  const int per = (hi - lo + kT - 1) / kT, i0 = lo + t * per, i1 = min(hi, i0 + per);
  double mine = 0.0;
  for (int i = i0; i < i1; ++i) mine += r(i);
  double inc = mine;  // inclusive sum over the wave's lanes
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double v = __shfl_up(inc, o, 64);
    if (lane >= o) inc += v;
  }
  if (lane == 63) s_w[wv] = inc;
  if (t == 0) {
    s_i[0] = 0x7fffffff;
    s_i[1] = -1;
  }
  __syncthreads();
  double run = before;
  for (int w = 0; w < wv; ++w) run += s_w[w];
  run += inc - mine;
  int hit = 0x7fffffff, last = -1;
  for (int i = i0; i < i1; ++i) {
    const double v = r(i);
    run += v;
    if (v > 0.0) {
      last = i;
      if (hit == 0x7fffffff && run > want) hit = i;
    }
  }
  atomicMin(&s_i[0], hit);  // minimum / maximum: no order
  atomicMax(&s_i[1], last);
  __syncthreads();
  return s_i[0] != 0x7fffffff ? s_i[0] : s_i[1];
}

// ---- pass 3: grid B
template <typename E>
__global__ void __launch_bounds__(kT) verify_pick_kernel(Args a) {
  __shared__ float s_m[kMaxRows];
  __shared__ double s_s[kMaxRows], s_w[kT / 64];
  __shared__ int s_i[2];
  const int b = blockIdx.x, t = threadIdx.x;
  const int j = decide<E>(a, b, s_m, s_s);
  int64_t next = -1;
  if (a.inv_temp == 0.0) {
    next = (int64_t)s_s[j];
  } else {
    const Rest<E> f = rest_of<E>(a, b, j, drafts(a, b), s_m, s_s);
    const double* pr = a.pr + (int64_t)b * a.nch;
    double total = 0.0;
    for (int c = 0; c < a.nch; ++c) total += pr[c];
    const bool none = !(total > 0.0);  // r = 0 everywhere: the target's own distribution
    if (none) total = f.ip > 0.0 ? 1.0 : 0.0;
    if (total > 0.0) {
      const double want = (double)a.u[(int64_t)b * (a.T + 1) + a.T] * total;
      // the chunk that `want` falls into; past the last sum (u >= 1, rounding): the last chunk with anything in it
      const int64_t o = ((int64_t)b * (2 * a.T + 1) + j) * a.nch;
      double run = 0.0, before = 0.0;
      int at = -1;
      for (int c = 0; c < a.nch; ++c) {
        const double v = none ? a.ps[o + c] * weight(a.pm[o + c], f.mp, a.inv_temp) * f.ip : pr[c];
        if (v > 0.0) {
          at = c;
          before = run;
          run += v;
          if (run > want) break;
        }
      }
      const int lo = at * a.chunk, hi = min(a.V, lo + a.chunk);
      next = none ? pick([&](int i) { return f.p(i); }, lo, hi, before, want, s_w, s_i)
                  : pick([&](int i) { return f.r(i); }, lo, hi, before, want, s_w, s_i);
    }
  }
  for (int i = t; i <= a.T; i += kT)
    a.out[(int64_t)b * (a.T + 1) + i] = i < j ? a.tokens[(int64_t)b * a.T + i] : i == j ? next : -1;
  if (t == 0) a.accepted[b] = j;
}

template <typename E>
int launch(const Args& a, hipStream_t stream) {
  verify_stats_kernel<E><<<dim3(a.nch, a.inv_temp == 0.0 ? a.T + 1 : 2 * a.T + 1, a.B), kT, 0, stream>>>(a);
  if (a.inv_temp != 0.0) verify_rest_kernel<E><<<dim3(a.nch, a.B), kT, 0, stream>>>(a);
  verify_pick_kernel<E><<<a.B, kT, 0, stream>>>(a);
  return hipGetLastError() == hipSuccess ? 0 : -9;
}
}  // namespace

static constexpr int kChunk = 8192;
int64_t verify_draft_workspace(int B, int T, int V) {
  const int64_t nch = (V + kChunk - 1) / kChunk, rows = (int64_t)B * (2 * T + 1);
  return rows * nch * (8 + 4) + (int64_t)B * nch * 8;
}

int verify_draft(const void* target, int64_t ts_b, int64_t ts_t, const void* draft, int64_t ds_b, int64_t ds_t, bool f32,
                 const int64_t* tokens, const float* u, const int* n_draft, int B, int T, int V, double temp,
                 void* workspace, int64_t* out, int* accepted, hipStream_t stream) {
  if (B < 0 || B > 65535 || T < 0 || T > kVerifyMaxDraft || V < 1 || !(temp >= 0.0)) return -1;
  if (B == 0) return 0;
  Args a;
  a.target = target, a.draft = draft;
  a.ts_b = ts_b, a.ts_t = ts_t, a.ds_b = ds_b, a.ds_t = ds_t;
  a.tokens = tokens, a.u = u, a.n_draft = n_draft;
  a.B = B, a.T = T, a.V = V;
  a.chunk = kChunk, a.nch = (V + kChunk - 1) / kChunk;
  a.inv_temp = temp > 0.0 ? 1.0 / temp : 0.0;
  const int64_t n = (int64_t)B * (2 * T + 1) * a.nch;
  a.ps = reinterpret_cast<double*>(workspace);
  a.pr = a.ps + n;
  a.pm = reinterpret_cast<float*>(a.pr + (int64_t)B * a.nch);
  a.out = out, a.accepted = accepted;
  return f32 ? launch<float>(a, stream) : launch<bf16_t>(a, stream);
}

}  // namespace kop
