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
// Three launches (greedy: two): maximum and sum of every 8192-logit chunk (the only pass over all logits, each held in
// registers between its maximum and its sum); acceptance and the sums of r over 1024-logit pieces (the two rows of each
// sequence's refusal, again); the pick inside the one piece that u_T falls into. A workgroup that needs the acceptance
// re-derives it from the chunk statistics (a few hundred numbers): no atomics, no order-dependent sums.
#include <float.h>

#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kT = 256;       // threads of a workgroup
constexpr int kChunk = 8192;  // logits per workgroup of the first pass: 32 per thread
constexpr int kPiece = 1024;  // logits per wave of the second pass, per workgroup of the third
constexpr int kMaxRows = 2 * kVerifyMaxDraft + 1;

template <typename E>
__device__ __forceinline__ float ld1(const E* p);
template <>
__device__ __forceinline__ float ld1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float ld1<bf16_t>(const bf16_t* p) { return bf2f(*p); }

// 16 bytes of a row; rows of odd length start off the 16-byte grid (global loads take any element's alignment)
template <typename E>
struct Vec {
  static constexpr int N = 16 / sizeof(E);
  struct __attribute__((packed, aligned(sizeof(E)))) U {
    u32x4 v;
  };
  u32x4 w;
  // logits [i, i + N) of x, -inf at and past `end`
  __device__ __forceinline__ void load(const E* x, int i, int end) {
    if (i + N <= end) {
      w = reinterpret_cast<const U*>(x + i)->v;
      return;
    }
    constexpr uint32_t pad = sizeof(E) == 4 ? 0xff800000u : 0xff80ff80u;
    w = u32x4{pad, pad, pad, pad};
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k < end) {
        if constexpr (sizeof(E) == 4) w[k] = __float_as_uint(x[i + k]);
        else w[k >> 1] = (k & 1) ? (w[k >> 1] & 0xffffu) | ((uint32_t)x[i + k] << 16) : (w[k >> 1] & 0xffff0000u) | x[i + k];
      }
  }
  __device__ __forceinline__ float get(int k) const {
    if constexpr (sizeof(E) == 4) return __uint_as_float(w[k]);
    else return __uint_as_float((k & 1) ? w[k >> 1] & 0xffff0000u : w[k >> 1] << 16);
  }
};

// 2^x for x <= 0 in 64 bits: 2^n times a degree-9 polynomial of the fraction (Chebyshev interpolation of 2^f on
// [-1/2, 1/2], 2e-14 relative). NaN and everything below -1100 give 0, everything above 0 gives 1 -- which is what logits of
// NaN, -inf and +inf are to weigh. (Rounding by adding 1.5 * 2^52 and writing n into the exponent, with a select for the zeros,
// measured slower: 65 against 61 us for the first pass over 64 x 9 rows of 128256.)
__device__ __forceinline__ double exp2_neg(double x) {
  x = fmin(fmax(x, -1100.0), 0.0);
  const double n = rint(x), f = x - n;
  double y = 0x1.b6557c7da8ca4p-24;
  y = fma(y, f, 0x1.63efd536dcb25p-20);
  y = fma(y, f, 0x1.ffcb7a04d3b13p-17);
  y = fma(y, f, 0x1.43088df6dd4a7p-13);
  y = fma(y, f, 0x1.5d87fe8e6c4b1p-10);
  y = fma(y, f, 0x1.3b2ab72b2b245p-7);
  y = fma(y, f, 0x1.c6b08d7045e60p-5);
  y = fma(y, f, 0x1.ebfbdff814945p-3);
  y = fma(y, f, 0x1.62e42fefa39e9p-1);
  y = fma(y, f, 0x1.000000000003dp+0);
  return __builtin_amdgcn_ldexp(y, (int)n);
}
// e^((z - m) / temp) for z <= m, c = log2 e / temp. The difference of two fp32 values is exact in 64 bits, or far below 2^-1100
__device__ __forceinline__ double weight(float z, float m, double c) { return exp2_neg(((double)z - (double)m) * c); }

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct Head;
struct Args {
  const void* target;
  const void* draft;
  int64_t ts_b, ts_t, ds_b, ds_t;  // strides of the sequence and token axes (elements)
  const int64_t* tokens;
  const float* u;
  const int* n_draft;  // null: T
  int B, T, V, nch, npc;  // chunks and pieces of a row
  double c;               // log2 e / temp
  double* ps;             // [B, 2T+1, nch] sums relative to the chunk's maximum; greedy: the argmax's index
  double* pr;             // [B, npc] sums of r
  float* pm;              // [B, 2T+1, nch] maxima (rows 0..T target, T+1..2T draft); -inf: an empty chunk
  Head* head;      // [B] the refused position and its rows' normalisers, from pass 2 to pass 3
  int64_t* out;           // [B, T+1]
  int* accepted;          // [B]
};
struct Head {
  double ip, iq;  // 1 / sum of the target's / the draft's row, 0 where it has no probability or is not needed
  float mp, mq;   // maxima
  int j, two;     // accepted tokens; whether the draft's row is needed
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
template <typename E, bool GREEDY>
__global__ void __launch_bounds__(kT) verify_stats_kernel(Args a) {
  constexpr int N = Vec<E>::N, NV = kChunk / (kT * N);
  __shared__ float s_m[kT / 64];
  __shared__ double s_s[kT / 64];
  const int c = blockIdx.x, r = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  const int nd = drafts(a, b);
  if (r <= a.T ? r > nd : r - a.T - 1 >= nd) return;  // a row that no drafted token of this sequence needs
  const E* x = row_ptr<E>(a, b, r);
  const int lo = c * kChunk, hi = min(a.V, lo + kChunk);
  Vec<E> v[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k].load(x, lo + (k * kT + t) * N, hi);
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, v[k].get(e));  // a NaN is passed over
  const float mine = m;
  m = wave_max(m);
  if ((t & 63) == 0) s_m[t >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const int64_t o = ((int64_t)b * (2 * a.T + 1) + r) * a.nch + c;
  if constexpr (GREEDY) {
    int at = 0x7fffffff;  // the lowest index that holds the maximum
    if (mine == m && m > -INFINITY) {
#pragma unroll
      for (int k = NV - 1; k >= 0; --k)
#pragma unroll
        for (int e = N - 1; e >= 0; --e)
          if (v[k].get(e) == m) at = lo + (k * kT + t) * N + e;
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) at = min(at, __shfl_xor(at, k, 64));
    if ((t & 63) == 0) s_s[t >> 6] = (double)at;
    __syncthreads();
    if (t == 0) {
      a.pm[o] = fminf(m, FLT_MAX);
      a.ps[o] = fmin(fmin(s_s[0], s_s[1]), fmin(s_s[2], s_s[3]));
    }
  } else {
    m = fminf(m, FLT_MAX);
    double s = 0.0;
    if (m > -INFINITY) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) s += weight(v[k].get(e), m, a.c);
    }
    s = wave_sum_d(s);
    if ((t & 63) == 0) s_s[t >> 6] = s;
    __syncthreads();
    if (t == 0) {
      a.pm[o] = m;
      a.ps[o] = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
    }
  }
}

// Called by whole workgroups: the chunk statistics of sequence b's rows folded to one (maximum, sum) per row -- greedy:
// (maximum, argmax or -1) -- by 16 lanes a row; returns the number of accepted tokens (one lane a token) in every thread.
template <typename E, bool GREEDY>
__device__ int decide(const Args& a, int b, float* s_m, double* s_s, int* s_j) {
  const int t = threadIdx.x, sub = t & 15;
  const int nd = drafts(a, b), rows = 2 * a.T + 1;
  // the drafted tokens' own logits, on their way while the statistics are folded
  int64_t x = -1;
  float lp = 0.f, lq = 0.f, u = 0.f;
  if (t < nd) {
    x = a.tokens[(int64_t)b * a.T + t];
    if (!GREEDY && x >= 0 && x < a.V) {
      lp = ld1(row_ptr<E>(a, b, t) + x);
      lq = ld1(row_ptr<E>(a, b, a.T + 1 + t) + x);
      u = a.u[(int64_t)b * (a.T + 1) + t];
    }
  }
  for (int r = t >> 4; r < (GREEDY ? a.T + 1 : rows); r += kT / 16) {
    if (r <= a.T ? r > nd : r - a.T - 1 >= nd) continue;
    const int64_t o = ((int64_t)b * rows + r) * a.nch;
    float m = -INFINITY;
    for (int c = sub; c < a.nch; c += 16) m = fmaxf(m, a.pm[o + c]);
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 16));
    double s = GREEDY ? 2147483647.0 : 0.0;
    for (int c = sub; c < a.nch; c += 16) {
      const float cm = a.pm[o + c];
      const double cs = a.ps[o + c];
      if (cm == -INFINITY) continue;
      if constexpr (GREEDY) s = cm == m ? fmin(s, cs) : s;
      else s += cs * weight(cm, m, a.c);
    }
#pragma unroll
    for (int k = 8; k > 0; k >>= 1) {
      const double v = __shfl_xor(s, k, 16);
      s = GREEDY ? fmin(s, v) : s + v;
    }
    if (sub == 0) {
      s_m[r] = m;
      s_s[r] = GREEDY && m == -INFINITY ? -1.0 : s;
    }
  }
  __syncthreads();
  if (t < 64) {
    bool ok = false;
    if (t < nd) {
      if (x >= 0 && x < a.V) {
        if constexpr (GREEDY) {
          ok = s_s[t] == (double)x;
        } else {
          const double zp = s_s[t], zq = s_s[a.T + 1 + t];
          const double p = zp > 0.0 ? weight(lp, s_m[t], a.c) / zp : 0.0;
          const double q = zq > 0.0 ? weight(lq, s_m[a.T + 1 + t], a.c) / zq : 0.0;
          ok = (double)u * q < p;
        }
      }
    }
    const uint64_t no = ~__ballot(ok);  // lanes past the drafts refuse
    if (t == 0) s_j[0] = __builtin_ctzll(no);
  }
  __syncthreads();
  return s_j[0];
}

// r_i at the refused (or last) position
template <typename E>
struct Rest {
  const E *x, *y;  // y null: r = p
  float mp, mq;
  double ip, iq, c;
  __device__ __forceinline__ Rest(const Args& a, int b, const Head& h)
      : x(row_ptr<E>(a, b, h.j)), y(h.two ? row_ptr<E>(a, b, a.T + 1 + h.j) : nullptr), mp(h.mp), mq(h.mq), ip(h.ip),
        iq(h.iq), c(a.c) {}
  __device__ __forceinline__ double p(float z) const { return weight(z, mp, c) * ip; }
  __device__ __forceinline__ double r(float z, float d) const {
    const double v = p(z);
    return y ? fmax(v - weight(d, mq, c) * iq, 0.0) : v;
  }
};
__device__ __forceinline__ Head head_of(const Args& a, int b, int j, const float* s_m, const double* s_s) {
  Head h;
  h.j = j;
  h.mp = s_m[j];
  h.ip = s_s[j] > 0.0 ? 1.0 / s_s[j] : 0.0;
  const int k = a.T + 1 + j;
  h.two = j < drafts(a, b) && s_s[k] > 0.0;
  h.mq = h.two ? s_m[k] : 0.f;
  h.iq = h.two ? 1.0 / s_s[k] : 0.0;
  return h;
}

// ---- pass 2 (not greedy): grid (pieces / 4, B), a wave per piece
template <typename E>
__global__ void __launch_bounds__(kT) verify_rest_kernel(Args a) {
  constexpr int N = Vec<E>::N, NV = kPiece / (64 * N);
  __shared__ float s_m[kMaxRows];
  __shared__ double s_s[kMaxRows];
  __shared__ int s_j[1];
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const int pc = blockIdx.x * (kT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = decide<E, false>(a, b, s_m, s_s, s_j);
  const Head h = head_of(a, b, j, s_m, s_s);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.head[b] = h;
  if (pc >= a.npc) return;
  const Rest<E> f(a, b, h);
  const int lo = pc * kPiece, hi = min(a.V, lo + kPiece);
  Vec<E> v[NV], d[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k].load(f.x, lo + (k * 64 + lane) * N, hi);
  if (f.y) {
#pragma unroll
    for (int k = 0; k < NV; ++k) d[k].load(f.y, lo + (k * 64 + lane) * N, hi);
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) d[k].w = u32x4{0u, 0u, 0u, 0u};
  }
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) s += f.r(v[k].get(e), d[k].get(e));
  s = wave_sum_d(s);
  if (lane == 0) a.pr[(int64_t)b * a.npc + pc] = s;
}

// inclusive sum over the workgroup's threads in order; every thread also gets the total
__device__ __forceinline__ double block_scan(double v, double* s_w, double& total) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double w = __shfl_up(v, o, 64);
    if (lane >= o) v += w;
  }
  __syncthreads();  // s_w may still be read
  if (lane == 63) s_w[wv] = v;
  __syncthreads();
  total = 0.0;
#pragma unroll
  for (int w = 0; w < kT / 64; ++w) {
    v += w < wv ? s_w[w] : 0.0;
    total += s_w[w];
  }
  return v;
}
// the lowest `i` of any thread (0x7fffffff: none), in every thread
__device__ __forceinline__ int block_min(int i, int* s_w) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) i = min(i, __shfl_xor(i, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_w[threadIdx.x >> 6] = i;
  __syncthreads();
  return min(min(s_w[0], s_w[1]), min(s_w[2], s_w[3]));
}

// ---- pass 3: grid B
template <typename E, bool GREEDY>
__global__ void __launch_bounds__(kT) verify_pick_kernel(Args a) {
  __shared__ double s_w[kT / 64];
  __shared__ int s_i[kT / 64];
  const int b = blockIdx.x, t = threadIdx.x;
  int j;
  int64_t next = -1;
  if constexpr (GREEDY) {
    __shared__ float s_m[kMaxRows];
    __shared__ double s_s[kMaxRows];
    j = decide<E, true>(a, b, s_m, s_s, s_i);
    next = (int64_t)s_s[j];
  } else {
    constexpr int PER = kPiece / kT;  // consecutive logits of a thread
    const Head h = a.head[b];
    Rest<E> f(a, b, h);
    j = h.j;
    const double* pr = a.pr + (int64_t)b * a.npc;
    // runs over groups of kT pieces, the last run one past the pieces that hold the answer
    double total = 0.0, part;
    for (int g = 0; g < a.npc; g += kT) {
      block_scan(g + t < a.npc ? pr[g + t] : 0.0, s_w, part);
      total += part;
    }
    const bool none = !(total > 0.0);  // r = 0 everywhere: the target's own distribution, by its chunks
    if (none) {
      f.y = nullptr;
      total = f.ip > 0.0 ? 1.0 : 0.0;
    }
    if (total > 0.0) {
      const int64_t o = ((int64_t)b * (2 * a.T + 1) + j) * a.nch;
      const int n = none ? a.nch : a.npc, size = none ? kChunk : kPiece;
      const double want = (double)a.u[(int64_t)b * (a.T + 1) + a.T] * total;
      // the piece that `want` falls into; past the last sum (u >= 1, rounding): the last piece with anything in it
      double run = 0.0, before = 0.0;
      int at = 0x7fffffff, last = -1;
      double last_before = 0.0;
      for (int g = 0; g < n && at == 0x7fffffff; g += kT) {
        const int i = g + t;
        double v = 0.0;
        if (i < n) v = none ? a.ps[o + i] * weight(a.pm[o + i], f.mp, f.c) * f.ip : pr[i];
        if (none && i < n && a.pm[o + i] == -INFINITY) v = 0.0;
        const double inc = run + block_scan(v, s_w, part);
        at = block_min(i < n && v > 0.0 && inc > want ? i : 0x7fffffff, s_i);
        const int nz = block_min(v > 0.0 ? -i : 0x7fffffff, s_i);  // minus the group's last piece with anything in it
        const int pick = at != 0x7fffffff ? at : nz != 0x7fffffff ? -nz : -1;
        if (pick >= 0) {
          __syncthreads();
          if (i == pick) s_w[0] = inc - v;
          __syncthreads();
          last = pick;
          last_before = s_w[0];
          __syncthreads();
        }
        run += part;
      }
      before = last_before;
      // inside it: PER consecutive logits a thread, so that the order is that of the indexes
      int hit = 0x7fffffff, tail = -1;
      const int lo = last * size, hi = min(a.V, lo + size);
      for (int base = lo; base < hi && hit == 0x7fffffff; base += kPiece) {
        double v[PER], mine = 0.0;
        const int i0 = base + t * PER;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const bool in = i0 + e < hi;
          v[e] = in ? f.r(ld1(f.x + i0 + e), f.y ? ld1(f.y + i0 + e) : 0.f) : 0.0;
          mine += v[e];
        }
        const double inc = block_scan(mine, s_w, part);
        double at_e = before + (inc - mine);
        int h = 0x7fffffff, l = 0x7fffffff;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          at_e += v[e];
          if (v[e] > 0.0) {
            l = -(i0 + e);
            if (h == 0x7fffffff && at_e > want) h = i0 + e;
          }
        }
        hit = block_min(h, s_i);
        l = block_min(l, s_i);
        if (l != 0x7fffffff) tail = -l;
        before += part;
      }
      next = hit != 0x7fffffff ? hit : tail;
    }
  }
  for (int i = t; i <= a.T; i += kT)
    a.out[(int64_t)b * (a.T + 1) + i] = i < j ? a.tokens[(int64_t)b * a.T + i] : i == j ? next : -1;
  if (t == 0) a.accepted[b] = j;
}

template <typename E>
int launch(const Args& a, bool greedy, hipStream_t stream) {
  const dim3 rows(a.nch, greedy ? a.T + 1 : 2 * a.T + 1, a.B);
  if (greedy) {
    verify_stats_kernel<E, true><<<rows, kT, 0, stream>>>(a);
    verify_pick_kernel<E, true><<<a.B, kT, 0, stream>>>(a);
  } else {
    verify_stats_kernel<E, false><<<rows, kT, 0, stream>>>(a);
    verify_rest_kernel<E><<<dim3((a.npc + kT / 64 - 1) / (kT / 64), a.B), kT, 0, stream>>>(a);
    verify_pick_kernel<E, false><<<a.B, kT, 0, stream>>>(a);
  }
  return hipGetLastError() == hipSuccess ? 0 : -9;
}
inline int64_t chunks(int V) { return (V + kChunk - 1) / kChunk; }
inline int64_t pieces(int V) { return (V + kPiece - 1) / kPiece; }
}  // namespace

int64_t verify_draft_workspace(int B, int T, int V) {
  return (int64_t)B * (2 * T + 1) * chunks(V) * (8 + 4) + (int64_t)B * (pieces(V) * 8 + sizeof(Head));
}

int verify_draft(const void* target, int64_t ts_b, int64_t ts_t, const void* draft, int64_t ds_b, int64_t ds_t, bool f32,
                 const int64_t* tokens, const float* u, const int* n_draft, int B, int T, int V, double temp,
                 void* workspace, int64_t* out, int* accepted, hipStream_t stream) {
  if (B < 0 || B > 65535 || T < 0 || T > kVerifyMaxDraft || V < 1 || V > 0x3fffffff || !(temp >= 0.0)) return -1;
  if (B == 0) return 0;
  Args a;
  a.target = target, a.draft = draft;
  a.ts_b = ts_b, a.ts_t = ts_t, a.ds_b = ds_b, a.ds_t = ds_t;
  a.tokens = tokens, a.u = u, a.n_draft = n_draft;
  a.B = B, a.T = T, a.V = V;
  a.nch = (int)chunks(V), a.npc = (int)pieces(V);
  a.c = temp > 0.0 ? 1.4426950408889634 / temp : 0.0;
  const int64_t n = (int64_t)B * (2 * T + 1) * a.nch;
  a.ps = reinterpret_cast<double*>(workspace);
  a.pr = a.ps + n;
  a.head = reinterpret_cast<Head*>(a.pr + (int64_t)B * a.npc);
  a.pm = reinterpret_cast<float*>(a.head + B);
  a.out = out, a.accepted = accepted;
  return f32 ? launch<float>(a, temp == 0.0, stream) : launch<bf16_t>(a, temp == 0.0, stream);
}

}  // namespace kop
