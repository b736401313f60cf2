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
// registers between its maximum and its sum); acceptance and the sums of r over small pieces (the two rows of each
// sequence's refusal, again); the pick inside the one piece that u_T falls into. A workgroup that needs the acceptance
// re-derives it from the chunk statistics (a few hundred numbers): no atomics, no order-dependent sums. Small problems, whose
// time is all launches, do the same in one: a workgroup per sequence.
//
// 64 sequences, 4 drafts, 128256 fp32 logits: 61 us for the first pass (295 MB, 4.9 TB/s, what a copy reaches; vector ALUs 73 %
// busy, and as long for bf16 logits, which are half the bytes), 20 for the second (128 rows again, mostly from cache; 16 million fp64
// exponentials), 5.2 for the pick. One sequence, 3 drafts, 50304 logits:
// 4.9 + 6.3 + 3.6 us, each a launch and its chain of loads. Joining the pick to the second pass (the sequence's last workgroup,
// told by a counter) costs more than the launch it saves: a fence for the whole device writes each XCD's L2 back (the two
// together 219 instead of 28 us for 64 sequences, 12.3 instead of 10.3 for one).
#include <float.h>

#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kT = 256;       // threads of a workgroup
constexpr int kChunk = 8192;  // logits per workgroup of the first pass: 32 per thread
// logits per sum of the second pass: what a wave reads with one access each
template <typename E>
constexpr int piece() { return 64 * 16 / (int)sizeof(E); }
constexpr int kPieces = 4;        // pieces per wave of the second pass
constexpr int kHeld = 16;           // pieces of a row per lane of the draw that are held in registers
// logits per row, and per sequence (sampling, greedy), up to which one launch does everything
constexpr int kOneRow = 4096, kOneLaunch = 16384, kOneGreedy = 24576;
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

// lane exchanges of 64-bit values in registers (a __shfl is two LDS round trips): DPP inside 16-lane rows, swaps across
template <int CTRL, bool ZERO = false>
__device__ __forceinline__ double dpp_d(double v) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, ZERO),
                          __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, ZERO));
}
// the sum over each 16-lane row / over the wave, in every lane
__device__ __forceinline__ double row_sum_d(double v) {
  v += dpp_d<0xB1>(v);
  v += dpp_d<0x4E>(v);
  v += dpp_d<0x141>(v);
  return v + dpp_d<0x140>(v);
}
__device__ __forceinline__ double row_min_d(double v) {
  v = fmin(v, dpp_d<0xB1>(v));
  v = fmin(v, dpp_d<0x4E>(v));
  v = fmin(v, dpp_d<0x141>(v));
  return fmin(v, dpp_d<0x140>(v));
}
__device__ __forceinline__ float row_max_f(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  return fmaxf(v, dpp_f32<0x140>(v));
}
__device__ __forceinline__ double readlane_d(double v, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane),
                          __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v = row_sum_d(v);
  return (readlane_d(v, 0) + readlane_d(v, 16)) + (readlane_d(v, 32) + readlane_d(v, 48));
}
// inclusive sum over the lanes in order
__device__ __forceinline__ double wave_scan_d(double v) {
  v += dpp_d<0x111, true>(v);  // row_shr 1, 2, 4, 8; zeros come in
  v += dpp_d<0x112, true>(v);
  v += dpp_d<0x114, true>(v);
  v += dpp_d<0x118, true>(v);
  const double a = readlane_d(v, 15), b = a + readlane_d(v, 31), c = b + readlane_d(v, 47);
  const int row = (threadIdx.x >> 4) & 3;
  return v + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? b : c);
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
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

// whether sequence b's row r is one that none of its drafted tokens needs
__device__ __forceinline__ bool idle(const Args& a, int r, int nd) { return r <= a.T ? r > nd : r - a.T - 1 >= nd; }

// ---- pass 1: grid (chunks, rows, B); greedy needs the target's T+1 rows only. Bound by memory: a chunk is loaded at once, 8
// (bf16: 4) 16-byte loads a thread, and its exponentials run while other workgroups load. Greedy, 32 x 8 rows of 128256 bf16
// logits: 12.9 us, 5.1 TB/s.
template <typename E, bool GREEDY>
__global__ void __launch_bounds__(kT) verify_stats_kernel(Args a) {
  constexpr int N = Vec<E>::N, NV = kChunk / (kT * N);
  __shared__ float s_m[kT / 64];
  __shared__ double s_s[kT / 64];
  const int c = blockIdx.x, r = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  if (idle(a, r, drafts(a, b))) return;
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
  m = fminf(fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), FLT_MAX);
  const int64_t o = ((int64_t)b * (2 * a.T + 1) + r) * a.nch + c;
  if constexpr (GREEDY) {
    int at = 0x7fffffff;  // the lowest index that holds the maximum, +inf being the largest finite value
    if (mine >= m && m > -INFINITY) {
#pragma unroll
      for (int k = NV - 1; k >= 0; --k)
#pragma unroll
        for (int e = N - 1; e >= 0; --e)
          if (v[k].get(e) >= m) at = lo + (k * kT + t) * N + e;
    }
    at = wave_min_i(at);
    if ((t & 63) == 0) s_s[t >> 6] = (double)at;
    __syncthreads();
    if (t == 0) {
      a.pm[o] = m;
      a.ps[o] = fmin(fmin(s_s[0], s_s[1]), fmin(s_s[2], s_s[3]));
    }
  } else {
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

// one drafted token's own logits, loaded before the rows' statistics are there
struct Drafted {
  int64_t x;
  float lp, lq, u;
};
template <typename E, bool GREEDY>
__device__ __forceinline__ Drafted drafted(const Args& a, int b, int nd) {
  const int t = threadIdx.x;
  Drafted d = {-1, 0.f, 0.f, 0.f};
  if (t < nd) {
    d.x = a.tokens[(int64_t)b * a.T + t];
    if (!GREEDY && d.x >= 0 && d.x < a.V) {
      d.lp = ld1(row_ptr<E>(a, b, t) + d.x);
      d.lq = ld1(row_ptr<E>(a, b, a.T + 1 + t) + d.x);
      d.u = a.u[(int64_t)b * (a.T + 1) + t];
    }
  }
  return d;
}
// The number of accepted tokens, one lane of the first wave a token, in every thread: s_m / s_s hold each row's (maximum, sum)
// -- greedy: (maximum, argmax or -1).
template <typename E, bool GREEDY>
__device__ __forceinline__ int accept(const Args& a, const Drafted& d, int nd, const float* s_m, const double* s_s, int* s_j) {
  const int t = threadIdx.x;
  if (t < 64) {
    bool ok = false;
    if (t < nd && d.x >= 0 && d.x < a.V) {
      if constexpr (GREEDY) {
        ok = s_s[t] == (double)d.x;
      } else {
        const double zp = s_s[t], zq = s_s[a.T + 1 + t];
        const double p = zp > 0.0 ? weight(d.lp, s_m[t], a.c) / zp : 0.0;
        const double q = zq > 0.0 ? weight(d.lq, s_m[a.T + 1 + t], a.c) / zq : 0.0;
        ok = (double)d.u * q < p;
      }
    }
    const uint64_t no = ~__ballot(ok);  // lanes past the drafts refuse
    if (t == 0) s_j[0] = __builtin_ctzll(no);
  }
  __syncthreads();
  return s_j[0];
}
// The same from the chunk statistics, folded to one (maximum, sum) per row by 16 lanes each. Called by whole workgroups.
template <typename E, bool GREEDY>
__device__ int decide(const Args& a, int b, float* s_m, double* s_s, int* s_j) {
  const int t = threadIdx.x, sub = t & 15;
  const int nd = drafts(a, b), rows = 2 * a.T + 1;
  const Drafted d = drafted<E, GREEDY>(a, b, nd);
  for (int r = t >> 4; r < (GREEDY ? a.T + 1 : rows); r += kT / 16) {
    if (idle(a, r, nd)) continue;
    const int64_t o = ((int64_t)b * rows + r) * a.nch;
    // the first 16 chunks' numbers in registers: most vocabularies have no more
    const float c0 = sub < a.nch ? a.pm[o + sub] : -INFINITY;
    const double s0 = sub < a.nch ? a.ps[o + sub] : 0.0;
    float m = c0;
    for (int c = sub + 16; c < a.nch; c += 16) m = fmaxf(m, a.pm[o + c]);
    m = row_max_f(m);
    double s = GREEDY ? 2147483647.0 : 0.0;
    auto fold = [&](float cm, double cs) {
      if (cm == -INFINITY) return;
      if constexpr (GREEDY) s = cm == m ? fmin(s, cs) : s;
      else s += cs * weight(cm, m, a.c);
    };
    fold(c0, s0);
    for (int c = sub + 16; c < a.nch; c += 16) fold(a.pm[o + c], a.ps[o + c]);
    s = GREEDY ? row_min_d(s) : row_sum_d(s);
    if (sub == 0) {
      s_m[r] = m;
      s_s[r] = GREEDY && m == -INFINITY ? -1.0 : s;
    }
  }
  __syncthreads();
  return accept<E, GREEDY>(a, d, nd, s_m, s_s, s_j);
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
  __device__ __forceinline__ double r(float z, float d) const {
    const double v = weight(z, mp, c) * ip;
    return y ? fmax(v - weight(d, mq, c) * iq, 0.0) : v;
  }
  // r of the lane's vector of piece pc (0 past the row's end)
  __device__ __forceinline__ void vec(int pc, int V, double* out) const {
    constexpr int N = Vec<E>::N;
    const int i = pc * piece<E>() + (threadIdx.x & 63) * N;
    Vec<E> v, d;
    v.load(x, i, V);
    if (y) d.load(y, i, V);
    else d.w = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = r(v.get(e), d.get(e));
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
// the sums of COUNT pieces from `pc` on into pr, by one wave
template <int COUNT, typename E>
__device__ __forceinline__ void piece_sums(const Args& a, const Rest<E>& f, int pc, double* pr) {
  constexpr int N = Vec<E>::N;
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    double v[N], s = 0.0;
    f.vec(pc + k, a.V, v);  // zeros past the last piece
#pragma unroll
    for (int e = 0; e < N; ++e) s += v[e];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0 && pc + k < a.npc) pr[pc + k] = s;
  }
}

// ---- pass 2 (not greedy): grid (pieces / (4 kPieces), B). A piece is what a wave reads at once, so that its sum is one fold of
// the wave; 4 pieces a wave share one derivation of the acceptance. 16 million exponentials in 20 us (64 sequences of 128256; the first pass,
// which also reads its logits from memory, does 1.2 per ps): vector ALUs 62 % busy, after a chain of loads for the acceptance.
template <typename E>
__global__ void __launch_bounds__(kT) verify_rest_kernel(Args a) {
  __shared__ float s_m[kMaxRows];
  __shared__ double s_s[kMaxRows];
  __shared__ int s_j[1];
  const int b = blockIdx.y, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = decide<E, false>(a, b, s_m, s_s, s_j);
  const Head h = head_of(a, b, j, s_m, s_s);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.head[b] = h;
  piece_sums<kPieces>(a, Rest<E>(a, b, h), (blockIdx.x * (kT / 64) + wv) * kPieces, a.pr + (int64_t)b * a.npc);
}

// One wave: the smallest of n items whose running sum, from `before` on, passes `want` -- past the last sum (u >= 1, rounding) the
// last item that is more than 0, -1 if there is none. Lane l owns items l * per .. and gives their values through `at`.
// `before` becomes the running sum in front of the item.
template <int PER, typename F>  // PER: `per` is at most that, and the loops over a lane's items are unrolled; 0: any number
__device__ __forceinline__ int search(int per, int n, F at, double want, double& before) {
  const int lane = threadIdx.x & 63, lim = PER > 0 ? PER : per;
  auto item = [&](int k) { return k < per && lane * per + k < n ? at(lane * per + k, k) : 0.0; };
  double mine = 0.0;
#pragma unroll
  for (int k = 0; k < lim; ++k) mine += item(k);
  const double inc = before + wave_scan_d(mine);
  const uint64_t over = __ballot(mine > 0.0 && inc > want), some = __ballot(mine > 0.0);
  if (!some) {
    before = readlane_d(inc, 63);
    return -1;
  }
  const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
  double run = inc - mine, front = 0.0;
  int found = -1;
  bool hit = false;
#pragma unroll
  for (int k = 0; k < lim; ++k) {
    const double v = item(k);
    const bool take = v > 0.0 && !hit;
    found = take ? lane * per + k : found;
    front = take ? run : front;
    run = take ? run + v : run;
    hit = hit || (take && run > want);
  }
  before = readlane_d(front, l);
  return __builtin_amdgcn_readlane(found, l);
}

// One wave: the token drawn from r (h.j's row), from its pieces' sums
template <typename E>
__device__ int64_t draw(const Args& a, int b, const Head& h, const double* pr) {
  constexpr int N = Vec<E>::N;
  Rest<E> f(a, b, h);
  double total = 0.0;
  const int lane = threadIdx.x & 63, per = (a.npc + 63) / 64;
  const double u = (double)a.u[(int64_t)b * (a.T + 1) + a.T];
  // up to kHeld sums a lane (rows of 262144 fp32 logits) in registers, loaded at once: one round trip to memory and not one a sum
  double held[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) held[k] = per <= kHeld && k < per && lane * per + k < a.npc ? pr[lane * per + k] : 0.0;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) total += held[k];
  if (per > kHeld)
    for (int i = lane; i < a.npc; i += 64) total += pr[i];
  total = wave_sum_d(total);
  double before = 0.0;
  int first, last;
  if (total > 0.0) {
    if (per <= kHeld) first = search<kHeld>(per, a.npc, [&](int, int k) { return held[k]; }, u * total, before);
    else first = search<0>(per, a.npc, [&](int i, int) { return pr[i]; }, u * total, before);
    last = first + 1;
  } else {  // r = 0 everywhere: the target's own distribution, whose total is 1, from the first piece on
    if (!(h.ip > 0.0)) return -1;
    f.y = nullptr;
    total = 1.0;
    first = 0;
    last = a.npc;
  }
  int token = -1;
  const double want = u * total;
  for (int pc = first; pc < last; ++pc) {
    double v[N], front = before, sum = 0.0;
    f.vec(pc, a.V, v);
#pragma unroll
    for (int e = 0; e < N; ++e) sum += v[e];
    sum = wave_sum_d(sum);
    const int i = search<N>(N, piece<E>(), [&](int, int k) { return v[k]; }, want, front);
    if (i >= 0) token = pc * piece<E>() + i;
    before += sum;
    if (before > want && token >= 0) break;
  }
  return token;
}
// by one wave: the kept tokens, the next one, then -1
__device__ __forceinline__ void put(const Args& a, int b, int j, int64_t next) {
  const int lane = threadIdx.x & 63;
  if (lane <= a.T)
    a.out[(int64_t)b * (a.T + 1) + lane] = lane < j ? a.tokens[(int64_t)b * a.T + lane] : lane == j ? next : -1;
  if (lane == 0) a.accepted[b] = j;
}

// ---- pass 3: grid B; one wave (greedy: one workgroup). Bound by its chain of loads: head, sums, the piece's logits.
template <typename E>
__global__ void __launch_bounds__(64) verify_draw_kernel(Args a) {
  const int b = blockIdx.x;
  const Head h = a.head[b];
  put(a, b, h.j, draw<E>(a, b, h, a.pr + (int64_t)b * a.npc));
}
template <typename E>
__global__ void __launch_bounds__(kT) verify_greedy_kernel(Args a) {
  __shared__ float s_m[kMaxRows];
  __shared__ double s_s[kMaxRows];
  __shared__ int s_j[1];
  const int b = blockIdx.x, j = decide<E, true>(a, b, s_m, s_s, s_j);
  if (threadIdx.x < 64) put(a, b, j, (int64_t)s_s[j]);
}

// ---- all of it for a small problem: grid B. A wave takes every fourth row, twice (maximum, then sum: the row is in cache). Bound
// by its chain of loads and sums: 64 sequences, 3 drafts, 1000 logits 10.2 us (three launches 17.6).
template <typename E, bool GREEDY>
__global__ void __launch_bounds__(kT) verify_small_kernel(Args a) {
  constexpr int N = Vec<E>::N;
  __shared__ float s_m[kMaxRows];
  __shared__ double s_s[kMaxRows], s_pr[kOneRow / piece<E>() + 1];
  __shared__ int s_j[1];
  const int b = blockIdx.x, t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int nd = drafts(a, b);
  const Drafted d = drafted<E, GREEDY>(a, b, nd);
  for (int r = wv; r < (GREEDY ? a.T + 1 : 2 * a.T + 1); r += kT / 64) {
    if (idle(a, r, nd)) continue;
    const E* x = row_ptr<E>(a, b, r);
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int i = lane * N; i < a.V; i += 64 * N) {
      Vec<E> v;
      v.load(x, i, a.V);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float z = v.get(e) > FLT_MAX ? FLT_MAX : v.get(e);  // (NaN stays, and is passed over)
        at = z > m ? i + e : at;
        m = fmaxf(m, z);
      }
    }
    const float mine = m;
    m = wave_max(m);
    double s = 0.0;
    if constexpr (GREEDY) {
      at = wave_min_i(mine == m ? at : 0x7fffffff);
      s = m > -INFINITY ? (double)at : -1.0;
    } else {
      if (m > -INFINITY)
        for (int i = lane * N; i < a.V; i += 64 * N) {
          Vec<E> v;
          v.load(x, i, a.V);
#pragma unroll
          for (int e = 0; e < N; ++e) s += weight(v.get(e), m, a.c);
        }
      s = wave_sum_d(s);
    }
    if (lane == 0) {
      s_m[r] = m;
      s_s[r] = s;
    }
  }
  __syncthreads();
  const int j = accept<E, GREEDY>(a, d, nd, s_m, s_s, s_j);
  if constexpr (GREEDY) {
    if (t < 64) put(a, b, j, (int64_t)s_s[j]);
  } else {
    const Head h = head_of(a, b, j, s_m, s_s);
    const Rest<E> f(a, b, h);
    for (int pc = wv; pc < a.npc; pc += kT / 64) piece_sums<1>(a, f, pc, s_pr);
    __syncthreads();
    if (t < 64) put(a, b, j, draw<E>(a, b, h, s_pr));
  }
}

template <typename E>
int launch(const Args& a, bool greedy, hipStream_t stream) {
  const int nrow = greedy ? a.T + 1 : 2 * a.T + 1;
  // One workgroup per sequence is short of threads for long rows, three launches cost more than they do for short ones: sampling, 7
  // rows of 2048 fp32 logits 13.5 us in one launch and 14.8 in three, of 2500 16.2 and 15.0; greedy, 9 rows of 2000 7.3 and 8.9 in
  // two, of 4096 11.7 and 8.7.
  if (a.V <= kOneRow && (int64_t)nrow * a.V <= (greedy ? kOneGreedy : kOneLaunch)) {
    if (greedy) verify_small_kernel<E, true><<<a.B, kT, 0, stream>>>(a);
    else verify_small_kernel<E, false><<<a.B, kT, 0, stream>>>(a);
  } else {
    const dim3 rows(a.nch, nrow, a.B);
    if (greedy) {
      verify_stats_kernel<E, true><<<rows, kT, 0, stream>>>(a);
      verify_greedy_kernel<E><<<a.B, kT, 0, stream>>>(a);
    } else {
      verify_stats_kernel<E, false><<<rows, kT, 0, stream>>>(a);
      constexpr int per = kT / 64 * kPieces;
      verify_rest_kernel<E><<<dim3((a.npc + per - 1) / per, a.B), kT, 0, stream>>>(a);
      verify_draw_kernel<E><<<a.B, 64, 0, stream>>>(a);
    }
  }
  return hipGetLastError() == hipSuccess ? 0 : -9;
}
inline int64_t chunks(int V) { return (V + kChunk - 1) / kChunk; }
inline int64_t pieces(int V, bool f32) {
  const int n = f32 ? piece<float>() : piece<bf16_t>();
  return (V + n - 1) / n;
}
}  // namespace

int64_t verify_draft_workspace(int B, int T, int V, bool f32) {
  return (int64_t)B * (2 * T + 1) * chunks(V) * (8 + 4) + (int64_t)B * (pieces(V, f32) * 8 + sizeof(Head));
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
  a.nch = (int)chunks(V), a.npc = (int)pieces(V, f32);
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
