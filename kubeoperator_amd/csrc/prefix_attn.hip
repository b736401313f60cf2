// Attention of a batch that shares a long prefix, for gfx950 (serving): the newest T tokens of every sequence (T = 1: a
// decode step; T > 1: drafted tokens under verification, or a prompt) against
//
//   the prefix   K, V [Hkv, P, D], one copy for the whole batch, seen by every row;
//   the own keys K, V [B, Hkv, Smax, D]: token t of T sees the first lens[b] - (T - 1 - t) of them.
//
// One softmax over both. The rows of ALL sequences meet the prefix together (B T G rows per KV head, G = Hq / Hkv), so its
// keys leave HBM once per row tile instead of once per sequence, and its products have enough rows for the matrix cores.
//
// S^T [keys x rows] = K . Q^T and O^T [dims x rows] += V^T . P^T on v_mfma_f32_16x16x32_bf16, with running maximum and sum
// per row (fp32). P goes through the matrix cores as a bf16 value and its bf16 remainder, two products (2^-15 relative per key): a
// value alone (2^-8) adds as much to the result's error as its own rounding does (0.0023 relative instead of 0.0016), saves nothing
// where memory is the bound and a sixth to a quarter elsewhere (drafts 86 us, with the remainder 103; 8 x 1024 tokens behind 2048
// 371 and 468). The 16 key rows of product b are keys
// 8 (i >> 2) + 4 b + (i & 3), so that a lane's scores of two products are its own P^T operand (keys 8 g .. 8 g + 7 of its row),
// with no lane exchange; V goes through an LDS image whose 16-byte chunks are XOR-permuted by the row, and is read transposed.
// A workgroup works in one of two ways:
//   * by keys (up to 32 rows): its 4 waves take every fourth 32-key block of all its rows. K goes straight to registers, V through
//     LDS-DMA; both of the next block are in flight while a block is computed; the waves' results meet in LDS. Bound by memory.
//   * by rows (128 rows): each wave has 32 rows of its own, and K and V of every 64-key tile come from LDS, where the four share
//     them. The next tile's scores (matrix cores) run beside this tile's weights (vector ALUs). Bound by those two.
// and a launch takes one of three forms (make_plan):
//   * split: workgroups of (row tile, key range) of the prefix, and of one sequence's own keys, write fp32 partials (O, max, sum);
//     a second launch folds them. Decode (64 sequences, 32/8 heads of 128, 2048 + up to 500 keys): 23 + 5 us, 3.3 TB/s in the
//     first. Drafts (64 x 5 tokens, 8192 + up to 1000 keys, prefix by rows): 96 + 7 us; the prefix alone 99, 435 TFLOP/s.
//   * short contexts, by keys: a workgroup takes prefix and own keys of its rows, one launch, no partials. 4 sequences, 500 + 60
//     keys: 7.3 us against 8.3 split.
//   * prompts, by rows: the same for sequences with many tokens. 8 x 1024 tokens behind 2048, 32/8 heads of 128: 470 us, 730
//     TFLOP/s; one prompt of 4096, no prefix: 200 us, 690 TFLOP/s (matrix cores 47-53 % busy, vector ALUs 54-60 %).
//
// A masked key has weight zero exactly: masked scores never enter the maximum or the sum, keys past the last valid one are
// never read (loads are clamped to it), and in the blocks where some rows see a key and others do not, values that are
// not finite are kept from the rows that do not.
#include <algorithm>
#include <cmath>

#include "attn_common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -3.402823466e38f;
// A row's reference for exp2 follows its maximum only when that is this much higher: any reference gives the same softmax, weights
// of up to 2^8 round as well as those of up to 1, and most tiles then need no rescaling of O^T.
constexpr float kSlack = 8.f;
constexpr int kLds = 65536;
constexpr int kByRows = 4;
constexpr int kTrans = 0x400, kMfma = 0x8, kDsRead = 0x100;  // instruction classes of sched_group_barrier

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// XOR of a V row's 16-byte chunk slots in the LDS image (row r = 8g + 4h + q of a wave's 32 keys): spreads the 8 rows that a
// 32-lane half reads per transposed read over distinct chunk slots
template <int ROWB>
__device__ __forceinline__ int vx(int r) {
  if constexpr (ROWB == 256) return ((r & 3) << 1) | (((r >> 3) & 1) << 3);
  else return (((r >> 1) & 1) << 1) | (((r >> 3) & 1) << 2);
}
// the V^T operands of four 16-dim blocks: 8 transposed reads, waited for here
template <int ROWB>
__device__ __forceinline__ void read_v4(const uint32_t* a, bf16x8* v) {
  bf16x4 t[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\t"
      "ds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\t"
      "ds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\t"
      "ds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3]), "=&v"(t[4]), "=&v"(t[5]), "=&v"(t[6]), "=&v"(t[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(4 * ROWB)
      : "memory");
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = cat44(t[2 * c], t[2 * c + 1]);
}
// the 8 bf16 values with those that are not finite replaced by 0, and 1 in their places, else 0
__device__ __forceinline__ void split_finite(bf16x8 v, bf16x8& fin, bf16x8& bad) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool nf = (v[i] & 0x7f80) == 0x7f80;
    fin[i] = nf ? (short)0 : v[i];
    bad[i] = nf ? (short)0x3f80 : (short)0;
  }
}
__device__ __forceinline__ bool not_finite(bf16x8 v) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return any;
}

struct Args {
  const bf16_t *q, *kp, *vp, *kc, *vc;
  const int* lens;
  int64_t qs, kph, kps, vph, vps;
  int B, T, G, Hkv, P, Smax, max_len;
  bool flip;            // scale < 0
  int pchunk, np, rtp;  // prefix: keys per range, ranges, row tiles of all sequences
  int ochunk, ns, rto;  // own keys: keys per range, ranges, row tiles of one sequence
  float sl2;            // |scale| log2 e
  bf16_t* o;
  int64_t os;
  float *po, *pml;  // partials [Hkv][B T G][np + ns][D] and [..][2] (max, sum)
};
}  // namespace

namespace {
// one workgroup's rows and keys
struct Work {
  int kvh, row0, nrow;   // rows [row0, row0 + nrow) of this KV head
  int slot;              // where its partial goes
  int k0, kend, nkeys;   // keys [k0, kend); no key at or past nkeys is read
  int seen0;             // own keys: what token 0 of the sequence sees (0 or less: nothing)
  int lim0;              // keys that every row of the tile sees
  bool own;
  const bf16_t *k, *v;
  int ks, vs;            // elements between keys (up to 2^23)
};
__device__ __forceinline__ int seen_by(const Args& p, const Work& w, int bt) { return w.own ? w.seen0 + bt % p.T : w.nkeys; }

// a row's Q^T operand: dims 32 s + 8 g .. + 7 (a negative scale is taken into Q's signs, so that maxima can be taken
// before scaling)
template <int D>
__device__ __forceinline__ void load_q(const Args& p, const Work& w, int r, int g, bf16x8* qf) {
  const int bt = r / p.G, h = w.kvh * p.G + r % p.G;
  const bf16_t* qr = p.q + (int64_t)bt * p.qs + (int64_t)h * D + 8 * g;
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    u32x4 v = *reinterpret_cast<const u32x4*>(qr + 32 * s);
    if (p.flip) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] ^= 0x80008000u;
    }
    qf[s] = __builtin_bit_cast(bf16x8, v);
  }
}

// maximum that passes a NaN on: no quieting of each operand first, two values per instruction
__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// One 16-row tile's running softmax over NB blocks of 32 keys: sc[b] = scores of products 2 b, 2 b + 1 (the lane's keys
// 32 (b / 2) + 8 g + 4 (b % 2) + e). `left`: the lane's keys of block 0 with a number below it are seen (block b:
// left - 32 b); only looked at on an edge. First the maximum: masked scores leave sc, and where a row's maximum rises by
// more than kSlack, acc (NC blocks of O^T) and l (the sum of the lane's own weights) are scaled down.
template <bool EDGE, int NB, int NC>
__device__ __forceinline__ void raise_max(f32x4* sc, int left, float sl2, float& m, float& l, f32x4* acc) {
  if constexpr (EDGE) {
#pragma unroll
    for (int j = 0; j < 8 * NB; ++j) sc[j >> 2][j & 3] = 32 * (j >> 3) + (j & 7) < left ? sc[j >> 2][j & 3] : kNegBig;
  }
  float mx = sc[0][0];
#pragma unroll
  for (int j = 1; j + 1 < 8 * NB; j += 2) mx = vmax(vmax(mx, sc[j >> 2][j & 3]), sc[(j + 1) >> 2][(j + 1) & 3]);
  mx = vmax(mx, sc[2 * NB - 1][3]);
  mx = xor32_max(xor16_max(mx)) * sl2;
  if (__any(mx > m + kSlack)) {
    const float nm = fmaxf(m, mx);
    const float al = __builtin_amdgcn_exp2f(m - nm);
    m = nm;
    l *= al;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[c][e] *= al;
  }
}
// Then the weights, P^T: their sum into l, in fp32, and each as a bf16 value (cut, not rounded) and the bf16 remainder. 2^-20 of the
// weight goes into the remainder, so that one of a weight above 0 is above 0 too: times an infinite value, the two add up to inf.
template <bool EDGE, int NB>
__device__ __forceinline__ void weights(const f32x4* sc, int left, float sl2, float m, float& l, bf16x8* hi, bf16x8* lo) {
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    u32x4 h, r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int j = 8 * b + 2 * i + k;
        v[k] = __builtin_amdgcn_exp2f(fmaf(sc[j >> 2][j & 3], sl2, -m));
        if constexpr (EDGE) v[k] = 32 * (j >> 3) + (j & 7) < left ? v[k] : 0.f;
        s[k] += v[k];
      }
      const uint32_t x = __float_as_uint(v[0]), y = __float_as_uint(v[1]);
      constexpr float up = 1.f + 0x1p-20f;
      const uint32_t xh = x & 0xffff0000u, yh = y & 0xffff0000u;
      h[i] = NB == 1 ? yh | (x >> 16) : __builtin_amdgcn_perm(y, x, 0x07060302u);  // (by keys no scalar register is left for the constant)
      r[i] = pack2(fmaf(v[0], up, -__uint_as_float(xh)), fmaf(v[1], up, -__uint_as_float(yh)));
    }
    hi[b] = __builtin_bit_cast(bf16x8, h);
    lo[b] = __builtin_bit_cast(bf16x8, r);
  }
  l += s[0] + s[1];
}
// a row's sum from its four lanes'
__device__ __forceinline__ float row_sum(float l) { return xor32_sum(xor16_sum(l)); }

// acc += V^T . P^T where some rows see a key and others do not: values that are not finite reach only the rows that see them
// (as NaN). True if there were any; `left` as in weights(), of this block.
template <int NT>
__device__ __forceinline__ bool edge_pv(bf16x8 vf, const bf16x8* hi, const bf16x8* lo, const int* left, f32x4* acc) {
  if (!__any(not_finite(vf))) return false;
  bf16x8 fin, bad;
  split_finite(vf, fin, bad);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    bf16x8 ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = j < left[n] ? (short)0x3f80 : (short)0;
    const f32x4 nb = mfma16(bad, ones, f32x4{0.f, 0.f, 0.f, 0.f});
    acc[n] = mfma16(fin, hi[n], mfma16(fin, lo[n], acc[n]));
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = nb[e] > 0.f ? __builtin_nanf("") : acc[n][e];
  }
  return true;
}

// ---- few rows: all 4 waves take the same 16 NT rows, and every fourth 32-key block. SEGS = 1: one key range of one part,
// to a partial; 2: the prefix and then the own keys, to the output.
template <int D, int NT, int SEGS, typename F>
__device__ __forceinline__ void by_keys(const Args& p, F part, char* smem) {
  constexpr int ROWB = D * 2, NS = D / 32, NC = D / 16, KW = 32, NWV = kThreads / 64, KSTEP = KW * NWV;
  constexpr int IMG = KW * ROWB, VPW = IMG / 1024, SLOTS = ROWB / 16, RPP = 1024 / ROWB;
  // two V images per wave; afterwards the waves' O^T (two of them at a time)
  static_assert(NWV * 2 * IMG <= kLds && 2 * NT * 16 * D * 4 <= kLds, "LDS");
  __shared__ float s_ml[NWV][NT * 16][2];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const Work w0 = part(0);
  bf16x8 qf[NT][NS];
  int bt[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = w0.row0 + (16 * n + col < w0.nrow ? 16 * n + col : 0);
    load_q<D>(p, w0, r, g, qf[n]);
    bt[n] = r / p.G;
  }
  char* const vimg = smem + wv * (2 * IMG);
  const int tq = (lane >> 2) & 3, tp = lane & 3;
  const int x = vx<ROWB>(8 * g + tq) >> 1;
  uint32_t va[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c)
    va[c] = lds_addr(vimg) + (8 * g + tq) * ROWB + 8 * (tp & 1) + 16 * ((2 * c + (tp >> 1)) ^ (2 * x));
  float m[NT], l[NT];
  f32x4 acc[NT][NC];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = kNegBig;
    l[n] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[n][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 1
  for (int seg = 0; seg < SEGS; ++seg) {
    const Work w = SEGS == 1 ? w0 : part(seg);
    int lim[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) lim[n] = seen_by(p, w, bt[n]);
    // 32-bit lane offsets from the block's first key; `LAST`: the block may reach past the last key, whose row is read instead
    const uint32_t ko = (uint32_t)((8 * (col >> 2) + (col & 3)) * w.ks + 8 * g) * 2;
    uint32_t vo[2];  // V pieces i: the swizzle has two forms, of i's bit 1 (D = 128) or 0 (D = 64)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      vo[h] = (uint32_t)((lane / SLOTS) * w.vs + 8 * ((lane % SLOTS) ^ vx<ROWB>(8 * h + lane / SLOTS))) * 2;
    static_assert(ROWB == 256 || ROWB == 128, "piece -> swizzle form");
    auto load_k = [&](auto last_, int kb, bf16x8 (*kf)[NS]) {
      const char* base = reinterpret_cast<const char*>(w.k + (int64_t)kb * w.ks);
#pragma unroll
      for (int bb = 0; bb < 2; ++bb) {
        uint32_t o = ko;
        if constexpr (decltype(last_)::value)
          o = (uint32_t)(min(8 * (col >> 2) + 4 * bb + (col & 3), w.nkeys - 1 - kb) * w.ks + 8 * g) * 2;
        else base += bb * 8 * w.ks;
#pragma unroll
        for (int s = 0; s < NS; ++s) kf[bb][s] = *reinterpret_cast<const bf16x8*>(base + o + 64 * s);
      }
    };
    auto load_v = [&](auto last_, int kb, char* img) {
      const char* base = reinterpret_cast<const char*>(w.v + (int64_t)kb * w.vs);
#pragma unroll
      for (int i = 0; i < VPW; ++i) {
        uint32_t o = vo[(ROWB == 256 ? i >> 1 : i) & 1];
        if constexpr (decltype(last_)::value) {
          const int r = RPP * i + lane / SLOTS;
          o = (uint32_t)(min(r, w.nkeys - 1 - kb) * w.vs + 8 * ((lane % SLOTS) ^ vx<ROWB>(r))) * 2;
          glds16(base + o, img + 1024 * i);
        } else {
          glds16(base + 2 * RPP * i * w.vs + o, img + 1024 * i);
        }
      }
    };
    auto load = [&](int kb, auto&& f) {  // (two parts: one form for all blocks, for the scalar registers)
      if (SEGS == 1 && kb + KW <= w.nkeys) f(std::false_type{});
      else f(std::true_type{});
    };
    // the wave's blocks. In flight during a block's softmax and second product: the next one's K (registers, free after the
    // first product) and V (LDS-DMA into the other image, issued before it)
    int kb = w.k0 + KW * wv, buf = 0;
    bf16x8 kf[2][NS];
    if (kb < w.kend) {
      load(kb, [&](auto last) {
        load_k(last, kb, kf);
        load_v(last, kb, vimg);
      });
    }
    auto block = [&](auto edge_) {
      constexpr bool EDGE = decltype(edge_)::value;
      const bool more = kb + KSTEP < w.kend;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (more) load(kb + KSTEP, [&](auto last) { load_v(last, kb + KSTEP, vimg + (buf ^ 1) * IMG); });
      f32x4 sc[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int bb = 0; bb < 2; ++bb) {
          sc[n][bb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < NS; ++s) sc[n][bb] = mfma16(kf[bb][s], qf[n][s], sc[n][bb]);
        }
      if (more) load(kb + KSTEP, [&](auto last) { load_k(last, kb + KSTEP, kf); });
      bf16x8 hi[NT], lo[NT];
      int left[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        left[n] = lim[n] - kb - 8 * g;
        raise_max<EDGE, 1, NC>(sc[n], left[n], p.sl2, m[n], l[n], acc[n]);
        if constexpr (EDGE && SEGS == 2) asm volatile("" : "+v"(left[n]));  // (its comparisons are made again, not held: scalar registers)
        weights<EDGE, 1>(sc[n], left[n], p.sl2, m[n], l[n], &hi[n], &lo[n]);
      }
#pragma unroll
      for (int c0 = 0; c0 < NC; c0 += 4) {
        uint32_t a[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) a[c] = va[c0 + c] + buf * IMG;
        bf16x8 vf[4];
        read_v4<ROWB>(a, vf);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if constexpr (EDGE) {
            f32x4 an[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) an[n] = acc[n][c0 + c];
            if (!edge_pv<NT>(vf[c], hi, lo, left, an)) {
#pragma unroll
              for (int n = 0; n < NT; ++n) an[n] = mfma16(vf[c], hi[n], mfma16(vf[c], lo[n], an[n]));
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][c0 + c] = an[n];
            __builtin_amdgcn_sched_barrier(0);
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][c0 + c] = mfma16(vf[c], hi[n], mfma16(vf[c], lo[n], acc[n][c0 + c]));
          }
        }
      }
    };
    for (; kb < w.kend && kb + KW <= w.lim0; kb += KSTEP, buf ^= 1) block(std::false_type{});
    for (; kb < w.kend; kb += KSTEP, buf ^= 1) block(std::true_type{});  // edges: some rows see some of the keys, others do not
  }
  // the 4 waves' (m, l, O^T) -> one partial: waves 2, 3 into 0, 1, then 1 into 0
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = row_sum(l[n]);
    if (g == 0) {
      s_ml[wv][16 * n + col][0] = m[n];
      s_ml[wv][16 * n + col][1] = l[n];
    }
  }
  __syncthreads();  // every wave is done with its V images
  f32x4* so = reinterpret_cast<f32x4*>(smem);  // [2][NT][NC][64]
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    if (wv >= half && wv < 2 * half) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < NC; ++c) so[(((wv - half) * NT + n) * NC + c) * 64 + lane] = acc[n][c];
    }
    __syncthreads();
    if (wv < half) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float om = s_ml[wv + half][16 * n + col][0], ol = s_ml[wv + half][16 * n + col][1];
        const float nm = fmaxf(m[n], om);
        const float wa = l[n] == 0.f ? 0.f : __builtin_amdgcn_exp2f(m[n] - nm);
        const float wb = ol == 0.f ? 0.f : __builtin_amdgcn_exp2f(om - nm);
        m[n] = nm;
        l[n] = l[n] * wa + ol * wb;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const f32x4 o = so[((wv * NT + n) * NC + c) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][c][e] = acc[n][c][e] * wa + o[e] * wb;
        }
      }
    }
    __syncthreads();
    if (wv < half && g == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s_ml[wv][16 * n + col][0] = m[n];
        s_ml[wv][16 * n + col][1] = l[n];
      }
    }
    __syncthreads();
  }
  if (wv != 0) return;
  if constexpr (SEGS == 2) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (16 * n + col >= w0.nrow) continue;
      const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];
      const int h = w0.kvh * p.G + (w0.row0 + 16 * n + col) % p.G;
      bf16_t* op = p.o + (int64_t)bt[n] * p.os + (int64_t)h * D + 4 * g;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        *reinterpret_cast<u32x2*>(op + 16 * c) =
            u32x2{pack2(acc[n][c][0] * inv, acc[n][c][1] * inv), pack2(acc[n][c][2] * inv, acc[n][c][3] * inv)};
    }
    return;
  }
  const Work& w = w0;
  const int RR = p.B * p.T * p.G;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (16 * n + col >= w.nrow) continue;
    const int64_t at = ((int64_t)w.kvh * RR + w.row0 + 16 * n + col) * (p.np + p.ns) + w.slot;
#pragma unroll
    for (int c = 0; c < NC; ++c) *reinterpret_cast<f32x4*>(p.po + at * D + 16 * c + 4 * g) = acc[n][c];
    if (g == 0) {
      p.pml[2 * at] = m[n];
      p.pml[2 * at + 1] = l[n];
    }
  }
}

// ---- many rows: each wave takes 32 rows of its own, all 4 take every 64-key tile from LDS (K and V images, two of each:
// the next tile travels through registers while one is computed)
// WHOLE: one sequence's rows over its own keys and then over the prefix, no partials; else a range of the prefix
template <int D, bool WHOLE, typename F>
__device__ __forceinline__ void by_rows(const Args& p, F part, char* smem) {
  constexpr int ROWB = D * 2, NS = D / 32, NC = D / 16, TK = 64, IMG = TK * ROWB, SLOTS = ROWB / 16, NT = 2;
  constexpr int PER = TK * SLOTS / kThreads;  // 16-byte pieces per thread and image
  static_assert(4 * IMG <= kLds, "LDS");
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Work w0 = part(0);
  const bool live = 32 * wv < w0.nrow;
  bf16x8 qf[NT][NS];
  // the rows' tokens and outputs, kept in LDS: over the loops there is no register to spare for them, of either kind
  __shared__ int s_bt[kThreads / 64 * 32];
  __shared__ bf16_t* s_op[WHOLE ? kThreads / 64 * 32 : 1];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    const int i = 32 * wv + 16 * n + col, r = w0.row0 + (i < w0.nrow ? i : 0);
    load_q<D>(p, w0, r, g, qf[n]);
    const int bt = r / p.G;
    s_bt[32 * wv + 16 * n + col] = bt;  // the same from all four lanes of a row; read by this wave alone
    if constexpr (WHOLE)
      s_op[32 * wv + 16 * n + col] =
          i >= w0.nrow ? nullptr : p.o + (int64_t)bt * p.os + (int64_t)(w0.kvh * p.G + r % p.G) * D;
  }
  // K image: chunk slots XORed with the row's number in a 16-row operand (8 a + 4 b + q -> 4 a + q), so that its 16 rows'
  // reads of one chunk fall on different banks; V image as in by_keys
  auto kx = [](int r) { return ROWB == 256 ? (((r >> 3) & 3) << 2) | (r & 3) : (((r >> 3) & 3) << 1) | ((r >> 1) & 1); };
  float m[NT], l[NT];
  f32x4 acc[NT][NC];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = kNegBig;
    l[n] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[n][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
#pragma unroll 1
  for (int seg = 0; seg < (WHOLE ? 2 : 1); ++seg) {
    const Work w = WHOLE ? part(seg) : w0;
    if (WHOLE && w.k0 >= w.kend) continue;
    if (seg > 0) barrier();  // the images are free
    int t = threadIdx.x;
    if constexpr (WHOLE) asm volatile("" : "+v"(t));  // what follows from it is made again for each part, not held over the other one's loop
    const int lane = t & 63, col = lane & 15, g = lane >> 4;
    // chunk 4 s + g of a K row is at ka ^ 64 s, 16-dim block c of V^T at va ^ 32 c
    const int krow = 8 * (col >> 2) + (col & 3), vrow = 8 * g + ((lane >> 2) & 3), tp = lane & 3;
    const int ka = krow * ROWB + 16 * (g ^ kx(krow));
    const int va = vrow * ROWB + 8 * (tp & 1) + 16 * ((tp >> 1) ^ vx<ROWB>(vrow));
    int lim[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) lim[n] = seen_by(p, w, s_bt[32 * wv + 16 * n + col]);
    // a thread's pieces are rows t / SLOTS + i * RSTEP of the tile, all at chunk t % SLOTS
    constexpr int RSTEP = kThreads / SLOTS;
    const int tr = t / SLOTS, ch = t % SLOTS;
    const uint32_t ko = (uint32_t)(tr * w.ks + 8 * ch) * 2, vo = (uint32_t)(tr * w.vs + 8 * ch) * 2;
    auto fetch = [&](const bf16_t* src, int step, uint32_t off, int kb, u32x4* to) {
      if constexpr (WHOLE) asm volatile("" : "+s"(step));  // its multiples are made here, not held over the loop: scalar registers
      const int64_t stride = step;
      const char* base = reinterpret_cast<const char*>(src + kb * stride);
      if (kb + TK <= w.nkeys) {
#pragma unroll
        for (int i = 0; i < PER; ++i) to[i] = *reinterpret_cast<const u32x4*>(base + 2 * RSTEP * i * stride + off);
      } else {  // rows past the last key: the last key's
#pragma unroll
        for (int i = 0; i < PER; ++i)
          to[i] = *reinterpret_cast<const u32x4*>(
              base + (uint32_t)(min(tr + RSTEP * i, w.nkeys - 1 - kb) * (int)stride + 8 * ch) * 2);
      }
    };
    // where they go in the images: RSTEP rows on, the K swizzle has one of two forms and the V swizzle stays
    static_assert(RSTEP == 16 || RSTEP == 32, "rows between a thread's pieces");
    int kw[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) kw[h] = tr * ROWB + 16 * (ch ^ kx(tr + RSTEP * h));
    const int vw = tr * ROWB + 16 * (ch ^ vx<ROWB>(tr));
    char* const kimg = smem;            // two K images, two V images
    char* const vimg = smem + 2 * IMG;
    auto put_k = [&](const u32x4* from, int buf) {
#pragma unroll
      for (int i = 0; i < PER; ++i) *reinterpret_cast<u32x4*>(kimg + buf * IMG + kw[i & 1] + i * RSTEP * ROWB) = from[i];
    };
    auto put_v = [&](const u32x4* from, int buf) {
#pragma unroll
      for (int i = 0; i < PER; ++i) *reinterpret_cast<u32x4*>(vimg + buf * IMG + vw + i * RSTEP * ROWB) = from[i];
    };
    f32x4 sc[NT][4];
    // a product's addresses, settled before its stretch of code is put in order (address arithmetic would count as work to place)
    auto k_at = [&](int buf, uint32_t* at) {
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        at[s] = (uint32_t)((buf * IMG + ka) ^ (64 * s));
        asm volatile("" : "+v"(at[s]));
      }
    };
    auto v_at = [&](int buf, uint32_t* at) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        at[c] = (uint32_t)((buf * IMG + va) ^ (32 * c));
        asm volatile("" : "+v"(at[c]));
      }
    };
    auto scores = [&](const uint32_t* at, f32x4 (*s4)[4]) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s4[n][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const bf16x8 kf = lds_read8(kimg + at[s] + (32 * (b >> 1) + 4 * (b & 1)) * ROWB);
#pragma unroll
          for (int n = 0; n < NT; ++n) s4[n][b] = mfma16(kf, qf[n][s], s4[n][b]);
        }
      }
    };
    // One tile: its scores are there. The next tile's scores (matrix cores) are computed beside this one's weights (vector ALUs), on
    // an edge afterwards (both at once and the sifting take more registers than two waves per SIMD have).
    auto tile = [&](auto edge_, auto next_, int kb, int buf) {
      constexpr bool EDGE = decltype(edge_)::value, NEXT = decltype(next_)::value, SIFT = EDGE && WHOLE;
#pragma unroll
      for (int n = 0; n < NT; ++n) raise_max<EDGE, 2, NC>(sc[n], lim[n] - kb - 8 * g, p.sl2, m[n], l[n], acc[n]);
      bf16x8 hi[NT][2], lo[NT][2];
      f32x4 nx[NT][4];
      uint32_t kat[NS], vat[NC];
      if constexpr (NEXT && !EDGE) k_at(buf ^ 1, kat);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (NEXT && !EDGE) scores(kat, nx);
#pragma unroll
      for (int n = 0; n < NT; ++n) weights<EDGE, 2>(sc[n], lim[n] - kb - 8 * g, p.sl2, m[n], l[n], hi[n], lo[n]);
      if constexpr (NEXT && !EDGE) {
        // issue order: operands of one 16-key product ahead, each read once its register's last value is used, and between two
        // matrix instructions what one of them leaves time for
        __builtin_amdgcn_sched_group_barrier(kDsRead, NS, 0);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
          for (int i = 0; i < NS * NT; ++i) {
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kTrans, 8 / (NS * NT), 0);
            if (b < 3 && i % NT == NT - 1) __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // waves in the vector stretch go first: the other wave of the SIMD has matrix instructions to fill the gaps with (8 x 1024 tokens
      // behind 4096: 858 us without, 847)
      __builtin_amdgcn_s_setprio(0);
      v_at(buf, vat);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const char* vp = vimg + vat[c] + 32 * b * ROWB;
          const bf16x8 vf = cat44(lds_tr_read(vp), lds_tr_read(vp + 4 * ROWB));
          if constexpr (SIFT) {
            bf16x8 hn[NT], ln[NT];
            f32x4 an[NT];
            int left[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              hn[n] = hi[n][b], ln[n] = lo[n][b], an[n] = acc[n][c], left[n] = lim[n] - kb - 8 * g - 32 * b;
              asm volatile("" : "+v"(left[n]));  // what is made of it is made where it is used, and not held for all blocks
            }
            if (!edge_pv<NT>(vf, hn, ln, left, an)) {
#pragma unroll
              for (int n = 0; n < NT; ++n) an[n] = mfma16(vf, hn[n], mfma16(vf, ln[n], an[n]));
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][c] = an[n];
            __builtin_amdgcn_sched_barrier(0);
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][c] = mfma16(vf, lo[n][b], acc[n][c]);
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][c] = mfma16(vf, hi[n][b], acc[n][c]);
          }
        }
      if constexpr (!SIFT) {  // issue order: three 16-dim blocks' operands ahead
        __builtin_amdgcn_sched_group_barrier(kDsRead, 6, 0);
#pragma unroll
        for (int i = 0; i < 2 * NC - 3; ++i) {
          __builtin_amdgcn_sched_group_barrier(kMfma, 2 * NT, 0);
          __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, 6 * NT, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      if constexpr (NEXT && EDGE) {
        k_at(buf ^ 1, kat);
        scores(kat, sc);
        __builtin_amdgcn_sched_barrier(0);
      } else if constexpr (NEXT) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int b = 0; b < 4; ++b) sc[n][b] = nx[n][b];
      }
    };
    // Tile i reads V image i and K image i + 1 (both modulo 2); meanwhile V i + 1 and K i + 2 go from registers into the images
    // that tile i - 1 has left, and V i + 2 and K i + 3 into the registers.
    u32x4 kr[PER], vr[PER];
    int kb = w.k0, buf = 0;
    fetch(w.k, w.ks, ko, kb, kr);
    fetch(w.v, w.vs, vo, kb, vr);
    put_k(kr, 0);
    put_v(vr, 0);
    if (kb + TK < w.kend) {
      fetch(w.k, w.ks, ko, kb + TK, kr);
      put_k(kr, 1);
      fetch(w.v, w.vs, vo, kb + TK, vr);
    }
    if (kb + 2 * TK < w.kend) fetch(w.k, w.ks, ko, kb + 2 * TK, kr);
    barrier();
    uint32_t kat0[NS];
    k_at(0, kat0);
    if (live) scores(kat0, sc);
    auto stage = [&](auto edge_, auto next_) {
      // every wave is done with the tile before: image `buf` of K (whose scores are taken) and the other one of V are free
      barrier();
      if (kb + TK < w.kend) put_v(vr, buf ^ 1);
      if (kb + 2 * TK < w.kend) {
        put_k(kr, buf);
        fetch(w.v, w.vs, vo, kb + 2 * TK, vr);
      }
      if (kb + 3 * TK < w.kend) fetch(w.k, w.ks, ko, kb + 3 * TK, kr);
      if (live) tile(edge_, next_, kb, buf);
      kb += TK;
      buf ^= 1;
    };
    while (kb + TK < w.kend && kb + TK <= w.lim0) stage(std::false_type{}, std::true_type{});
    while (kb + TK < w.kend) stage(std::true_type{}, std::true_type{});
    stage(std::true_type{}, std::false_type{});
  }
  if (!live) return;
  const int col = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n) l[n] = row_sum(l[n]);
  if constexpr (WHOLE) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      bf16_t* op = s_op[32 * wv + 16 * n + col];
      if (!op) continue;
      const float inv = l[n] == 0.f ? 0.f : 1.f / l[n];
#pragma unroll
      for (int c = 0; c < NC; ++c)
        *reinterpret_cast<u32x2*>(op + 4 * g + 16 * c) =
            u32x2{pack2(acc[n][c][0] * inv, acc[n][c][1] * inv), pack2(acc[n][c][2] * inv, acc[n][c][3] * inv)};
    }
    return;
  }
  const int RR = p.B * p.T * p.G;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int i = 32 * wv + 16 * n + col;
    if (i >= w0.nrow) continue;
    const int64_t at = ((int64_t)w0.kvh * RR + w0.row0 + i) * (p.np + p.ns) + w0.slot;
#pragma unroll
    for (int c = 0; c < NC; ++c) *reinterpret_cast<f32x4*>(p.po + at * D + 16 * c + 4 * g) = acc[n][c];
    if (g == 0) {
      p.pml[2 * at] = m[n];
      p.pml[2 * at + 1] = l[n];
    }
  }
}

constexpr int tile_rows(int mode) { return mode == kByRows ? 128 : 16 * mode; }
}  // namespace

// PM / OM: how the prefix's / the own keys' workgroups work (1, 2: by keys, that many 16-row tiles; the prefix's also kByRows).
// Two workgroups per CU: 256 registers.
template <int D, int PM, int OM>
__global__ void __launch_bounds__(kThreads, 2) prefix_attn_kernel(Args p) {
  __shared__ __attribute__((aligned(16))) char smem[kLds];
  Work w;
  int id = blockIdx.x;
  const int nprefix = p.Hkv * p.rtp * p.np;
  if (id < nprefix) {
    w.own = false;
    w.slot = id / (p.Hkv * p.rtp);
    id -= w.slot * p.Hkv * p.rtp;
    w.kvh = id % p.Hkv;
    w.row0 = (id / p.Hkv) * tile_rows(PM);
    w.nrow = min(tile_rows(PM), p.B * p.T * p.G - w.row0);
    w.k0 = w.slot * p.pchunk;
    w.nkeys = w.lim0 = p.P;
    w.kend = min(p.P, w.k0 + p.pchunk);
    w.k = p.kp + w.kvh * p.kph;
    w.v = p.vp + w.kvh * p.vph;
    w.ks = (int)p.kps;
    w.vs = (int)p.vps;
  } else {
    w.own = true;
    id -= nprefix;
    const int split = id % p.ns;
    id /= p.ns;
    w.kvh = id % p.Hkv;
    id /= p.Hkv;
    const int b = id / p.rto, first = (id % p.rto) * tile_rows(OM);
    w.nrow = min(tile_rows(OM), p.T * p.G - first);
    w.row0 = b * p.T * p.G + first;
    w.slot = p.np + split;
    w.k0 = split * p.ochunk;
    w.nkeys = min(max(p.lens[b], 0), p.max_len);
    w.seen0 = w.nkeys - p.T + 1;
    w.lim0 = w.seen0 + first / p.G;
    w.kend = min(w.seen0 + (first + w.nrow - 1) / p.G, w.k0 + p.ochunk);  // up to what the tile's last token sees
    w.k = p.kc + ((int64_t)b * p.Hkv + w.kvh) * p.Smax * D;
    w.v = p.vc + ((int64_t)b * p.Hkv + w.kvh) * p.Smax * D;
    w.ks = w.vs = D;
  }
  if (w.k0 >= w.kend) return;  // nothing to see: pass 2 does not read this range's partials
  const auto part = [&](int) { return w; };
  if (PM == OM || w.own) by_keys<D, OM, 1>(p, part, smem);
  else if constexpr (PM == kByRows) by_rows<D, false>(p, part, smem);
  else if constexpr (PM != OM) by_keys<D, PM, 1>(p, part, smem);
}

// What workgroup `id` of a launch without partials takes: a (sequence, tile of ROWS rows, KV head), the prefix (seg 0) or the own
// keys (seg 1). The last tiles, which see the most, come first.
template <int D, int ROWS>
__device__ __forceinline__ Work whole_part(const Args& p, int id, int seg) {
  Work w;
  w.kvh = id % p.Hkv;
  id /= p.Hkv;
  const int b = id % p.B, first = (p.rto - 1 - id / p.B) * ROWS;
  w.own = seg != 0;
  w.row0 = b * p.T * p.G + first;
  w.nrow = min(ROWS, p.T * p.G - first);
  w.slot = 0;
  w.k0 = 0;
  if (seg == 0) {
    w.nkeys = w.lim0 = w.kend = p.P;
    w.k = p.kp + w.kvh * p.kph;
    w.v = p.vp + w.kvh * p.vph;
    w.ks = (int)p.kps;
    w.vs = (int)p.vps;
  } else {
    w.nkeys = min(max(p.lens[b], 0), p.max_len);
    w.seen0 = w.nkeys - p.T + 1;
    w.lim0 = w.seen0 + first / p.G;
    w.kend = w.seen0 + (first + w.nrow - 1) / p.G;
    w.k = p.kc + ((int64_t)b * p.Hkv + w.kvh) * p.Smax * D;
    w.v = p.vc + ((int64_t)b * p.Hkv + w.kvh) * p.Smax * D;
    w.ks = w.vs = D;
  }
  return w;
}
// Short contexts: a workgroup takes the prefix and the own keys by itself, and no partials are written.
template <int D, int NT>
__global__ void __launch_bounds__(kThreads, 2) prefix_attn_short_kernel(Args p) {
  __shared__ __attribute__((aligned(16))) char smem[kLds];
  by_keys<D, NT, 2>(p, [&](int seg) { return whole_part<D, 16 * NT>(p, blockIdx.x, seg); }, smem);
}
// Many tokens per sequence (a prompt): the same, by rows.
template <int D>
__global__ void __launch_bounds__(kThreads, 2) prefix_attn_long_kernel(Args p) {
  __shared__ __attribute__((aligned(16))) char smem[kLds];
  by_rows<D, true>(p, [&](int seg) { return whole_part<D, tile_rows(kByRows)>(p, blockIdx.x, 1 - seg); }, smem);
}

// one wave per (row, KV head): the ranges that its row sees, then o = sum O 2^(m - M) / sum l 2^(m - M). Bound by its chain of
// loads: 64 sequences 4.9 us, 64 x 5 tokens (21 MB of partials) 7
template <int D>
__global__ void __launch_bounds__(kThreads) prefix_attn_combine_kernel(Args p) {
  constexpr int DPT = D / 64;
  const int lane = threadIdx.x & 63;
  const int RR = p.B * p.T * p.G, nslot = p.np + p.ns;
  const int64_t id = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (id >= (int64_t)RR * p.Hkv) return;
  const int kvh = (int)(id / RR), r = (int)(id % RR);
  const int bt = r / p.G, b = bt / p.T;
  const int seen = min(max(p.lens[b], 0), p.max_len) - p.T + 1 + bt % p.T;
  const int own = seen > 0 ? (seen + p.ochunk - 1) / p.ochunk : 0;
  const int64_t at = id * nslot;
  const float* ml = p.pml + 2 * at;
  const float* po = p.po + at * D + DPT * lane;
  const int n = p.np + own;
  float M = kNegBig;
  for (int s = lane; s < n; s += 64) M = fmaxf(M, ml[2 * s]);
  M = wave_max(M);
  float L = 0.f, a[DPT];
#pragma unroll
  for (int d = 0; d < DPT; ++d) a[d] = 0.f;
#pragma unroll 4
  for (int s = 0; s < n; ++s) {
    const float li = ml[2 * s + 1];
    const float w = li == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[2 * s] - M);
    L += li * w;
#pragma unroll
    for (int d = 0; d < DPT; ++d) a[d] += po[(int64_t)s * D + d] * w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bf16_t* op = p.o + (int64_t)bt * p.os + (int64_t)(kvh * p.G + r % p.G) * D + DPT * lane;
  if constexpr (DPT == 2) *reinterpret_cast<uint32_t*>(op) = pack2(a[0] * inv, a[1] * inv);
  else op[0] = f2bf(a[0] * inv);
}

namespace {
struct Plan {
  int pm, om;               // how each part's workgroups work
  int rtp, rto, np, pchunk, ns, ochunk;
  bool whole;               // both parts by one workgroup, without partials (om: kByRows too)
};
inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
inline int mode_of(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : kByRows; }
Plan make_plan(int B, int T, int G, int Hkv, int P, int max_len) {
  Plan q;
  const int64_t rows = (int64_t)B * T * G;
  // Prompts: with a workgroup for every CU, both parts by rows in one launch where that costs less. In row-keys: by rows, 128-row
  // tiles over prefix and own keys; split, prefix tiles filled from all sequences, own keys in 32-row tiles at half that rate,
  // and partials worth 1100 keys a row; up to 32 rows go by keys. Measured (64 sequences, 32/8 heads of 128; split, by rows): 16 tokens behind 2048 + 500 own
  // 101, 108 us; 24: 136, 110; 48: 260, 217; 33 tokens behind 8192 570, 618; 60: 793, 757; 9 tokens, no prefix, 1000 own 81, 51; where it errs
  // the two are close (9 tokens, 500 + 1000: it splits, 84, 72).
  const int64_t tg = (int64_t)T * G, rt = cdiv(tg, tile_rows(kByRows)), seen = std::max(max_len - T / 2, 0);
  q.whole = tg > 32 && B * Hkv * rt >= 256 && 128 * rt * (P + seen) <= tg * (P + (int64_t)1100) + 64 * cdiv(tg, 32) * seen;
  // Otherwise own keys go by keys, also where 32-row tiles read them more than once: by rows (64 x 16 tokens, 8192 + 1000 keys,
  // measured before P had its remainder) 313 us against 230.
  q.om = q.whole ? kByRows : std::min(2, mode_of(tg));
  q.pm = P > 0 ? mode_of(rows) : q.om;
  q.rtp = P > 0 ? cdiv(rows, tile_rows(q.pm)) : 0;
  q.rto = cdiv(tg, tile_rows(q.om));
  // key ranges of at least `least` keys, as many as make `want` workgroups
  auto ranges = [](int keys, int64_t groups, int want, int least, int& chunk) {
    chunk = least;
    if (keys == 0) return 0;
    const int n = (int)std::min<int64_t>(cdiv(keys, least), std::max<int64_t>(1, want / std::max<int64_t>(1, groups)));
    chunk = cdiv(cdiv(keys, n), 128) * 128;
    return cdiv(keys, chunk);
  };
  // Short contexts: at most 8 steps of 128 keys per wave, and a prefix that it does not hurt to read once per sequence: one step
  // long, or at most one workgroup per CU. Saves the second launch (4 sequences x 4 heads, 500 + 60 keys: 7.3 us against 8.3; 64 x 32/8 heads of 128,
  // 128 + 200 keys: 14.6 against 20.6; 16 of them, 500 + 200 keys: 12.1 against 15.4; one, 400 + 100: 10.1 against 9.3).
  const int64_t groups = (int64_t)B * Hkv * q.rto;
  q.whole = q.whole || (cdiv(P, 128) + cdiv(max_len, 128) <= 8 && (P <= 128 || groups <= 256) &&
                        (max_len <= 256 || groups >= 128));
  if (q.whole) {
    q.np = q.ns = q.pchunk = q.ochunk = 0;
    return q;
  }
  // One workgroup per CU for each part: half as many leave CUs without work, more write and fold more partials (64 x 5 tokens
  // behind 8192 keys, 1000 own, prefix workgroups wanted 128, 256, 512, 1024: 237, 114, 122, 127 us; 16 x 8 tokens behind 4000: 41,
  // 32, 41, 40; for the own keys all within 3 %, for one token behind 8192 with 8 sequences 29, 26, 30, 32).
  q.np = ranges(P, (int64_t)Hkv * q.rtp, 256, q.pm == kByRows ? 256 : 128, q.pchunk);
  q.ns = ranges(max_len, (int64_t)B * Hkv * q.rto, 256, 128, q.ochunk);
  return q;
}
}  // namespace

int64_t prefix_attn_workspace(int B, int T, int Hq, int Hkv, int D, int P, int max_len) {
  const Plan q = make_plan(B, T, Hq / Hkv, Hkv, P, max_len);
  return (int64_t)B * T * Hq * (q.np + q.ns) * (D + 2) * 4;
}

int prefix_attn(const bf16_t* q, int64_t qs, const bf16_t* kp, int64_t kph, int64_t kps, const bf16_t* vp, int64_t vph,
                int64_t vps, int P, const bf16_t* kc, const bf16_t* vc, const int* lens, int max_len, bf16_t* o, int64_t os,
                int B, int T, int Smax, int Hq, int Hkv, int D, float scale, void* workspace, hipStream_t stream) {
  if (B < 0 || T < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || (D != 64 && D != 128) || P < 0 || max_len < 0 || max_len > Smax ||
      (int64_t)B * T * Hq > 0x3fffffff)
    return -1;
  if (B == 0) return 0;
  const int G = Hq / Hkv;
  const Plan pl = make_plan(B, T, G, Hkv, P, max_len);
  Args a;
  a.q = q, a.kp = kp, a.vp = vp, a.kc = kc, a.vc = vc, a.lens = lens;
  a.qs = qs, a.kph = kph, a.kps = kps, a.vph = vph, a.vps = vps;
  a.B = B, a.T = T, a.G = G, a.Hkv = Hkv, a.P = P, a.Smax = Smax, a.max_len = max_len;
  a.pchunk = pl.pchunk, a.np = pl.np, a.rtp = pl.rtp;
  a.ochunk = pl.ochunk, a.ns = pl.ns, a.rto = pl.rto;
  a.sl2 = std::abs(scale) * kLog2e;
  a.flip = scale < 0.f;
  const int64_t parts = (int64_t)B * T * Hq * (pl.np + pl.ns);
  a.o = o, a.os = os;
  a.po = reinterpret_cast<float*>(workspace);
  a.pml = a.po + parts * D;
  if (pl.whole) {
    const int64_t n = (int64_t)B * Hkv * pl.rto;
    if (n > 0x7fffffff) return -1;
#define KOP_PS(DV, NT) \
  if (D == DV && pl.om == NT) prefix_attn_short_kernel<DV, NT><<<(unsigned)n, kThreads, 0, stream>>>(a);
    KOP_PS(128, 1) KOP_PS(128, 2) KOP_PS(64, 1) KOP_PS(64, 2)
#undef KOP_PS
    if (pl.om == kByRows) {
      if (D == 128) prefix_attn_long_kernel<128><<<(unsigned)n, kThreads, 0, stream>>>(a);
      else prefix_attn_long_kernel<64><<<(unsigned)n, kThreads, 0, stream>>>(a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -9;
  }
  const int64_t grid = (int64_t)Hkv * pl.rtp * pl.np + (int64_t)B * Hkv * pl.rto * pl.ns;
  if (grid > 0x7fffffff) return -1;
#define KOP_PA(DV, PM, OM)                                   \
  if (D == DV && pl.pm == PM && pl.om == OM && grid > 0)     \
    prefix_attn_kernel<DV, PM, OM><<<(unsigned)grid, kThreads, 0, stream>>>(a);
  KOP_PA(128, 1, 1) KOP_PA(128, 2, 1) KOP_PA(128, 2, 2) KOP_PA(128, 4, 1) KOP_PA(128, 4, 2)
  KOP_PA(64, 1, 1) KOP_PA(64, 2, 1) KOP_PA(64, 2, 2) KOP_PA(64, 4, 1) KOP_PA(64, 4, 2)
#undef KOP_PA
  const unsigned cg = (unsigned)(((int64_t)B * T * Hq + 3) / 4);
  if (D == 128)
    prefix_attn_combine_kernel<128><<<cg, kThreads, 0, stream>>>(a);
  else
    prefix_attn_combine_kernel<64><<<cg, kThreads, 0, stream>>>(a);
  return hipGetLastError() == hipSuccess ? 0 : -9;
}

}  // namespace kop
