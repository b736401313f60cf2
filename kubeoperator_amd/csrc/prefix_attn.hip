// Attention of a batch that shares a long prefix, for gfx950 (serving): the newest T tokens of every sequence (T = 1: a
// decode step; T > 1: drafted tokens under verification, or a prompt) against
//
//   the prefix   K, V [Hkv, P, D], one copy for the whole batch, seen by every row;
//   the own keys K, V [B, Hkv, Smax, D]: token t of T sees the first lens[b] - (T - 1 - t) of them.
//
// One softmax over both. The rows of ALL sequences meet the prefix together (B T G rows per KV head, G = Hq / Hkv), so its
// keys leave HBM once per row tile instead of once per sequence, and its products have enough rows for the matrix cores.
//
// Pass 1, one launch: a workgroup takes (row tile, key range) of the prefix or of one sequence; its 4 waves take every
// fourth 32-key block. S^T [keys x rows] = K . Q^T and O^T [dims x rows] += V^T . P^T on v_mfma_f32_16x16x32_bf16:
//   * the 16 key rows of product b are keys 8 (i >> 2) + 4 b + (i & 3), so that a lane's scores of the two products are
//     its own P^T operand (keys 8 g .. 8 g + 7 of its row), with no lane exchange;
//   * V goes through an LDS image filled by LDS-DMA (source chunks XOR-permuted by the row) and is read transposed;
//   * running maximum and sum per row (fp32), P rounded to bf16 for the matrix cores: 2^-9 relative per key.
// The next block's K (registers) and V (second LDS image) are in flight while a block is computed; the waves' results
// meet in LDS, and one fp32 partial (O, max, sum) per row and range goes out.
// Pass 2: one wave per (row, head) folds the ranges' partials.
//
// A masked key has weight zero exactly: masked scores never enter the maximum or the sum, keys past the last valid one are
// never read (loads are clamped to it), and in the blocks where some rows see a key and others do not, values that are
// not finite are kept from the rows that do not.
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -3.402823466e38f;

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
// true if one of 8 bf16 values is not finite; `fin` = the values with those replaced by 0, `bad` = 1 in their places, else 0
__device__ __forceinline__ bool split_finite(bf16x8 v, bf16x8& fin, bf16x8& bad) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool nf = (v[i] & 0x7f80) == 0x7f80;
    any |= nf;
    fin[i] = nf ? (short)0 : v[i];
    bad[i] = nf ? (short)0x3f80 : (short)0;
  }
  return any;
}

struct Args {
  const bf16_t *q, *kp, *vp, *kc, *vc;
  const int* lens;
  int64_t qs, kph, kps, vph, vps;
  int B, T, G, Hkv, P, Smax, max_len;
  int pchunk, np, rtp;  // prefix: keys per range, ranges, row tiles of all sequences
  int ochunk, ns, rto;  // own keys: keys per range, ranges, row tiles of one sequence
  float scale_log2;
  float *po, *pml;  // partials [Hkv][B T G][np + ns][D] and [..][2] (max, sum)
};
}  // namespace

template <int D, int NT>  // NT: 16-row tiles per workgroup
__global__ void __launch_bounds__(kThreads) prefix_attn_kernel(Args p) {
  static_assert(D == 64 || D == 128, "head dim");
  constexpr int ROWB = D * 2, NS = D / 32, NC = D / 16, KW = 32, NWV = kThreads / 64, KSTEP = KW * NWV;
  constexpr int IMG = KW * ROWB, VPW = IMG / 1024, SLOTS = ROWB / 16, RPP = 1024 / ROWB;
  // two V images per wave; afterwards the waves' O^T (two of them at a time)
  __shared__ __attribute__((aligned(16))) char s_v[NWV * 2 * IMG > 2 * NT * 16 * D * 4 ? NWV * 2 * IMG : 2 * NT * 16 * D * 4];
  __shared__ float s_ml[NWV][NT * 16][2];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int RR = p.B * p.T * p.G, nslot = p.np + p.ns;
  // ---- which rows and keys
  int kvh, row0, nrow, slot, k0, kend, nkeys, lim0 = 0;  // rows [row0, row0 + nrow) of this KV head; own keys: lim0 = len - T
  bool own_keys;
  const bf16_t *kb_ptr, *vb_ptr;
  int64_t ks, vs;
  int id = blockIdx.x;
  const int nprefix = p.Hkv * p.rtp * p.np;
  if (id < nprefix) {
    own_keys = false;
    const int split = id / (p.Hkv * p.rtp);
    id -= split * p.Hkv * p.rtp;
    kvh = id % p.Hkv;
    row0 = (id / p.Hkv) * NT * 16;
    nrow = min(NT * 16, RR - row0);
    slot = split;
    k0 = split * p.pchunk;
    nkeys = p.P;
    kend = min(p.P, k0 + p.pchunk);
    kb_ptr = p.kp + kvh * p.kph;
    vb_ptr = p.vp + kvh * p.vph;
    ks = p.kps;
    vs = p.vps;
  } else {
    own_keys = true;
    id -= nprefix;
    const int split = id % p.ns;
    id /= p.ns;
    kvh = id % p.Hkv;
    id /= p.Hkv;
    const int rt = id % p.rto, b = id / p.rto;
    const int first = rt * NT * 16;
    nrow = min(NT * 16, p.T * p.G - first);
    row0 = b * p.T * p.G + first;
    slot = p.np + split;
    k0 = split * p.ochunk;
    nkeys = min(max(p.lens[b], 0), p.max_len);
    lim0 = nkeys - p.T + 1;
    const int most = lim0 + (first + nrow - 1) / p.G;  // keys that the tile's last token sees
    kend = min(most, k0 + p.ochunk);
    kb_ptr = p.kc + ((int64_t)b * p.Hkv + kvh) * p.Smax * D;
    vb_ptr = p.vc + ((int64_t)b * p.Hkv + kvh) * p.Smax * D;
    ks = vs = D;
  }
  if (k0 >= kend) return;  // nothing to see: pass 2 does not read this range's partials
  // ---- Q^T operands and each lane's rows
  bf16x8 qf[NT][NS];
  int lim[NT];  // keys that the lane's row sees
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool in = 16 * n + col < nrow;
    const int r = row0 + (in ? 16 * n + col : 0);
    const int bt = r / p.G, h = kvh * p.G + r % p.G;
    const bf16_t* qr = p.q + (int64_t)bt * p.qs + (int64_t)h * D + 8 * g;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      qf[n][s] = *reinterpret_cast<const bf16x8*>(qr + 32 * s);
    }
    lim[n] = own_keys ? lim0 + bt % p.T : nkeys;
  }
  char* const vimg = s_v + wv * (2 * IMG);
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
  auto load_k = [&](int kb, bf16x8 (*kf)[NS]) {
#pragma unroll
    for (int bb = 0; bb < 2; ++bb) {
      const int key = min(kb + 8 * (col >> 2) + 4 * bb + (col & 3), nkeys - 1);
      const bf16_t* kr = kb_ptr + key * ks + 8 * g;
#pragma unroll
      for (int s = 0; s < NS; ++s) kf[bb][s] = *reinterpret_cast<const bf16x8*>(kr + 32 * s);
    }
  };
  auto load_v = [&](int kb, char* img) {
#pragma unroll
    for (int i = 0; i < VPW; ++i) {
      const int r = RPP * i + lane / SLOTS, slot_ = lane % SLOTS;
      const int key = min(kb + r, nkeys - 1);
      glds16(vb_ptr + key * vs + 8 * (slot_ ^ vx<ROWB>(r)), img + 1024 * i);
    }
  };
  auto step = [&](int kb, const bf16x8 (*kf)[NS], int buf) {
    const bool edge = own_keys && kb + KW > lim0;  // some rows see some of these keys and others do not
    bf16x8 pf[NT], pm[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 sc[2];
#pragma unroll
      for (int bb = 0; bb < 2; ++bb) {
        sc[bb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s) sc[bb] = mfma16(kf[bb][s], qf[n][s], sc[bb]);
      }
      float pv[8], mx = kNegBig;
      const int left = lim[n] - kb - 8 * g;  // the lane's keys 0 .. left - 1 are seen
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pv[j] = j < left ? sc[j >> 2][j & 3] * p.scale_log2 : kNegBig;
        mx = fmaxf(mx, pv[j]);
      }
      mx = xor32_max(xor16_max(mx));
      if (__any(mx > m[n])) {
        const float nm = fmaxf(m[n], mx);
        const float al = __builtin_amdgcn_exp2f(m[n] - nm);
        m[n] = nm;
        l[n] *= al;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][c][e] *= al;
      }
      float ls = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pv[j] = j < left ? __builtin_amdgcn_exp2f(pv[j] - m[n]) : 0.f;
        ls += pv[j];
      }
      l[n] += ls;  // the lane's own keys; the four groups' sums meet at the end
      const u32x4 pw = {pack2(pv[0], pv[1]), pack2(pv[2], pv[3]), pack2(pv[4], pv[5]), pack2(pv[6], pv[7])};
      pf[n] = __builtin_bit_cast(bf16x8, pw);
      if (edge) {
#pragma unroll
        for (int j = 0; j < 8; ++j) pm[n][j] = j < left ? (short)0x3f80 : (short)0;
      }
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
        if (edge) {
          bf16x8 fin, bad;
          if (__any(split_finite(vf[c], fin, bad))) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const f32x4 nb = mfma16(bad, pm[n], f32x4{0.f, 0.f, 0.f, 0.f});
              acc[n][c0 + c] = mfma16(fin, pf[n], acc[n][c0 + c]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[n][c0 + c][e] = nb[e] > 0.f ? __builtin_nanf("") : acc[n][c0 + c][e];
            }
            continue;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][c0 + c] = mfma16(vf[c], pf[n], acc[n][c0 + c]);
      }
    }
  };
  // ---- the wave's blocks: the next one's K and V in flight during a block's products
  int kb = k0 + KW * wv;
  bf16x8 ka[2][NS], kn[2][NS];
  if (kb < kend) {
    load_k(kb, ka);
    load_v(kb, vimg);
  }
  while (kb < kend) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (kb + KSTEP < kend) {
      load_k(kb + KSTEP, kn);
      load_v(kb + KSTEP, vimg + IMG);
    }
    step(kb, ka, 0);
    kb += KSTEP;
    if (kb >= kend) break;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (kb + KSTEP < kend) {
      load_k(kb + KSTEP, ka);
      load_v(kb + KSTEP, vimg);
    }
    step(kb, kn, 1);
    kb += KSTEP;
  }
  // ---- the 4 waves' (m, l, O^T) -> one partial: waves 2, 3 into 0, 1, then 1 into 0
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = xor32_sum(xor16_sum(l[n]));
    if (g == 0) {
      s_ml[wv][16 * n + col][0] = m[n];
      s_ml[wv][16 * n + col][1] = l[n];
    }
  }
  __syncthreads();  // every wave is done with its V images
  f32x4* so = reinterpret_cast<f32x4*>(s_v);  // [2][NT][NC][64]
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
        const float wa = l[n] > 0.f ? __builtin_amdgcn_exp2f(m[n] - nm) : l[n] != l[n] ? 1.f : 0.f;
        const float wb = ol > 0.f ? __builtin_amdgcn_exp2f(om - nm) : ol != ol ? 1.f : 0.f;
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
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (16 * n + col >= nrow) continue;
    const int64_t at = ((int64_t)kvh * RR + row0 + 16 * n + col) * nslot + slot;
#pragma unroll
    for (int c = 0; c < NC; ++c) *reinterpret_cast<f32x4*>(p.po + at * D + 16 * c + 4 * g) = acc[n][c];
    if (g == 0) {
      p.pml[2 * at] = m[n];
      p.pml[2 * at + 1] = l[n];
    }
  }
}

// one wave per (row, KV head): the ranges that its row sees, then o = sum O 2^(m - M) / sum l 2^(m - M)
template <int D>
__global__ void __launch_bounds__(kThreads) prefix_attn_combine_kernel(Args p, bf16_t* __restrict__ o, int64_t os) {
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
  bf16_t* op = o + (int64_t)bt * os + (int64_t)(kvh * p.G + r % p.G) * D + DPT * lane;
  if constexpr (DPT == 2) *reinterpret_cast<uint32_t*>(op) = pack2(a[0] * inv, a[1] * inv);
  else op[0] = f2bf(a[0] * inv);
}

namespace {
// row tiles of 16 or 32; ranges of whole 128-key steps, as many as fill the chip
struct Plan {
  int nt, rtp, rto, np, pchunk, ns, ochunk;
};
inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
Plan make_plan(int B, int T, int G, int Hkv, int P, int max_len) {
  Plan q;
  const int64_t rows = (int64_t)B * T * G;
  q.nt = (P > 0 ? rows : (int64_t)T * G) <= 16 ? 1 : 2;
  q.rtp = P > 0 ? cdiv(rows, 16 * q.nt) : 0;
  q.rto = cdiv((int64_t)T * G, 16 * q.nt);
  auto ranges = [](int keys, int64_t groups, int& chunk) {
    if (keys == 0) {
      chunk = 128;
      return 0;
    }
    int n = (int)std::min<int64_t>(cdiv(keys, 128), std::max<int64_t>(1, cdiv(1024, groups)));
    chunk = cdiv(cdiv(keys, n), 128) * 128;
    return cdiv(keys, chunk);
  };
  q.np = ranges(P, (int64_t)Hkv * std::max(q.rtp, 1), q.pchunk);
  q.ns = ranges(max_len, (int64_t)B * Hkv * q.rto, q.ochunk);
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
  a.scale_log2 = scale * kLog2e;
  const int64_t parts = (int64_t)B * T * Hq * (pl.np + pl.ns);
  a.po = reinterpret_cast<float*>(workspace);
  a.pml = a.po + parts * D;
  const int64_t grid = (int64_t)Hkv * pl.rtp * pl.np + (int64_t)B * Hkv * pl.rto * pl.ns;
  if (grid > 0x7fffffff) return -1;
#define KOP_PA(DV, NT)                                                                                        \
  if (D == DV && pl.nt == NT && grid > 0)                                                                     \
    prefix_attn_kernel<DV, NT><<<(unsigned)grid, kThreads, 0, stream>>>(a);
  KOP_PA(128, 1)
  KOP_PA(128, 2)
  KOP_PA(64, 1)
  KOP_PA(64, 2)
#undef KOP_PA
  const unsigned cg = (unsigned)(((int64_t)B * T * Hq + 3) / 4);
  if (D == 128)
    prefix_attn_combine_kernel<128><<<cg, kThreads, 0, stream>>>(a, o, os);
  else
    prefix_attn_combine_kernel<64><<<cg, kThreads, 0, stream>>>(a, o, os);
  return hipGetLastError() == hipSuccess ? 0 : -9;
}

}  // namespace kop
