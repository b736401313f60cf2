// Low-rank adapters of many requests beside one shared projection (serving), for gfx950:
//
//   out[i] = y[i] + scale[j] * b[j] (a[j] x[i]),   j = index[i]        (j outside [0, n): out[i] = y[i])
//   x [M, K], y / out [M, N] bf16 rows; a [n, r, K], b [n, N, r] bf16; index [M] int32; scale [n] fp32
//
// Two launches: the rows' products with a (K split over workgroups, fp32 partials), then their products with b added to y.
// Both take rows as 16-column operands of v_mfma_f32_16x16x32_bf16, in one of two forms:
//   * by adapter (few rows: a decode step): a workgroup collects up to 64 rows (ranks above 64: 32; second launch: 128) of ONE
//     adapter from the index list, so every adapter that occurs is read once, however its rows are scattered; one more "adapter"
//     collects the rows without any;
//   * by rows (many rows: a prefill): 32 (second launch: 64) consecutive rows, the adapters that occur among them taken one after
//     another (lowest row first), each row keeping the result of its own only -- by selection, not by a zero factor, so a request's
//     NaN weights stay with its own rows.
// The low-rank values enter the second product as a bf16 pair (value and remainder: 2^-16 relative), so the only rounding
// that counts is the output's.
//
// Bound by memory for wide projections and long prefills, by its two launches' chains of loads for a decode step. 64 rows, 32
// adapters of rank 16, 4096 x 4096: 4.0 + 5.3 us. 100 rows, 48 adapters of rank 64, 4096 x 28672: 10 us for a (22 MB) and 41 for b
// (3.8 TB/s). 8100 rows in runs, rank 16, 4096 x 6144: 22 us for x (3.0 TB/s) and 54 for y (3.7 TB/s). Both products in one launch
// (every column block makes the low-rank values again) measured 9.5 us against 8.6 for the first, 147 against 39 for the second.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace kop {

namespace {
constexpr int kT = 256;
// Up to this many rows a launch goes by adapter. On scattered rows that form reads every adapter once (600 rows of 64 adapters,
// 4096 x 4096, rank 16: 25 us against 85 by rows); on long runs of one adapter it has fewer, longer workgroups (600 rows of 8
// adapters: 25 us against 17), and past some thousand rows scanning the index list costs more than it saves (1200 rows:
// 59 us against 105 scattered, 38 against 21 in runs).
constexpr int kGroupRows = 1024;

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 zero8() { return bf16x8{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ bf16x8 ld8(const bf16_t* p) { return *reinterpret_cast<const bf16x8*>(p); }

// 16-row groups per workgroup of the first launch: fewer at high ranks, for the registers
constexpr int down_groups(int RB, bool group) { return group ? (RB <= 4 ? 4 : 2) : 2; }
constexpr int up_rows(bool group) { return group ? 128 : 64; }  // rows per workgroup of the second launch

// By adapter: rows number z * ROWS ... of those with index `aj` (aj = n: of those without an adapter), in order, into `list`;
// returns how many there are for this workgroup (0 .. ROWS). Every wave scans the whole index list by itself into a
// list of its own: one round of loads, no barrier.
template <int ROWS>
__device__ __forceinline__ int collect(const int* __restrict__ index, int M, int n, int aj, int z, int* list) {
  const int lane = threadIdx.x & 63;
  int before = -z * ROWS;
  for (int i0 = 0; i0 < M; i0 += 256) {
    int j[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 64 * k + lane;
      j[k] = i < M ? index[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + 64 * k + lane;
      const bool hit = i < M && (aj == n ? j[k] < 0 || j[k] >= n : j[k] == aj);
      const uint64_t mask = __ballot(hit);
      const int at = before + __popcll(mask & ((1ull << lane) - 1));
      if (hit && at >= 0 && at < ROWS) list[at] = i;
      before += __popcll(mask);
    }
  }
  return __builtin_amdgcn_readfirstlane(min(max(before, 0), ROWS));
}
}  // namespace

// ---- part[split][row][r] = a[index[row]] . x[row] over the split's part of K. By adapter: grid (adapters, splits, lists);
// by rows: grid (tiles, splits). The 4 waves take a quarter of the part each and meet in LDS. What counts is loads in flight: a's and
// x's rows go straight to the matrix operands, 64 bytes a row and access, U steps of 32 elements at once.
template <int RB, bool GROUP>  // RB: 16-row blocks of the rank
__global__ void __launch_bounds__(kT) lora_down_kernel(const bf16_t* __restrict__ x, int64_t xs,
                                                       const bf16_t* __restrict__ a, const int* __restrict__ index,
                                                       float* __restrict__ part, int64_t M, int K, int n, int r, int kpart) {
  constexpr int NG = down_groups(RB, GROUP), ROWS = 16 * NG, U = RB <= 2 ? 4 : 2;
  __shared__ f32x4 s_acc[kT / 64 - 1][RB * NG * 64];
  __shared__ int s_lists[kT / 64][ROWS];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  int64_t row[NG];
  int j[NG], ng;
  if constexpr (GROUP) {
    int* const list = s_lists[wv];
    const int cnt = collect<ROWS>(index, (int)M, n, blockIdx.x, blockIdx.z, list);
    if (cnt == 0) return;
    ng = (cnt + 15) / 16;
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      const bool in = 16 * q + col < cnt;
      row[q] = list[in ? 16 * q + col : 0];
      j[q] = in ? (int)blockIdx.x : -1;
    }
  } else {
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    ng = (int)std::min<int64_t>(NG, (M - row0 + 15) / 16);
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      row[q] = row0 + 16 * q + col;
      const bool in = row[q] < M;
      row[q] = in ? row[q] : M - 1;
      j[q] = in ? index[row[q]] : -1;
      if (j[q] >= n) j[q] = -1;
    }
  }
  const bf16_t* xr[NG];
#pragma unroll
  for (int q = 0; q < NG; ++q) xr[q] = x + row[q] * xs + 8 * g;
  const int k0 = blockIdx.y * kpart, k1 = min(K, k0 + kpart);
  const int per = ((k1 - k0 + 127) / 128) * 32;  // a wave's part, a multiple of the product's 32
  const int w0 = k0 + wv * per, w1 = min(k1, w0 + per);
  auto product = [&](int aj, f32x4 (*acc)[RB]) {
    const bf16_t* ar = a + ((int64_t)aj * r + col) * K + 8 * g;
#pragma unroll
    for (int q = 0; q < NG; ++q)
#pragma unroll
      for (int i = 0; i < RB; ++i) acc[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    int k = w0;
    for (; k + 32 * U <= w1; k += 32 * U) {
      bf16x8 af[U][RB], xf[U][NG];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < RB; ++i) af[u][i] = 16 * i + col < r ? ld8(ar + (int64_t)16 * i * K + k + 32 * u) : zero8();
#pragma unroll
      for (int q = 0; q < NG; ++q)
        if (q < ng)
#pragma unroll
          for (int u = 0; u < U; ++u) xf[u][q] = ld8(xr[q] + k + 32 * u);
#pragma unroll
      for (int q = 0; q < NG; ++q)
        if (q < ng)
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RB; ++i) acc[q][i] = mfma16(af[u][i], xf[u][q], acc[q][i]);
    }
    for (; k < w1; k += 32) {
      const bool kin = k + 8 * g < w1;  // K and the parts' ends are multiples of 8
      bf16x8 af[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i) af[i] = kin && 16 * i + col < r ? ld8(ar + (int64_t)16 * i * K + k) : zero8();
#pragma unroll
      for (int q = 0; q < NG; ++q)
        if (q < ng) {
          const bf16x8 xf = kin ? ld8(xr[q] + k) : zero8();
#pragma unroll
          for (int i = 0; i < RB; ++i) acc[q][i] = mfma16(af[i], xf, acc[q][i]);
        }
    }
  };
  f32x4 mine[NG][RB];
  if constexpr (GROUP) {
    product(blockIdx.x, mine);
  } else {
    uint64_t todo[NG];
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      todo[q] = __ballot(j[q] >= 0) & 0xffffull;
#pragma unroll
      for (int i = 0; i < RB; ++i) mine[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    while (true) {
      int aj = -1;
#pragma unroll
      for (int q = NG - 1; q >= 0; --q)
        if (todo[q]) aj = __builtin_amdgcn_readlane(j[q], __builtin_ctzll(todo[q]));
      if (aj < 0) break;
      f32x4 acc[NG][RB];
      product(aj, acc);
#pragma unroll
      for (int q = 0; q < NG; ++q) {
        const bool match = j[q] == aj;
        todo[q] &= ~__ballot(match);
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) mine[q][i][e] = match ? acc[q][i][e] : mine[q][i][e];
      }
    }
  }
  if (wv > 0) {
#pragma unroll
    for (int q = 0; q < NG; ++q)
      if (q < ng)
#pragma unroll
        for (int i = 0; i < RB; ++i) s_acc[wv - 1][(q * RB + i) * 64 + lane] = mine[q][i];
  }
  __syncthreads();
  if (wv != 0) return;
#pragma unroll
  for (int q = 0; q < NG; ++q) {
    if (j[q] < 0) continue;
    float* p = part + ((int64_t)blockIdx.y * M + row[q]) * r + 4 * g;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      f32x4 v = mine[q][i];
#pragma unroll
      for (int w = 0; w < kT / 64 - 1; ++w) {
        const f32x4 o = s_acc[w][(q * RB + i) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += o[e];
      }
      if (16 * i + 4 * g < r) *reinterpret_cast<f32x4*>(p + 16 * i) = v;
    }
  }
}

// ---- out[row] = y[row] + scale b[index[row]] . (sum over splits of part). By adapter: grid (adapters + 1, column blocks,
// lists); by rows: grid (tiles, column blocks). A column block is `chunks` times 256 columns, 64 per wave. The rows'
// low-rank values are put together once per workgroup, in LDS; the waves then go through the rows in groups of 16, the
// next group's y on its way (by rows, 8100 x 6144: all four groups' on their way measured 58 us, y and out by whole 128-byte lines
// through LDS 59, tiles of 16 rows with two steps of y and b on their way 69, this 55: b, 32 bytes a row at rank 16, wants to be read
// for many rows). The 16 b rows of product c are columns n0 + 8 (i >> 2) + (i & 3) + 4 (c & 1) + 32 (c >> 1):
// over the 4 products a lane ends up with two runs of 8 columns of its row, 64 bytes a row and access.
template <int RS, bool GROUP>  // RS: 32-steps of the rank
__global__ void __launch_bounds__(kT) lora_up_kernel(const bf16_t* y, int64_t ys, const bf16_t* __restrict__ b,
                                                     const int* __restrict__ index, const float* __restrict__ scale,
                                                     const float* __restrict__ part, int splits, bf16_t* out, int64_t os,
                                                     int64_t M, int N, int n, int r, int chunks) {
  constexpr int ROWS = up_rows(GROUP), PADR = 32 * RS + 8;  // a row's values and 16 bytes that spread the rows over the banks
  __shared__ __attribute__((aligned(16))) bf16_t s_hi[ROWS * PADR], s_lo[ROWS * PADR];
  __shared__ int s_lists[GROUP ? kT / 64 : 1][ROWS], s_j[ROWS];
  const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  int* const s_list = s_lists[GROUP ? wv : 0];
  int cnt;
  if constexpr (GROUP) {
    const int aj = blockIdx.x;
    if (aj == n && y == out) return;  // in place: the rows without an adapter are there already
    cnt = collect<ROWS>(index, (int)M, n, aj, blockIdx.z, s_list);
    if (cnt == 0) return;
    if (t < ROWS) s_j[t] = t < cnt && aj < n ? aj : -1;
  } else {
    const int64_t row0 = (int64_t)blockIdx.x * ROWS;
    cnt = (int)std::min<int64_t>(ROWS, M - row0);
    if (t < ROWS) {
      const int v = t < cnt ? index[row0 + t] : -1;
      s_j[t] = v < n ? v : -1;
      s_list[t] = (int)(row0 + std::min(t, cnt - 1));
    }
  }
  __syncthreads();
  const int ng = (cnt + 15) / 16;
  int n0 = blockIdx.y * chunks * 256 + wv * 64;
  u32x4 yv[2], yn[2];
  auto load_y = [&](int q, u32x4* v) {  // columns n0 + 8 g .. + 7 and + 32 .. + 39 of the group's rows
    const int nc = n0 + 8 * g;
    if (16 * q + col >= cnt) return;
    const bf16_t* yr = y + (int64_t)s_list[16 * q + col] * ys + nc;
    if (nc < N) v[0] = *reinterpret_cast<const u32x4*>(yr);
    if (nc + 32 < N) v[1] = *reinterpret_cast<const u32x4*>(yr + 32);
  };
  bf16x8 bf[4][RS];
  auto load_b = [&](int aj) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int nr = n0 + 8 * (col >> 2) + (col & 3) + 4 * (c & 1) + 32 * (c >> 1);
      const bf16_t* br = b + ((int64_t)aj * N + nr) * r + 8 * g;
#pragma unroll
      for (int s = 0; s < RS; ++s) bf[c][s] = nr < N && 32 * s + 8 * g < r ? ld8(br + 32 * s) : zero8();
    }
  };
  // the first columns' operands are on their way while the low-rank values are put together
  int cur = GROUP && (int)blockIdx.x < n ? (int)blockIdx.x : -1;  // the adapter whose b operands are loaded
  if (cur >= 0) load_b(cur);
  load_y(0, yv);
  // low-rank values, scaled, as a bf16 value and its remainder; zeros past the rank
  for (int i = t; i < ((cnt + 15) & ~15) * 4 * RS; i += kT) {
    const int q = i / (4 * RS), k = 8 * (i % (4 * RS)), aj = s_j[q];
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, h[8];
    if (aj >= 0 && k < r) {
      const float* p = part + (int64_t)s_list[q] * r + k;
#pragma unroll 4
      for (int c = 0; c < splits; ++c) {
        const f32x4* pc = reinterpret_cast<const f32x4*>(p + (int64_t)c * M * r);
        const f32x4 p0 = pc[0], p1 = pc[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] += p0[e];
          v[4 + e] += p1[e];
        }
      }
      const float sc = scale[aj];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= sc;
    }
    const u32x4 hp = pack8(v);
    unpack8(hp, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = fabsf(h[e]) < INFINITY ? v[e] - h[e] : 0.f;
    *reinterpret_cast<u32x4*>(s_hi + q * PADR + k) = hp;
    *reinterpret_cast<u32x4*>(s_lo + q * PADR + k) = pack8(h);
  }
  __syncthreads();
  for (int ch = 0; ch < chunks; ++ch, n0 += 256) {
    if (n0 >= N) break;
    if (ch > 0) {
      cur = GROUP && (int)blockIdx.x < n ? (int)blockIdx.x : -1;
      if (cur >= 0) load_b(cur);
      load_y(0, yv);
    }
    for (int q = 0; q < ng; ++q) {
      if (q + 1 < ng) load_y(q + 1, yn);
      const int j = s_j[16 * q + col];
      f32x4 mine[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) mine[c] = f32x4{0.f, 0.f, 0.f, 0.f};
      uint64_t todo = __ballot(j >= 0) & 0xffffull;
      if (todo) {
        bf16x8 hi[RS], lo[RS];
#pragma unroll
        for (int s = 0; s < RS; ++s) {
          hi[s] = *reinterpret_cast<const bf16x8*>(s_hi + (16 * q + col) * PADR + 32 * s + 8 * g);
          lo[s] = *reinterpret_cast<const bf16x8*>(s_lo + (16 * q + col) * PADR + 32 * s + 8 * g);
        }
        while (todo) {
          const int aj = __builtin_amdgcn_readlane(j, __builtin_ctzll(todo));
          const bool match = j == aj;
          todo &= ~__ballot(match);
          if (aj != cur) {
            cur = aj;
            load_b(aj);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < RS; ++s) {
              acc = mfma16(bf[c][s], lo[s], acc);
              acc = mfma16(bf[c][s], hi[s], acc);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) mine[c][e] = match ? acc[e] : mine[c][e];
          }
        }
      }
      const int nc = n0 + 8 * g;
      if (16 * q + col < cnt) {
        bf16_t* orow = out + (int64_t)s_list[16 * q + col] * os + nc;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (nc + 32 * h >= N) continue;
          u32x4 v = yv[h];
          if (j >= 0) {
            float f[8];
            unpack8(v, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[e] += mine[2 * h][e];
              f[4 + e] += mine[2 * h + 1][e];
            }
            v = pack8(f);
          }
          *reinterpret_cast<u32x4*>(orow + 32 * h) = v;
        }
      }
      yv[0] = yn[0];
      yv[1] = yn[1];
    }
  }
}

namespace {
struct Plan {
  bool group;
  int splits, kpart;           // parts of K
  unsigned dgx, dgz, ugx, ugz;  // workgroups of each launch besides its splits / column blocks
  int chunks, blocks;          // 256-column chunks per column block, column blocks
};
Plan make_plan(int64_t M, int K, int N, int n, int r) {
  Plan p;
  p.group = M <= kGroupRows;
  const int drows = 16 * down_groups((r + 15) / 16, p.group), urows = up_rows(p.group);
  const int64_t dt = (M + drows - 1) / drows, ut = (M + urows - 1) / urows;
  p.dgx = (unsigned)(p.group ? n : dt), p.dgz = (unsigned)(p.group ? dt : 1);
  p.ugx = (unsigned)(p.group ? n + 1 : ut), p.ugz = (unsigned)(p.group ? ut : 1);
  // workgroups that have rows: adapters cannot outnumber rows
  const int64_t dw = p.group ? std::min<int64_t>(M, n) : dt, uw = p.group ? std::min<int64_t>(M, n) : ut;
  // Parts of K: enough workgroups for the chip, at least 256 elements each. By rows the parts are what keeps loads in flight
  // (8100 rows x 4096: 29 us with 2 parts, 23 with 8); by adapter a part more costs the second launch as much as it saves
  const int64_t want = p.group ? 256 : 1024;
  p.splits = 1;
  while (p.splits < 16 && dw * p.splits < want && K / (2 * p.splits) >= 256) p.splits *= 2;
  p.kpart = ((K + p.splits - 1) / p.splits + 31) & ~31;
  const int nc = (N + 255) / 256;
  // columns per workgroup: about 1024 workgroups, so that they all run at once (8100 rows x 6144: 54 us, with 1.5 times as
  // many 66) and put the low-rank values together as seldom as that allows
  p.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(8, (uw * nc + 1023) / 1024));
  p.blocks = (nc + p.chunks - 1) / p.chunks;
  return p;
}
}  // namespace

int64_t lora_workspace(int64_t M, int K, int N, int n, int r) { return (int64_t)make_plan(M, K, N, n, r).splits * M * r * 4; }

int lora_add(const bf16_t* y, int64_t ys, const bf16_t* x, int64_t xs, const bf16_t* a, const bf16_t* b,
             const int* index, const float* scale, bf16_t* out, int64_t os, int64_t M, int K, int N, int n, int r,
             void* workspace, hipStream_t stream) {
  if (K < 8 || K % 8 || N < 8 || N % 8 || r < 8 || r % 8 || r > kLoraMaxRank || n < 0 || M < 0 || xs % 8 || ys % 8 ||
      os % 8 || M > kLoraMaxRows || (N + 255) / 256 > 65535)
    return -1;
  if (M == 0) return 0;
  const Plan p = make_plan(M, K, N, n, r);
  float* part = reinterpret_cast<float*>(workspace);
  const dim3 gd(p.dgx, p.splits, p.dgz), gu(p.ugx, p.blocks, p.ugz);
#define KOP_DOWN(RB)                                                                                             \
  case RB:                                                                                                       \
    if (p.group) lora_down_kernel<RB, true><<<gd, kT, 0, stream>>>(x, xs, a, index, part, M, K, n, r, p.kpart);  \
    else lora_down_kernel<RB, false><<<gd, kT, 0, stream>>>(x, xs, a, index, part, M, K, n, r, p.kpart);         \
    break;
  if (n > 0) switch ((r + 15) / 16) {
      KOP_DOWN(1) KOP_DOWN(2) KOP_DOWN(3) KOP_DOWN(4) KOP_DOWN(5) KOP_DOWN(6) KOP_DOWN(7) KOP_DOWN(8)
    }
#undef KOP_DOWN
#define KOP_UP(RS)                                                                                                  \
  case RS:                                                                                                          \
    if (p.group)                                                                                                    \
      lora_up_kernel<RS, true><<<gu, kT, 0, stream>>>(y, ys, b, index, scale, part, p.splits, out, os, M, N, n, r,  \
                                                    p.chunks);                                                    \
    else                                                                                                            \
      lora_up_kernel<RS, false><<<gu, kT, 0, stream>>>(y, ys, b, index, scale, part, p.splits, out, os, M, N, n, r, \
                                                     p.chunks);                                                   \
    break;
  switch ((r + 31) / 32) { KOP_UP(1) KOP_UP(2) KOP_UP(3) KOP_UP(4) }
#undef KOP_UP
  return hipGetLastError() == hipSuccess ? 0 : -9;
}

}  // namespace kop
