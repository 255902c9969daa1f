// Products with 4-bit weights (quantized_weight.hip's layout):
//   linear  y = x W^T (+ r)
//   gated   h = silu(x G^T) * (x U^T), both projections in one kernel
// and the feed-forward block y = h D^T (+ r) of the two.
//
// The weight's values are exact in bf16 and go to v_mfma_f32_16x16x32_bf16 as they
// are; what x has more bits than bf16 goes as further products: x is the sum of
// bf16 pieces, two for fp16 (11 bits) and three for fp32 (24 bits), each the leading
// bits of what is left, so the sum is x itself (fp32 below 2^-110: to the nearest 2^-133,
// bf16's lowest step; pieces held at other scales would take a conversion of the weight for
// each).  With scales from 2^-15 to 1 the weight's values are exact in fp16 too, and rows of
// fp16 go to v_mfma_f32_16x16x32_f16 as they are, in pieces where one is another: in that
// block of 128 columns alone (the kernel of few rows), or with all of the rows of the weight
// that a wave has (of many).  Sums are fp32 and are rounded once, with the residual added.
// The gated product h is rounded to one bf16 piece for bf16 x (2^-8, as the model's own
// activation: y is off by sqrt(2) times its own rounding, 0.0023 of its norm for 0.0017, and a
// second piece is the second half's products again, 193 of 605 us with 32768 rows of 1024 and a
// width of 3584), else to as many pieces as x has: 2^-15 for fp16, whose range h may leave, and
// 2^-22 for fp32.

#include <type_traits>

#include "quantized_common.h"

namespace {

using namespace kad_q4;

template <typename T> constexpr int kPieces = sizeof(T) == 4 ? 3 : 2;
template <> constexpr int kPieces<bf16_t> = 1;

// what the kernel of many rows reads of x: rows of 16 bits as they are, fp32 in pieces
template <typename T> constexpr int kPlanes = sizeof(T) == 2 ? 1 : kPieces<T>;

// f as the sum of P bf16 pieces, the leading 8 bits each time (truncated, so that no
// piece is infinite where f is finite) and the last one rounded.  Infinities and NaN
// are one piece.
template <int P>
__device__ __forceinline__ void split(float f, bf16_t (&p)[P]) {
  if constexpr (P == 1) {
    p[0] = f2bf(f);
  } else {
    const float whole = f;
#pragma unroll
    for (int i = 0; i < P - 1; ++i) {
      const uint32_t hi = __float_as_uint(f) & 0xffff0000u;
      p[i] = (bf16_t)(hi >> 16);
      f -= __uint_as_float(hi);
    }
    p[P - 1] = f2bf(f);
    if (!(fabsf(whole) < INFINITY)) {
      p[0] = f2bf(whole);
#pragma unroll
      for (int i = 1; i < P; ++i) p[i] = 0;
    }
  }
}

// Rows of x as P bf16 pieces [P][M][KP], or (P = 1) rows of 16 bits as they are; zeros past
// column K.  8 elements a thread.  (1024 x 4096 fp32, 42 MB: 8.6 us, 4.9 TB/s; 1726 x 4560 bf16,
// 31 MB: 9.5 us.  Split in the products' kernel instead, they would be split by each column
// tile again.)
template <typename T, int P>
__global__ __launch_bounds__(256) void split_rows_kernel(const T* __restrict__ x, int64_t ldx,
                                                         uint16_t* __restrict__ out, int M, int K,
                                                         int KP) {
  const int per_row = KP / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = i / per_row;
  if (m >= M) return;
  const int k = (int)(i - m * per_row) * 8;
  // one access, wherever the row begins; at its end the last 8, and the thread's own below
  T v[8];
  if (K >= 8) __builtin_memcpy(v, x + m * ldx + min(k, K - 8), sizeof(v));
  if (k + 8 > K) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < K ? x[m * ldx + k + e] : T(0);
  }
  uint32_t w[P][4];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint16_t p[P];
    if constexpr (P == 1) p[0] = __builtin_bit_cast(uint16_t, v[e]);
    else split<P>(Elem<T>::to_f(v[e]), p);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (e & 1) w[j][e / 2] |= (uint32_t)p[j] << 16;
      else w[j][e / 2] = p[j];
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j)
    *(u32x4*)(out + ((int64_t)j * M + m) * KP + k) = u32x4{w[j][0], w[j][1], w[j][2], w[j][3]};
}

struct Args {
  const void* x;             // rows of T, or their pieces: (p, m, k) at x[p * xp + m * ldx + k]
  int64_t ldx, xp;
  const uint8_t* codes[2];   // the weight, or gate and up
  const uint8_t* scales[2];
  const void* r;             // residual (linear; may be null)
  int64_t ldr;
  void* y;                   // linear: rows of T; gated: pieces, (p, m, n) as for x
  int64_t ldy, yp;
  int M, N, K, KB;           // KB blocks of 128 columns
  int cols;                  // columns that are written: N, or (gated) N padded to 128
  int order;                 // few rows: 1 where an XCD has all columns of a share of the row
                             // tiles, 2 all rows of a share of the columns, 0 the grid's order
};

// Workgroup b of n in 8 runs, each of an XCD (which workgroups b, b + 8, .. are on).
__device__ __forceinline__ int xcd_run(int b, int n) {
  const int x = b % 8;
  return x * (n / 8) + min(x, n % 8) + b / 8;
}

// a word of 8 codes times its group's scale, as an MFMA operand
__device__ __forceinline__ bf16x8 operand(uint32_t codes, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// the same in fp16, for scales from 2^-15 to 1
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f16x8 operand_f16(uint32_t codes, float scale) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ float silu_of(float g) {
  if constexpr (sizeof(T) == 4) return g / (1.0f + expf(-g));
  else return silu_f(g);
}

// The residual of outputs (m, n .. n + 3): loaded early, on no condition of the lane's, so
// that the loads of a tile are in flight together.  (Lanes that have no whole four, at the
// row's end or past it, read others' here and their own in finish.)
template <typename T>
struct Residual {
  T v[4];
  __device__ __forceinline__ void load(const Args& a, int m, int n) {
    __builtin_memcpy(v, (const T*)a.r + min(m, a.M - 1) * a.ldr + min(n, a.N - 4), sizeof(v));
  }
};

// Outputs (m, n .. n + 3) from their sums: s[0], or the gate's and the up's.
template <typename T, bool GATED>
__device__ __forceinline__ void finish(const Args& a, int m, int n, const f32x4* s,
                                       const Residual<T>& res) {
  if (m >= a.M || n >= a.cols) return;
  if constexpr (GATED) {
    constexpr int P = kPieces<T>;
    bf16_t p[4][P];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      split<P>(n + i < a.N ? silu_of<T>(s[0][i]) * s[1][i] : 0.f, p[i]);
#pragma unroll
    for (int j = 0; j < P; ++j)
      *(u32x2*)((bf16_t*)a.y + j * a.yp + m * a.ldy + n) =
          u32x2{p[0][j] | (uint32_t)p[1][j] << 16, p[2][j] | (uint32_t)p[3][j] << 16};
  } else {
    T* y = (T*)a.y + m * a.ldy + n;
    if (n + 4 <= a.N) {  // one access, wherever it begins
      T v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = Elem<T>::from_f(a.r ? s[0][i] + Elem<T>::to_f(res.v[i]) : s[0][i]);
      __builtin_memcpy(y, v, sizeof(v));
    } else {
      const T* r = (const T*)a.r + (a.r ? m * a.ldr + n : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) y[i] = Elem<T>::from_f(a.r ? s[0][i] + Elem<T>::to_f(r[i]) : s[0][i]);
    }
  }
}

// A lane of the product has 4 neighbours of a row of its own, so what a wave stores at once
// would lie in 16 rows.  NT tiles of sums (16 rows x 16 columns, side by side) change places
// through LDS first: taken lane by lane they are 16 / NT whole rows of 16 NT columns a time.
// Neither side has bank conflicts.
template <int NT>
struct Sums {
  static __device__ __forceinline__ int slot(int tile, int row, int quad) {
    return tile * 64 + quad * 16 + (row ^ (quad * 4 + tile * (4 / NT)));
  }
  // the q-th of 64 NT quads of columns, rows first
  int tile, row, quad;
  __device__ __forceinline__ explicit Sums(int q)
      : tile(q % (4 * NT) / 4), row(q / (4 * NT)), quad(q % 4) {}
  __device__ __forceinline__ int slot() const { return slot(tile, row, quad); }
};

// A wave's blocks of 128 columns: codes and scales of NW row blocks of the weight(s).
template <int NW>
struct Codes {
  u32x4 c[NW];
  uint32_t s[NW];  // a row's scales of the block's four groups
};
__device__ __forceinline__ float scale_of(uint32_t s, int j) {
  return __uint_as_float((s >> (8 * j) & 255u) << 23);
}
__device__ __forceinline__ bf16x8 operand(u32x4 c, uint32_t s, int j) {
  return operand(c[j], scale_of(s, j));
}
// nonzero where a word of scales has one that is not from 2^-15 to 1
__device__ __forceinline__ uint32_t not_f16(uint32_t s) { return (s & 0xf0f0f0f0u) ^ 0x70707070u; }
// whether fp16 holds a block's values: the same for all lanes
template <int NW>
__device__ __forceinline__ bool fits_f16(const Codes<NW>& f) {
  uint32_t other = 0;
#pragma unroll
  for (int n = 0; n < NW; ++n) other |= not_f16(f.s[n]);
  return !__any(other != 0);
}

// The row blocks' codes and scales, by their first block of 128 columns.
template <int NW>
struct Source {
  const uint8_t* c[NW];
  const uint8_t* s[NW];
  // whether fp16 holds the values of all KB blocks of columns
  __device__ __forceinline__ bool fits_f16(int KB, int lane) const {
    uint32_t other = 0;
#pragma unroll
    for (int n = 0; n < NW; ++n)
      for (int i = lane; i < KB * 4; i += 64) {
        const u32x4 v = ((const u32x4*)s[n])[i];
        other |= not_f16(v[0]) | not_f16(v[1]) | not_f16(v[2]) | not_f16(v[3]);
      }
    return !__any(other != 0);
  }
  __device__ __forceinline__ void load(Codes<NW>& f, int kb, int lane) const {
#pragma unroll
    for (int n = 0; n < NW; ++n) {
      f.c[n] = *(const u32x4*)(c[n] + (int64_t)kb * 1024 + lane * 16);
      f.s[n] = *(const uint32_t*)(s[n] + (int64_t)kb * 64 + (lane & 15) * 4);
    }
  }
};
// blocks first .. first + NW / W - 1 of each of W weights (past the last: the last)
template <int NW, int W>
__device__ __forceinline__ Source<NW> source(const Args& a, int first) {
  Source<NW> f;
  const int NB = (a.N + 15) / 16;
#pragma unroll
  for (int n = 0; n < NW; ++n) {
    const int w = n / (NW / W), nb = min(first + n % (NW / W), NB - 1);
    f.c[n] = a.codes[w] + (int64_t)nb * a.KB * 1024;
    f.s[n] = a.scales[w] + (int64_t)nb * a.KB * 64;
  }
  return f;
}

// 8 neighbours of a row of fp16 or fp32 (2 V words) as MFMA operands: split() of all, the
// leading halves by byte permutes, the rest by packed conversions.  Nothing is left of an
// infinity, which the first piece holds: any other number in its place, times a weight, may
// pass fp32's range with the other sign.  fp32 selects (what is left of a NaN is one, also
// where its leading half is an infinity's).  fp16 takes magnitudes, as the larger of a NaN and
// 0 is 0, and the signs in pairs: its select is in the way of the products (300 x 4096 x 2048
// 16.8 us, so 13.1).
template <typename T>
__device__ __forceinline__ void pieces_of(const u32x4 (&v)[sizeof(T) / 2],
                                          bf16x8 (&p)[kPieces<T>]) {
  constexpr int P = kPieces<T>;
  if constexpr (P == 1) {
    p[0] = as_bf16x8(v[0]);
  } else {
    float f[8];
    T t[8];
    __builtin_memcpy(t, v, sizeof(v));
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)t[i];
    u32x4 w[P];
#pragma unroll
    for (int q = 0; q < P - 1; ++q)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const uint32_t lo = __float_as_uint(f[i]), hi = __float_as_uint(f[i + 1]);
        w[q][i / 2] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
#pragma unroll
        for (int k = i; k < i + 2; ++k) {
          const float head = __uint_as_float(__float_as_uint(f[k]) & 0xffff0000u);
          if constexpr (P == 2) f[k] = fmaxf(fabsf(f[k]) - fabsf(head), 0.f);
          else f[k] = q == 0 && fabsf(f[k]) == INFINITY ? 0.f : f[k] - head;
        }
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[P - 1][i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
      if constexpr (P == 2) w[1][i] |= w[0][i] & 0x80008000u;
    }
#pragma unroll
    for (int q = 0; q < P; ++q) p[q] = as_bf16x8(w[q]);
  }
}

// Few rows: a workgroup has 16 MT rows of x and 16 NT columns of y, K split over its KS
// waves, whose sums meet in LDS.  Codes and rows are loaded D blocks of 128 columns ahead,
// into registers.  A lane of the product holds 16 bytes of a row of its own, which the cache
// would serve one by one; so rows are loaded in runs of 256 bytes and more, and take their
// places through LDS, of which each wave has a part that no other touches.  RAW: x is the
// rows themselves, whatever their type, alignment and length; else their pieces, padded to
// whole blocks.  R: rows of a tile that are loaded, 16, or 4 where x has no more (the
// product's other columns repeat them).
// One row takes what the codes take to arrive (1 x 248320 x 1024, 135 MB: 24 us, 5.6 TB/s),
// or, where they are few, a launch and a wave's walk over its blocks (1 x 1024 x 3584: 3.8 us,
// 0.4 of it the codes at 5 TB/s; 10 x 8192 x 1024 4.2).  More rows take what comes through
// the L2 caches: each workgroup reads its rows and codes itself (64 x 8192 x 8192, 256
// workgroups of 32 x 64: 20 us, from the caches 17.6, 0.13 GB of rows and 0.07 GB of codes,
// 11 TB/s).  fp32 rows are three times the products, and their pieces are made in each
// workgroup: 300 x 1024 x 2048 12.6 us, 0.30 PFLOP/s of the three.  (Traced kernels, with a
// residual and, where nothing else is said, weights from beyond the caches.)
template <typename T, bool RAW, bool GATED, int MT, int NT, int KS, int D, int R>
__global__ __launch_bounds__(64 * KS) void q4_stream_kernel(Args a) {
  constexpr int P = kPieces<T>, W = GATED ? 2 : 1, NW = W * NT;
  constexpr bool HALF = RAW && std::is_same_v<T, _Float16>;
  // a block's rows: planes (the pieces) of 16 MT rows of RB bytes, loaded L x 1 KB a tile
  constexpr int PLANES = RAW ? 1 : P, RB = RAW ? 128 * (int)sizeof(T) : 256;
  constexpr int CPR = RB / 16, RPI = 64 / CPR, L = R / RPI;
  static_assert(R == 16 || (R == 4 && MT == 1), "whole tiles, or one of 4 rows");
  constexpr int kRows = PLANES * MT * R * RB, kSums = NW * MT * 1024;
  constexpr int kWave = kRows > kSums ? kRows : kSums;
  __shared__ __attribute__((aligned(1024))) char lds[KS * kWave];
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int nt = blockIdx.x, mt = blockIdx.y;
  if (a.order) {
    const int lid = xcd_run(mt * gridDim.x + nt, gridDim.x * gridDim.y);
    const int n = a.order == 1 ? gridDim.x : gridDim.y, q = lid / n, r = lid - q * n;
    mt = a.order == 1 ? q : r, nt = a.order == 1 ? r : q;
  }
  const int m0 = mt * (16 * MT);
  nt *= NT;
  char* own = lds + wave * kWave;
  f32x4 acc[NW][MT];
#pragma unroll
  for (int n = 0; n < NW; ++n)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the wave's share of y: quads of columns t * 64 + lane of the row tiles, t = wave, wave + KS, ..
  constexpr int kShare = (NT * MT + KS - 1) / KS;
  Residual<T> res[kShare];
  if (!GATED && a.r && a.N >= 4) {
#pragma unroll
    for (int u = 0; u < kShare; ++u) {
      const int t = u * KS + wave;
      const Sums<NT> at(t % NT * 64 + lane);
      res[u].load(a, m0 + t / NT * 16 + at.row, (nt + at.tile) * 16 + at.quad * 4);
    }
  }
  const Source<NW> src = source<NW, W>(a, nt);
  constexpr int kItem = RAW ? sizeof(T) : 2;
  const int chunk = lane % CPR;
  const char* row[MT][L];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < L; ++t)
      row[i][t] = (const char*)a.x + chunk * 16 +
                  (int64_t)min(m0 + i * 16 + t * RPI + lane / CPR, a.M - 1) * a.ldx * kItem;
  struct Block {
    Codes<NW> w;
    u32x4 x[PLANES][MT][L];
  };
  auto load = [&](Block& b, int kb) {
    src.load(b.w, kb, lane);
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < L; ++t)  // (rows may begin anywhere: no alignment is needed)
          __builtin_memcpy(&b.x[p][i][t], row[i][t] + (p * a.xp + kb * 128) * kItem, 16);
  };
  // 16 bytes, c-th of row r, are at c ^ r: neither side has bank conflicts
  const int rr = fr % R;
  auto mul = [&](const Block& b) {
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const int r = t * RPI + lane / CPR;
          *(u32x4*)(own + ((p * MT + i) * R + r) * RB + (chunk ^ r) * 16) = b.x[p][i][t];
        }
    if constexpr (HALF) {
      if (__builtin_expect(fits_f16(b.w), true)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f16x8 xf[MT];
#pragma unroll
          for (int i = 0; i < MT; ++i)
            xf[i] = *(const f16x8*)(own + (i * R + rr) * RB + ((j * 4 + fq) ^ rr) * 16);
#pragma unroll
          for (int n = 0; n < NW; ++n) {
            const f16x8 wf = operand_f16(b.w.c[n][j], scale_of(b.w.s[n], j));
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[n][i] = mfma_f16(wf, xf[i], acc[n][i]);
          }
        }
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 xf[MT][P];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if constexpr (RAW) {
          constexpr int V = sizeof(T) / 2;
          u32x4 v[V];
#pragma unroll
          for (int h = 0; h < V; ++h)
            v[h] = *(const u32x4*)(own + (i * R + rr) * RB + (((j * 4 + fq) * V + h) ^ rr) * 16);
          pieces_of<T>(v, xf[i]);
        } else {
#pragma unroll
          for (int p = 0; p < P; ++p)
            xf[i][p] = as_bf16x8(
                *(const u32x4*)(own + ((p * MT + i) * R + rr) * RB + ((j * 4 + fq) ^ rr) * 16));
        }
      }
#pragma unroll
      for (int n = 0; n < NW; ++n) {
        const bf16x8 wf = operand(b.w.c[n], b.w.s[n], j);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[n][i] = mfma16x16x32(wf, xf[i][p], acc[n][i]);
      }
    }
  };
  // this wave's whole blocks: wave, wave + KS, ..  (No load below hangs on a condition: the
  // compiler's waits would then allow for its absence, and nothing stay in flight.)
  const int whole = RAW ? a.K / 128 : a.KB;
  const int n = wave < whole ? (whole - wave + KS - 1) / KS : 0;
  if (n > 0) {
    Block b[D];
    auto fill = [&](Block& f, int i) { load(f, wave + KS * min(i, n - 1)); };
#pragma unroll
    for (int d = 0; d < D; ++d) fill(b[d], d);
    int i = 0;
    for (; i + D < n; i += D)
#pragma unroll
      for (int d = 0; d < D; ++d) {
        mul(b[d]);
        fill(b[d], i + D + d);
      }
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (i + d < n) mul(b[d]);
  }
  if constexpr (RAW) {
    if (whole < a.KB && whole % KS == wave) {  // the last columns, which are no whole block
      Block f;
      src.load(f.w, whole, lane);
      constexpr int E = 16 / sizeof(T);
      const int left = a.K - whole * 128 - chunk * E;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < L; ++t) {
          const T* from = (const T*)(row[i][t]) + whole * 128;
          T part[E];
#pragma unroll
          for (int e = 0; e < E; ++e) part[e] = e < left ? from[e] : T(0);
          __builtin_memcpy(&f.x[0][i][t], part, 16);
        }
      mul(f);
    }
  }
  // a wave's sums take the place of its rows
  auto sums = [&](int k, int w, int i) {
    return (f32x4*)(lds + k * kWave) + (i * NW + w * NT) * 64;
  };
#pragma unroll
  for (int n = 0; n < NW; ++n)
#pragma unroll
    for (int i = 0; i < MT; ++i)
      sums(wave, n / NT, i)[Sums<NT>::slot(n % NT, fr, fq)] = acc[n][i];
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kShare; ++u) {
    const int t = u * KS + wave;
    if (t >= NT * MT) break;
    const Sums<NT> at(t % NT * 64 + lane);
    f32x4 s[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      s[w] = sums(0, w, t / NT)[at.slot()];
#pragma unroll
      for (int k = 1; k < KS; ++k) s[w] += sums(k, w, t / NT)[at.slot()];
    }
    finish<T, GATED>(a, m0 + t / NT * 16 + at.row, (nt + at.tile) * 16 + at.quad * 4, s, res[u]);
  }
}

typedef __attribute__((address_space(3))) void lds_void_t;

// what is loaded in place of columns past the rows' end
__device__ __attribute__((aligned(16))) const bf16_t kZeros[8] = {};

// Many rows: a workgroup has 16 MT rows of x, which 4 waves share through LDS in slices of
// BK columns, and each of the waves NW row blocks of the weight (gated: half of them the
// gate's), whose codes it reads by itself, D - 1 blocks of 128 ahead.  A ring of SLOTS slices
// is filled by direct loads.
// The matrix unit bounds the largest tile, for about half its time: a workgroup's four waves
// wait for a slice together, and what converts codes shares the issue slots (8192 x 8192 x
// 8192 bf16 741 us, 1.48 PFLOP/s; 32768 x 1024 x 3584 192 us, 1.25; the unit alone, 2.37).  Smaller
// calls are bound by what the tiles load through the L2 caches: 50 x 248320 x 1024 in tiles of
// 64 x 256 42 us, 3.2 TB/s of codes, as much of rows, and 50 MB of y and the residual.  fp16
// 2048 x 8192 x 4096 114 us, 1.2 PFLOP/s; fp32 1024 x 4096 x 4096 77 us and 8.4 for the
// pieces, 1.3 PFLOP/s of its three products.  (Traced kernels, with a residual, weights in the
// caches; from beyond them 1.01 to 1.1 times as long.)
// HALF: x is rows of fp16, else pieces.  RAGGED: rows that end inside a block of columns, at
// whole 16 bytes (1726 x 960 x 4560 25 us, copied and padded first 33; where all kernels
// looked for an end the others took 2 % longer, the largest tile twice as long for registers).
template <typename T, bool HALF, bool RAGGED, bool GATED, int MT, int NW, int BK, int SLOTS, int D>
__global__ __launch_bounds__(256, 2) void q4_tile_kernel(Args a, int mtiles, int ntiles) {
  constexpr int P = HALF ? 1 : kPieces<T>, W = GATED ? 2 : 1, NT = NW / W;
  constexpr int BM = 16 * MT, GROUP = 8;
  constexpr int CPR = BK / 8, RPI = 64 / CPR;  // chunks of 8 in a slice row, rows a load
  constexpr int LPW = BM / RPI / 4;            // loads per wave and slice
  constexpr int HALVES = 128 / BK, STEPS = BK / 32;
  // PIPE: a slice goes to registers while the one before multiplies
  constexpr bool PIPE = MT <= 4;
  constexpr int AHEAD = PIPE ? SLOTS : SLOTS - 1;  // slices loaded ahead
  // Rows of fp16 in pieces: whether a row block's operand is made anew for each row tile.  Held
  // for all of them it takes registers from the rows' addresses, which then come from scratch
  // memory in either walk (fp16 4000 x 2880 x 2880: 109 us, made anew 78; in pieces 249 and 197).
  // Rows of whole blocks need fewer addresses (in pieces 2048 x 8192 x 4096 329 us, anew 339).
  constexpr bool ANEW = HALF && RAGGED && MT * NW >= 16;
  // loads that a wave issues after a slice's own before it waits for that slice: those of
  // SLOTS - 2 later ones, and the codes' and scales' of the blocks that begin meanwhile
  constexpr int LATER = LPW * (SLOTS - 2) + 2 * NW * ((SLOTS - 2) / (HALVES * P));
  static_assert(D * HALVES * P % SLOTS == 0 && SLOTS % 2 == 0,
                "a slice's slot and registers are known when the D blocks are unrolled");
  static_assert(LPW * RPI * 4 == BM && LATER < 64, "loads");
  __shared__ __attribute__((aligned(1024))) bf16_t ring[SLOTS][BM * BK];
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lid = xcd_run(blockIdx.x, gridDim.x);
  // runs of 8 row tiles a column tile, so that an XCD's L2 holds what its run shares
  const int g0 = lid / (GROUP * ntiles) * GROUP, in_group = lid - g0 * ntiles;
  const int gm = min(GROUP, mtiles - g0);
  const int m0 = (g0 + in_group % gm) * BM, nt = (in_group / gm * 4 + wave) * NT;

  // Chunk c (of 8 columns) of slice row r is at chunk c ^ swizzle(r), so that the 16 rows
  // of a fragment read hit 16 distinct bank groups.
  auto swizzle = [](int r) { return BK == 64 ? (r >> 1) & 7 : r & 15; };
  const bf16_t* src[LPW];
#pragma unroll
  for (int i = 0; i < LPW; ++i) {
    const int r = (wave + 4 * i) * RPI + lane / CPR;
    src[i] = (const bf16_t*)a.x + (int64_t)min(m0 + r, a.M - 1) * a.ldx +
             ((lane % CPR) ^ swizzle(r)) * 8;
  }
  const int col = ((lane % CPR) ^ swizzle(wave * RPI + lane / CPR)) * 8;  // (of every load)
  // slice t (counted from a block kb's first) to its slot; past the last block, that one's
  // again (never multiplied)
  auto issue = [&](int kb, int t) {
    const int p = t % P, h = t / P % HALVES;
    const int64_t k = (int64_t)min(kb + t / (P * HALVES), a.KB - 1) * 128 + h * BK;
    const int64_t from = k + p * a.xp;
    const bool in = !RAGGED || (int)k + col < a.K;
#pragma unroll
    for (int i = 0; i < LPW; ++i)
      __builtin_amdgcn_global_load_lds(
          (__attribute__((address_space(1))) void*)(in ? src[i] + from : kZeros),
          (lds_void_t*)(ring[t % SLOTS] + (wave + 4 * i) * RPI * BK), 16, 0, 0);
  };
  const Source<NW> w = source<NW, W>(a, nt);
  f32x4 acc[NW][MT];
#pragma unroll
  for (int n = 0; n < NW; ++n)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  Codes<NW> codes[D];
#pragma unroll
  for (int d = 0; d < D - 1; ++d) w.load(codes[d], min(d, a.KB - 1), lane);
#pragma unroll
  for (int t = 0; t < AHEAD; ++t) issue(0, t);
  const bool fits = HALF && w.fits_f16(a.KB, lane);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  bf16x8 frags[PIPE ? 2 : 1][STEPS][MT];
  auto read = [&](bf16x8 (&f)[STEPS][MT], int at) {
    const bf16_t* x = ring[at] + fr * BK;
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i)  // (rows differ by multiples of 16)
        f[j][i] = as_bf16x8(*(const u32x4*)(x + i * 16 * BK + ((j * 4 + fq) ^ swizzle(fr)) * 8));
  };
  if constexpr (PIPE) {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(frags[0], 0);
  }
  // F16: the row blocks' values are all fp16's, and the rows multiply as they are
  auto walk = [&](auto f16) {
    constexpr bool F16 = decltype(f16)::value;
    auto made = [&](const Codes<NW>& f, int j, int n) {
      if constexpr (F16) return operand_f16(f.c[n][j], scale_of(f.s[n], j));
      else return operand(f.c[n], f.s[n], j);
    };
    for (int kb0 = 0; kb0 < a.KB; kb0 += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int kb = kb0 + d;
        if (kb >= a.KB) break;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const int t = (d * HALVES + h) * P + p, set = PIPE ? t % 2 : 0;
            // PIPE: the next slice has landed (later ones may be in flight), and every wave
            // has this one in registers, so its slot takes the slice SLOTS ahead.  Else: this
            // slice has landed, and every wave has read the one before.
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(LATER) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (h == 0 && p == 0)
              w.load(codes[(d + D - 1) % D], min(kb + D - 1, a.KB - 1), lane);
            if constexpr (PIPE) read(frags[set ^ 1], (t + 1) % SLOTS);
            issue(kb0, t + AHEAD);
            if constexpr (!PIPE) read(frags[0], t % SLOTS);
            if constexpr (HALF && !F16) {
#pragma unroll
              for (int j = 0; j < STEPS; ++j)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                  bf16x8 xf[kPieces<T>];
                  pieces_of<T>({__builtin_bit_cast(u32x4, frags[set][j][i])}, xf);
#pragma unroll
                  for (int n = 0; n < NW; ++n) {
                    if constexpr (ANEW) asm volatile("" : "+v"(codes[d].s[n]));
#pragma unroll
                    for (int q = 0; q < kPieces<T>; ++q)
                      acc[n][i] = mfma16x16x32(made(codes[d], h * STEPS + j, n), xf[q], acc[n][i]);
                    if constexpr (ANEW) __builtin_amdgcn_sched_barrier(0);
                  }
                  __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
                }
            } else {
              // the next row block's operand is made among the products of the present one:
              // a conversion right before the product that reads it holds up the matrix unit
              auto wf = made(codes[d], h * STEPS, 0);
#pragma unroll
              for (int jn = 0; jn < STEPS * NW; ++jn) {
                const int j = jn / NW, n = jn % NW;
                auto ahead = wf;
                if (jn + 1 < STEPS * NW)
                  ahead = made(codes[d], h * STEPS + (jn + 1) / NW, (jn + 1) % NW);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                  if constexpr (F16)
                    acc[n][i] =
                        mfma_f16(wf, __builtin_bit_cast(f16x8, frags[set][j][i]), acc[n][i]);
                  else
                    acc[n][i] = mfma16x16x32(wf, frags[set][j][i], acc[n][i]);
                }
                wf = ahead;
              }
            }
            if constexpr (PIPE) __builtin_amdgcn_sched_barrier(0);
          }
      }
    }
  };
  // (every wave waits at the same barriers, whichever walk it takes)
  if (HALF && fits) walk(std::integral_constant<bool, HALF>{});
  else walk(std::integral_constant<bool, false>{});
  Residual<T> res[MT][NT];
  if (!GATED && a.r && a.N >= 4) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const Sums<NT> at(t * 64 + lane);
        res[i][t].load(a, m0 + i * 16 + at.row, (nt + at.tile) * 16 + at.quad * 4);
      }
  }
  // the ring is free once every wave's loads have landed and been read
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  static_assert(sizeof(ring) >= 4 * 2 * NW * 1024, "two row tiles' sums a wave");
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    f32x4* sums = (f32x4*)ring + (wave * 2 + i % 2) * NW * 64;
#pragma unroll
    for (int n = 0; n < NW; ++n)
      sums[n / NT * NT * 64 + Sums<NT>::slot(n % NT, fr, fq)] = acc[n][i];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const Sums<NT> at(t * 64 + lane);
      f32x4 s[W];
#pragma unroll
      for (int v = 0; v < W; ++v) s[v] = sums[v * NT * 64 + at.slot()];
      finish<T, GATED>(a, m0 + i * 16 + at.row, (nt + at.tile) * 16 + at.quad * 4, s, res[i][t]);
    }
  }
}

int64_t pad128(int64_t k) { return kad_cdiv(k, 128) * 128; }

template <typename T>
bool in_place(const void* x, int64_t ldx, int K) {
  return sizeof(T) == 2 && K % 8 == 0 && (uintptr_t)x % 16 == 0 && ldx % 8 == 0;
}

// Which kernel and tile.  n: rows of the weights in all (gated: the gate's and the up's).
// While there is a CU for each workgroup (256) a call takes what one workgroup's walk over K
// takes, so the smallest tile that needs no more wins; with many workgroups a CU, the
// largest.  The kernel of few rows has tiles of up to 32 x 64 (rows x rows of the weights),
// its largest up to 640 workgroups (32 x 30000 x 8192, 469 of them: bf16 39 us, the other
// kernel 42, fp16 38 and 45, fp32 72 and 68; 300 x 4096 x 2048, 640: 12.5 and 12.7, 12.4 and
// 13.3, 29 and 27; 32 x 50000 x 1024, 782: 12.8 and 11.1, 12.6 and 11.5, 24 and 18), and up
// to 16 rows its tile of 16 x 64 whatever the weight (16 x 248320 x 1024: 33.4 us, of the
// other kernel's 32.1 at best; fp16 33.6 and 36.4, fp32 46 and 54: one rule for all types).
// These figures and those beside the rules below are of calls behind one another in a graph,
// without a residual, weights from beyond the caches; bf16, us:
//   M x N x K            16x16  16x32  16x64  32x64 | 32x128 64x128 64x256 128x256
//   16 x 1024 x 3584       5.0    5.6    6.9    8.4 |  17     21     30      45
//   128 x 1024 x 3584      7.5    5.4    6.4    8.9 |  17     22     31      47
//   256 x 1024 x 3584     11.9    7.3    6.4    8.8 |  17     22     31      47
//   32 x 8192 x 8192      26     16     13.2   17.9 |  36     44     65     106
//   64 x 8192 x 8192      45     25     20.4   17.5 |  36     46     67     106
//   128 x 8192 x 8192     85     43     33     29   |  37     46     66     108
//   256 x 8192 x 8192    161     79     59     50   |  46     47     66     108
//   512 x 8192 x 8192    307    158    112     89   |  81     64     70     108
//   1024 x 8192 x 8192                        171   | 143    124    107     117
//   32 x 100000 x 1024    98     38     25     20.8 |  19.8   23.5   19.4    28.6
//   64 x 100000 x 1024   185     66     42     32   |  28.8   26.5   21.0    29.7
//   1024 x 32768 x 1024                       115   | 100     89     69      62
bool few(int64_t M, int64_t n) {
  return M <= 16 || kad_cdiv(M, 32) * kad_cdiv(n, 64) <= 640;
}

// bytes of the rows' pieces; 0 where the rows are read as they are
template <typename T>
int64_t piece_bytes(const void* x, int64_t ldx, int64_t M, int64_t n, int K) {
  return few(M, n) || in_place<T>(x, ldx, K) ? 0 : kPlanes<T> * M * pad128(K) * 2;
}

template <typename T, bool RAW, bool GATED, int MT, int NT, int KS, int D, int R = 16>
void launch_stream(Args a, hipStream_t s) {
  const dim3 grid((unsigned)kad_cdiv(a.cols, 16 * NT), (unsigned)kad_cdiv(a.M, 16 * MT));
  // In the grid's order an XCD has an eighth of the columns, or a few of them, and reads all
  // rows; where those pass its L2 (4 MB) and the codes in bytes, it has an eighth of the rows
  // and reads all codes: bf16 2048 x 512 x 4096 15.7 us, in the grid's order 23.6; 1951 x 368 x
  // 8912 26.9 and 38.1; fp32 300 x 1024 x 2048, 2.4 MB of rows: 12.4 and 11.4; bf16 32 x 8192 x
  // 8192, 36 MB of codes: 13.4 and 10.5.
  const int64_t rows = (int64_t)a.M * a.K * (RAW ? sizeof(T) : 2 * kPieces<T>);
  const bool by_rows = rows > (4 << 20) && rows > (int64_t)a.KB * 68 * a.cols * (GATED ? 2 : 1);
  // Else the row tiles of a column tile share an XCD by themselves where a row of the grid is
  // whole rounds of 8; elsewhere they are numbered so, for the widest tiles (fp16 37 x 5001 x
  // 2007, 79 column tiles: 6.0 us, in the grid's order 6.7; bf16 100 x 5000 x 2048 9.3 and 10.0;
  // narrower ones gain nothing: 64 x 1400 x 8192 7.6 and 7.6).
  const bool by_columns = NT * (GATED ? 2 : 1) == 4 && grid.y > 1 && grid.x % 8;
  a.order = by_rows ? 1 : by_columns ? 2 : 0;
  hipLaunchKernelGGL((q4_stream_kernel<T, RAW, GATED, MT, NT, KS, D, R>), grid, dim3(64 * KS), 0,
                     s, a);
}

template <typename T, bool HALF, bool RAGGED, bool GATED, int MT, int NW, int BK, int SLOTS, int D>
void launch_tile(const Args& a, hipStream_t s) {
  const int64_t mtiles = kad_cdiv(a.M, 16 * MT);
  const int64_t ntiles = kad_cdiv(a.cols, 64 * NW / (GATED ? 2 : 1));
  hipLaunchKernelGGL((q4_tile_kernel<T, HALF, RAGGED, GATED, MT, NW, BK, SLOTS, D>),
                     dim3((unsigned)(mtiles * ntiles)), dim3(256), 0, s, a, (int)mtiles,
                     (int)ntiles);
}

template <typename T, bool RAW, bool GATED>
void stream(const Args& a, hipStream_t s) {
  // (P: the products a row block and step take; rows of fp16 are pieces in the second half of
  // a feed-forward block alone)
  constexpr int W = GATED ? 2 : 1, P = RAW && sizeof(T) == 2 ? 1 : kPieces<T>;
  const int64_t tiles = kad_cdiv(a.M, 16), n = (int64_t)a.cols * W;
  // 8 waves share K from 12 blocks of it on (16 x 1024 x 1536 fp32: 4.9 us, 4 waves 5.5;
  // 16 x 2048 x 16384: 12.9 and 14.3; 1 x 1024 x 1024, 8 blocks: 2.9 and 2.2)
  const bool wide = a.KB >= 12;
  // 4 rows or fewer load no more (1 x 1024 x 3584: 3.5 us, all 16 of the tile 4.3)
  auto rows = [&](auto r) {
    constexpr int R = decltype(r)::value;
    if constexpr (!GATED)
      if (tiles * kad_cdiv(n, 16) <= 256) {
        // 4 blocks ahead where a wave has as many (1 x 2048 x 16384: 7.7 us, 2 ahead 9.4)
        if constexpr (P < 3)
          if (a.KB >= 24) return launch_stream<T, RAW, GATED, 1, 1, 8, 4, R>(a, s);
        if (wide) return launch_stream<T, RAW, GATED, 1, 1, 8, 2, R>(a, s);
        return launch_stream<T, RAW, GATED, 1, 1, 4, 2, R>(a, s);
      }
    if (tiles * kad_cdiv(n, 32) <= 256) {
      if (wide) return launch_stream<T, RAW, GATED, 1, 2 / W, 8, 2, R>(a, s);
      return launch_stream<T, RAW, GATED, 1, 2 / W, 4, 2, R>(a, s);
    }
    // (fp32 rows, one block ahead, have too few in flight: 128 x 2048 x 16384 45 us, two ahead
    // 39; and with two ahead no registers for a second workgroup: 300 x 1024 x 2048, 304 of
    // them, 12.9 us, of 4 waves 11.4)
    if (wide && (P < 3 || tiles * kad_cdiv(n, 64) <= 256))
      return launch_stream<T, RAW, GATED, 1, 4 / W, 8, P == 3 ? 2 : 1, R>(a, s);
    return launch_stream<T, RAW, GATED, 1, 4 / W, 4, 2, R>(a, s);
  };
  if (a.M <= 4) return rows(std::integral_constant<int, 4>{});
  // (128 x 4096 x 4096, 512 workgroups of 16 x 64: fp32 21.3 us, of 32 x 64 25; bf16 10.3 and
  // 9.7)
  if (a.M <= 16 || tiles * kad_cdiv(n, 64) <= (P > 1 ? 512 : 320))
    return rows(std::integral_constant<int, 16>{});
  // (pieces two blocks ahead leave registers for one workgroup a CU: fp16 block of 600 x 1024 x
  // 1024, one ahead 18.3 us, two 22.2)
  return launch_stream<T, RAW, GATED, 2, 4 / W, 4, P == 1 ? 2 : 1>(a, s);
}

template <typename T, bool HALF, bool RAGGED, bool GATED>
void tiles(const Args& a, hipStream_t s) {
  constexpr int P = HALF ? 1 : kPieces<T>;
  const int64_t n = (int64_t)a.cols * (GATED ? 2 : 1);
  auto count = [&](int rows, int cols) { return kad_cdiv(a.M, rows) * kad_cdiv(n, cols); };
  // up to two workgroups a CU, and up to 32 rows (32 x 248320 x 1024: bf16 35.3 us, 64 x 128
  // 45.9, 64 x 256 36.9; fp32 61, 83 and 72)
  if (count(32, 128) <= 512 || a.M <= 32)
    return launch_tile<T, HALF, RAGGED, GATED, 2, 2, 128, 4, 4>(a, s);
  // slices of 64 columns and fewer codes ahead where the pieces of fp16 rows leave no
  // registers for more
  if (count(64, 128) <= 512) {
    constexpr int BK = HALF ? 64 : 128, D = HALF || P == 2 ? 2 : 4;
    return launch_tile<T, HALF, RAGGED, GATED, 4, 2, BK, 4, D>(a, s);
  }
  // Two of the largest tiles run on a CU at a time, and take twice as long as four of half
  // the size, or somewhat less: the larger ones where that halves the rounds (69 x 100000 x
  // 1024, one round against two: 29.6 us, smaller 35.4; 130 rows, two and three: 57.4 and
  // 46.8; 1024 x 32768 x 1024, two and four: 62 and 69).  fp16 and fp32 rows have no registers
  // for them (fp16, spilled: 1024 x 32768 x 1024 121 us, smaller 75, which itself keeps 9 to 30
  // registers of its walk in pieces in scratch memory), nor have ragged ones (4000 x 2880 x
  // 2880: 150 us, smaller 72).
  if constexpr (kPieces<T> == 1 && !RAGGED)
    if (2 * kad_cdiv(count(128, 256), 512) <= kad_cdiv(count(64, 256), 512))
      return launch_tile<T, HALF, RAGGED, GATED, 8, 4, 64, 4, 2>(a, s);
  return launch_tile<T, HALF, RAGGED, GATED, 4, 4, 64, 4, 2>(a, s);
}

// a product of the rows x as they are, or of their pieces in `ws`
template <typename T, bool GATED>
void multiply(Args a, const void* x, int64_t ldx, void* ws, hipStream_t s) {
  a.x = x, a.ldx = ldx, a.xp = 0;
  if (few(a.M, (int64_t)a.cols * (GATED ? 2 : 1))) return stream<T, true, GATED>(a, s);
  if (!in_place<T>(x, ldx, a.K)) {
    const int KP = (int)pad128(a.K);
    a.x = ws, a.ldx = KP, a.xp = (int64_t)a.M * KP;
    hipLaunchKernelGGL((split_rows_kernel<T, kPlanes<T>>),
                       dim3((unsigned)kad_cdiv((int64_t)a.M * (KP / 8), 256)), dim3(256), 0, s,
                       (const T*)x, ldx, (uint16_t*)ws, a.M, a.K, KP);
  }
  constexpr bool HALF = std::is_same_v<T, _Float16>;
  if constexpr (sizeof(T) == 2)
    if (a.x == x && a.K % 128) return tiles<T, HALF, true, GATED>(a, s);
  tiles<T, HALF, false, GATED>(a, s);
}

// the same of rows that are pieces already, padded to whole blocks
template <typename T>
void multiply_pieces(Args a, const bf16_t* x, hipStream_t s) {
  a.x = x, a.ldx = pad128(a.K), a.xp = a.M * a.ldx, a.K = (int)a.ldx;
  if (few(a.M, a.cols)) return stream<T, kPieces<T> == 1, false>(a, s);
  tiles<T, false, false, false>(a, s);
}

struct Weight {
  const void *codes, *scales;
};

// everything of a product but its rows
template <typename T>
Args linear(Weight w, const void* r, int64_t ldr, void* y, int64_t ldy, int M, int N, int K) {
  Args a{};
  a.codes[0] = a.codes[1] = (const uint8_t*)w.codes;
  a.scales[0] = a.scales[1] = (const uint8_t*)w.scales;
  a.r = r, a.ldr = ldr, a.y = y, a.ldy = ldy, a.yp = 0;
  a.M = M, a.N = N, a.K = K, a.KB = (int)kad_cdiv(K, 128), a.cols = N;
  return a;
}

Args gated(Weight g, Weight u, bf16_t* h, int M, int F, int K) {
  Args a{};
  a.codes[0] = (const uint8_t*)g.codes, a.codes[1] = (const uint8_t*)u.codes;
  a.scales[0] = (const uint8_t*)g.scales, a.scales[1] = (const uint8_t*)u.scales;
  a.r = nullptr, a.ldr = 0, a.y = h, a.ldy = pad128(F), a.yp = M * pad128(F);
  a.M = M, a.N = F, a.K = K, a.KB = (int)kad_cdiv(K, 128), a.cols = (int)pad128(F);
  return a;
}

int check_sizes(int64_t M, int64_t N, int K) {
  KAD_REQUIRE(M > 0 && N > 0 && K > 0, "empty dimensions");
  KAD_REQUIRE(K <= kMaxK && N <= kMaxN, "a weight of %lld rows of %d columns", (long long)N, K);
  // (a grid holds fewer than 2^32 work-items a dimension, and 65535 rows of tiles)
  KAD_REQUIRE(M <= 16 * 65535 && kad_cdiv(M, 32) * kad_cdiv(2 * N, 128) < (1ll << 32) / 256,
              "a product of %lld x %lld outputs", (long long)M, (long long)N);
  // (a thread of the pieces' kernel takes 8 elements; workgroups of 256)
  KAD_REQUIRE(M * pad128(K) <= (1ll << 35) - 2048, "%lld rows of %d columns", (long long)M, K);
  return KAD_OK;
}

int check_weight(Weight w) {
  KAD_REQUIRE(w.codes && w.scales, "null pointer argument");
  KAD_REQUIRE((uintptr_t)w.codes % 16 == 0 && (uintptr_t)w.scales % 16 == 0,
              "codes and scales must be 16-byte aligned");
  return KAD_OK;
}

// f.template operator()<T>() for the type of a dtype code
template <typename F>
int for_dtype(int dtype, F f) {
  if (dtype == KAD_DTYPE_BF16) return f(bf16_t{});
  if (dtype == KAD_DTYPE_F16) return f(_Float16{});
  if (dtype == KAD_DTYPE_F32) return f(float{});
  KAD_UNSUPPORTED("dtype code %d", dtype);
}

}  // namespace

extern "C" int kad_quantized_linear_workspace_bytes(const void* x, int64_t ldx, int dtype, int M,
                                                    int N, int K, int64_t* bytes) {
  KAD_REQUIRE(bytes, "null pointer argument");
  KAD_TRY(check_sizes(M, N, K));
  return for_dtype(dtype, [&](auto t) {
    *bytes = piece_bytes<decltype(t)>(x, ldx, M, N, K);
    return KAD_OK;
  });
}

extern "C" int kad_quantized_linear(const void* x, int64_t ldx, int dtype, const void* codes,
                                    const void* scales, const void* residual, int64_t ldr, void* y,
                                    int64_t ldy, void* workspace, int64_t workspace_bytes, int M,
                                    int N, int K, kad_stream_t stream) {
  int64_t need = 0;
  KAD_TRY(kad_quantized_linear_workspace_bytes(x, ldx, dtype, M, N, K, &need));
  KAD_REQUIRE(x && y, "null pointer argument");
  KAD_TRY(check_weight({codes, scales}));
  KAD_REQUIRE(ldx >= K && ldy >= N && (!residual || ldr >= N), "rows longer than their stride");
  KAD_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0), "workspace");
  KAD_REQUIRE(workspace_bytes >= need, "workspace of %lld bytes, %lld needed",
              (long long)workspace_bytes, (long long)need);
  return for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    multiply<T, false>(linear<T>({codes, scales}, residual, ldr, y, ldy, M, N, K), x, ldx,
                       workspace, (hipStream_t)stream);
    return kad_launch_status("quantized product");
  });
}

extern "C" int kad_quantized_gated_ffn_workspace_bytes(const void* x, int64_t ldx, int dtype,
                                                       int M, int H, int F, int64_t* bytes) {
  KAD_REQUIRE(bytes, "null pointer argument");
  KAD_TRY(check_sizes(M, F, H));
  KAD_TRY(check_sizes(M, H, F));
  return for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    *bytes = piece_bytes<T>(x, ldx, M, 2 * pad128(F), H) + kPieces<T> * (int64_t)M * pad128(F) * 2;
    return KAD_OK;
  });
}

extern "C" int kad_quantized_gated_ffn(const void* x, int64_t ldx, int dtype,
                                       const void* gate_codes, const void* gate_scales,
                                       const void* up_codes, const void* up_scales,
                                       const void* down_codes, const void* down_scales,
                                       const void* residual, int64_t ldr, void* y, int64_t ldy,
                                       void* workspace, int64_t workspace_bytes, int M, int H,
                                       int F, kad_stream_t stream) {
  int64_t need = 0;
  KAD_TRY(kad_quantized_gated_ffn_workspace_bytes(x, ldx, dtype, M, H, F, &need));
  KAD_REQUIRE(x && y, "null pointer argument");
  const Weight g{gate_codes, gate_scales}, u{up_codes, up_scales}, d{down_codes, down_scales};
  KAD_TRY(check_weight(g));
  KAD_TRY(check_weight(u));
  KAD_TRY(check_weight(d));
  KAD_REQUIRE(ldx >= H && ldy >= H && (!residual || ldr >= H), "rows longer than their stride");
  KAD_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0, "workspace");
  KAD_REQUIRE(workspace_bytes >= need, "workspace of %lld bytes, %lld needed",
              (long long)workspace_bytes, (long long)need);
  return for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const hipStream_t s = (hipStream_t)stream;
    bf16_t* h = (bf16_t*)((char*)workspace + piece_bytes<T>(x, ldx, M, 2 * pad128(F), H));
    multiply<T, true>(gated(g, u, h, M, F, H), x, ldx, workspace, s);
    multiply_pieces<T>(linear<T>(d, residual, ldr, y, ldy, M, H, F), h, s);
    return kad_launch_status("quantized product");
  });
}
