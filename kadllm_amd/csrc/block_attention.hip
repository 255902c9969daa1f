// Attention of beams over a request's prefix in the 8-bit cache, then over
// their own causal suffix: for a query row (beam n of request b, token t,
// head h, KV head kh = h / (H / HK))
//   s_j = scale * q . k_j   over the request's cached keys, j < lengths[b],
//                           and the beam's suffix keys j <= Tk - T + t
//   out = sum_j softmax(s)_j v_j, times sigmoid(gate) where one is given
// with k_j, v_j = code * scale of the page and KV head that holds token j.  A
// row that sees no key gives zeros.
//
// Both products over the cache run on v_mfma_scale_f32_32x32x64_f8f6f4, which
// reads the cache's e4m3 codes as they are and applies the page's power of two
// itself.  The other operand is split into e4m3 pieces: x = 2^E (y0 + y1 / 16
// + y2 / 256), each y the e4m3 rounding of 16 times what the pieces before it
// left.  A piece keeps 4 significant bits, so two hold a bf16 value exactly
// (8 bits) and three an fp16 one (11 bits), as far down as 2^-10 of the row's
// largest element; below that the error is at most 2^-21 of the largest (the last
// piece of two is off by up to 2^-10 / 16 where the largest is 2^7 or more).  Two
// pieces cost what one bf16 product would (e4m3 runs at twice the rate), and
// the cache is neither widened in registers nor stored wide in LDS.
//
// The softmax weights of 32 keys are split the same way against the block's own
// power of two, which the second product's scale operand restores: 2^-8
// relative per weight with two pieces (bf16), 2^-12 with three (fp16).

#include <cmath>
#include <type_traits>

#include "kad_common.h"

namespace {

// n / d for 0 <= n < 2^31 as n m / 2^(31 + s), m = floor(2^(31 + s) / d) + 1 and s =
// ceil(log2 d): 0 < m d - 2^(31 + s) <= d <= 2^s, so the quotient is over n / d by
// less than 1 / d
struct Divide {
  uint32_t m;
  int s, d;
};
inline Divide divide_by(int d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return Divide{(uint32_t)((1ull << (31 + s)) / (uint32_t)d + 1), 31 + s, d};
}
__device__ __forceinline__ int operator/(int n, Divide by) {
  return (int)((uint64_t)(uint32_t)n * by.m >> by.s);
}

struct BlockAttnArgs {
  const void* q;
  int64_t sq_n, sq_t, sq_h;
  const uint8_t *kc, *vc, *ksc, *vsc;
  const int* tables;
  const int* lengths;
  const void* sk;
  int64_t ssk_n, ssk_t, ssk_h;
  const void* sv;
  int64_t ssv_n, ssv_t, ssv_h;
  const void* gate;
  int64_t sg_n, sg_t, sg_h;
  void* out;
  int64_t so_n, so_t, so_h;
  float* part_o;    // splits > 1: [split][B*HK][R][D] unnormalised outputs
  float* part_ml;   // and [split][B*HK][R][2]: the exponent they are relative to, the sum
  int pages, width, B, W, T, Tk, H, HK, G, lblock;
  int splits, nqblk;
  Divide by_splits, by_nqblk, by_HK, by_G, by_T, by_Tk;
  int R;            // query rows of a request and KV head, W * T * (H / HK)
  float qmul, sl2;  // sign of the scale (0 for none), |scale| in log2 units
};

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_t;

// f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>)
template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

// A wave's fragment layout of v_mfma_scale_f32_32x32x64 for 8-bit operands:
// lane l holds row (column for B) l % 32; its bytes 0-15 are k = 16 (l / 32) +
// 0..15 and its bytes 16-31 k = 32 + 16 (l / 32) + 0..15; the scale byte of
// lanes 0-31 serves k < 32 and that of lanes 32-63 k >= 32.
__device__ __forceinline__ f32x16 mfma_scaled(i32x8 a, i32x8 b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// 4 floats to a dword of e4m3 codes, and what they leave
__device__ __forceinline__ int piece4(const float* y, float* rest) {
  int c;
  asm("" : "=v"(c));              // (both halves are written below)
  c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], c, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  rest[0] = y[0] - lo[0];
  rest[1] = y[1] - lo[1];
  rest[2] = y[2] - hi[0];
  rest[3] = y[3] - hi[1];
  return c;
}
__device__ __forceinline__ float pow2i(int e) {  // 2^e, -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// the largest of three, NaN where one is (fmaxf would first quiet each operand)
__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

template <typename T> struct Pieces;
template <> struct Pieces<bf16_t> { static constexpr int n = 2; };
template <> struct Pieces<_Float16> { static constexpr int n = 3; };

// 8 elements as floats
__device__ __forceinline__ void widen8(const bf16_t*, u32x4 v, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(v[i] << 16);
    f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void widen8(const _Float16*, u32x4 x, float* f) {
  const f16x8 v = __builtin_bit_cast(f16x8, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)v[i];
}
// the products of the suffix, in the queries' type
__device__ __forceinline__ f32x16 mfma_wide(const bf16_t*, u32x4 a, u32x4 b, f32x16 c) {
  return mfma32x32x16(as_bf16x8(a), as_bf16x8(b), c);
}
__device__ __forceinline__ f32x16 mfma_wide(const _Float16*, u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack2(const bf16_t*, float a, float b) {
  return pack_bf16x2(a, b);
}
__device__ __forceinline__ uint32_t pack2(const _Float16*, float a, float b) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}
// the exponent bits of a pair of elements: all set in an infinity or NaN
template <typename T>
constexpr uint32_t kExponents = std::is_same<T, bf16_t>::value ? 0x7f807f80u : 0x7c007c00u;
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

constexpr int kKeys = 64;       // keys per tile: two halves of 32, each within a page
// A row's scores may lie this far above its reference, in powers of two, before the
// reference moves: by 60, or less where the values are so large that weights of
// that size times them could pass 2^120.  Of up to 2^30 cached keys of V scale byte
// sv the values are below 2^(sv - 118); a suffix has up to 2^22 keys, whose values may
// reach 2^38 (kBigValue) under weights of up to 2^60.
constexpr int kMaxUp = 60;
constexpr uint32_t kBigValue = (127 + 38) << 7;   // as a bf16 (fp16 values end before it)
__device__ __forceinline__ float climb_of(int sv) { return (float)min(kMaxUp, 208 - sv); }
// A reference that has moved lies this far above the row's true maximum, so that
// outputs stay below the largest value while they are summed (2^30 keys of weight
// 2^-30).  Not in fp16, where suffix weights are fp16 and an output that passes fp32
// on the way does not fit its type.
template <typename T>
constexpr float kRoom = std::is_same<T, bf16_t>::value ? 30.f : 0.f;

template <int D>
struct Shape {
  static constexpr int KS = D / 64, DT = D / 32;   // k-steps of q . k, 32-wide tiles of the output
  static constexpr int CPR = D / 16;               // 16-byte chunks per key
  static constexpr int RPI = 64 / CPR;             // keys per 1 KB load instruction
  static constexpr int tile = kKeys * D;           // bytes of a K (or V) tile
  static constexpr int slot = 2 * tile;
  static constexpr int LT = tile / 1024;           // load instructions per K (or V) tile
  static constexpr int stages = 4;
  static constexpr int EpiLd = D + 4;              // fp32 row stride of the output transpose
  static constexpr int epi = 4 * 32 * EpiLd * 4;
  static constexpr int lds = stages * slot > epi ? stages * slot : epi;
  // physical 16-byte chunk of logical chunk c in key row r is c ^ sw(r): the 8
  // rows that one fragment read serves together then lie in 8 different bank
  // groups.  K fragments take rows 0-7 of 8; V's transpose reads rows {0-3,
  // 8-11} + 4 (l / 32).
  __device__ static __forceinline__ int swk(int r) {
    return D == 256 ? r & 15 : D == 128 ? r & 7 : (r >> 1) & 3;
  }
  __device__ static __forceinline__ int swv(int r) {
    const int b0 = r & 1, b1 = r >> 1 & 1, b2 = r >> 2 & 1, b3 = r >> 3 & 1;
    return D == 256 ? b0 | b1 << 1 | b3 << 2 | b2 << 3 : D == 128 ? b0 | b1 << 1 | b3 << 2
                                                                  : b1 | b3 << 1;
  }
};

// V^T fragments of two 32-wide output tiles of 16-bit rows (the suffix): for each,
// 16 keys, 2 transpose reads of 4 keys (lane i of 16 receives element i % 4 of
// the 8-byte pieces that lanes 4e + i / 4 address, e < 4), waited for inside
template <int D>
__device__ __forceinline__ void read_wide2(uint32_t p0, uint32_t p1, u32x4& f0, u32x4& f1) {
  u32x2 a0, a1, b0, b1;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %2, %5\n\t"
      "ds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a0), "=&v"(a1), "=&v"(b0), "=&v"(b1)
      : "v"(p0), "v"(p1), "i"(16 * D)
      : "memory");
  f0 = u32x4{a0[0], a0[1], a1[0], a1[1]};
  f1 = u32x4{b0[0], b0[1], b1[0], b1[1]};
}

__device__ __forceinline__ void wait_vm(int n) {
  // vmcnt(n), lgkmcnt and expcnt left alone; n a constant after inlining
  switch (n) {
#define KAD_W(N) case N: __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14)); break;
    KAD_W(0) KAD_W(1) KAD_W(2) KAD_W(3) KAD_W(4) KAD_W(6) KAD_W(8) KAD_W(12) KAD_W(16)
    KAD_W(24) KAD_W(32)
#undef KAD_W
    default: __builtin_amdgcn_s_waitcnt(0x0f70);
  }
  asm volatile("" ::: "memory");   // (reads of what has landed stay behind the wait)
}
__device__ __forceinline__ void tile_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 16 bytes a lane from base + off (zeros from nbytes on) into LDS at lds + 16 *
// lane; base, nbytes and lds wave-uniform.  In assembly so that the compiler does
// not make the next transpose read wait for every such load in flight: waits are
// the callers' (wait_vm).  (No register is written; the nops cover scalar
// operands that a vector instruction has just written, and m0.)
// AT goes to both addresses (as the instruction's offset field does).
template <int AT>
__device__ __forceinline__ void load_lds16(u32x4 rsrc, uint32_t off, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %2\n\t"
      "s_nop 4\n\t"
      "buffer_load_dwordx4 %0, %1, 0 offen offset:%3 lds"
      :
      : "v"(off), "s"(rsrc), "s"(lds), "n"(AT)
      : "memory");
}

// the same from an address of each lane's own
__device__ __forceinline__ void load_lds16(const void* src, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %1\n\t"
      "s_nop 4\n\t"
      "global_load_lds_dwordx4 %0, off"
      :
      : "v"(src), "s"(lds)
      : "memory");
}

// y times the sigmoid of a gate element (by the hardware's reciprocal, 1 ulp)
__device__ __forceinline__ float gate1(float g, float y) {
  return y * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
}
template <typename T>
__device__ __forceinline__ void gate8(const T* kind, u32x4 gate, float* y) {
  float g[8];
  widen8(kind, gate, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = gate1(g[i], y[i]);
}
// 4 elements of an output row: times inv, gated, rounded once
template <typename T>
__device__ __forceinline__ void store_row4(T* out, const float* o, float inv, bool gated,
                                           u32x2 gate) {
  const T* const kind = nullptr;
  float y[4], g[8];
  widen8(kind, u32x4{gate[0], gate[1], 0u, 0u}, g);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = o[e] * inv;
    if (gated) y[e] = gate1(g[e], y[e]);
  }
  *(u32x2*)out = u32x2{pack2(kind, y[0], y[1]), pack2(kind, y[2], y[3])};
}

// 4 accumulation registers cut to at most a bound each, which stays a rare branch
// between products only if it leaves them where they are.  (The first nops cover
// a product still writing them, the last one the next reader.)
__device__ __forceinline__ void min_acc(float& x0, float& x1, float& x2, float& x3, f32x4 bound) {
  float t0, t1, t2, t3;
  asm volatile(
      "s_nop 15\n\ts_nop 15\n\t"
      "v_accvgpr_read_b32 %4, %0\n\tv_accvgpr_read_b32 %5, %1\n\t"
      "v_accvgpr_read_b32 %6, %2\n\tv_accvgpr_read_b32 %7, %3\n\ts_nop 1\n\t"
      "v_min_f32 %4, %4, %8\n\tv_min_f32 %5, %5, %9\n\t"
      "v_min_f32 %6, %6, %10\n\tv_min_f32 %7, %7, %11\n\ts_nop 1\n\t"
      "v_accvgpr_write_b32 %0, %4\n\tv_accvgpr_write_b32 %1, %5\n\t"
      "v_accvgpr_write_b32 %2, %6\n\tv_accvgpr_write_b32 %3, %7\n\ts_nop 4"
      : "+a"(x0), "+a"(x1), "+a"(x2), "+a"(x3), "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
      : "v"(bound[0]), "v"(bound[1]), "v"(bound[2]), "v"(bound[3]));
}

// A workgroup of 4 waves takes a request, a KV head, a range of the prefix
// (one of `splits`) and query rows, ordered (beam, head in the group, token).
// A wave holds 32 rows: Q's pieces, the output O^T and the softmax state stay
// in its registers.  S^T = K Q^T gives a lane the scores of one row (16 of a
// half tile's 32 keys, the other 16 in lane l ^ 32), and the bytes of its
// weights are the second product's operand O^T += V^T P^T as they stand.
//   SHARED: the waves hold 128 rows and walk the same tiles, which arrive in
//     rings of 4 K and 4 V tiles in LDS, three steps ahead of their use.
//   otherwise: the waves hold the same 32 rows and take every fourth tile, each
//     through an LDS slot of its own, K refilled while V is used and V refilled
//     while the next K is, so no wave waits for another; their states are
//     joined at the end.
// Weights are 2^(s - m) for a reference m, the maximum of the first keys that the
// row sees.  Scores above it need no rescaling, because the weights of 32 keys
// carry an exponent of their own; only when one lies more than 2^60 above (2^14
// among fp16 suffix keys, less among values past 2^30: climb_of) is the walk done
// again, with the row's true maximum.
// What bounds it, bf16, D 256, 2 KV heads for 8 heads (traced kernel times, which are
// some us longer than those of calls that follow each other):
//   16 requests of 1 beam over 32768 keys: HBM, 95 to 100 us for 537 MB (private, 8
//     ranges each), and 5 us of join.
//   32 requests of 256 beams over 1024 keys, gated: 106 to 112 us (102 in a row of
//     calls) for 69 GFLOP and 168 MB, two rounds of workgroups that load q, walk and
//     store together.  Fitted over calls without a gate, a step of the walk takes 1.8 us
//     (its 32 MFMAs 2048 cycles, about half of that; the softmax and the pieces of the
//     weights are the rest) and a round 19 us besides: q and its pieces, the first
//     tiles, the results through LDS and out, with no other workgroup on the CU (512
//     registers and 133 KB of LDS).  Half the first round started late, to set the
//     phases apart, measured the same.  fp16, with three pieces: 145 to 150 us; 2.6 us a
//     step and 24 us a round.
//   1 request of 256 beams over 8192 keys: 35 to 37 us (private, 4 ranges; 2.5 us a step
//     of four tiles, 13 us besides), and 4 us of join.
//   1 request of 1 beam over 100 keys: 10.5 us, most of it that fixed part.
// Vector registers that do not fit and go to scratch: 6 in the shared form of bf16 at
// D 256, 54 in that of fp16, 12 in the private form of fp16 at D 128.
template <typename T, int D, bool SHARED>
__global__ __launch_bounds__(256, D == 256 || SHARED ? 1 : 2) void
block_attn_kernel(BlockAttnArgs a) {
  using S = Shape<D>;
  constexpr int NP = Pieces<T>::n, KS = S::KS, DT = S::DT;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  __shared__ float sm_m[4][32], sm_l[4][32];
  __shared__ int sm_over[4];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hi = lane >> 5, col = lane & 31;
  const int lid = xcd_logical_id(blockIdx.x, gridDim.x);
  const int bks = lid / a.by_nqblk, bk = bks / a.by_splits, b = bk / a.by_HK;
  const int qb = lid - bks * a.nqblk, split = bks - bk * a.splits, kh = bk - b * a.HK;
  const int G = a.G;

  // ---- this lane's row (rows past the end repeat the last one and are not stored)
  const int row0 = qb * (SHARED ? 128 : 32) + (SHARED ? wave * 32 : 0);
  const int r = min(row0 + col, a.R - 1);
  const int rt = r / a.by_T, t = r - rt * a.T, w = rt / a.by_G, g = rt - w * G;
  const int64_t n = (int64_t)b * a.W + w;
  const int h = kh * G + g;
  const T* const kind = nullptr;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_t*)smem;
  u32x4 qr[4 * KS];        // q: elements 64 s + 32 (c / 2) + 16 hi + 8 (c % 2) + 0..7
  // 16-bit rows (of q, of the suffix) into LDS, `count` of them (16 or 32), lane i's
  // `at` the offset of row i: whole rows at a time, chunk c of row r at place c ^
  // sw(r)
  constexpr int CPV = D / 8, RPV = 512 / D;          // 16-byte chunks per row, rows per load
  auto of_lane = [](int64_t v, int from) {
    return (int64_t)((uint64_t)(uint32_t)__shfl((int)v, from, 64) |
                     (uint64_t)(uint32_t)__shfl((int)(v >> 32), from, 64) << 32);
  };
  auto load_rows = [&](auto count_c, auto values_c, const T* base, int64_t at, uint32_t dst) {
    constexpr bool kValues = decltype(values_c)::value;   // (read by transposes)
    constexpr int LOADS = decltype(count_c)::value / RPV;
    const T* src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = i * RPV + lane / CPV;
      const int sw = !kValues ? row & 7 : D == 64 ? (row >> 1 & 1) * 4 : (row & 3) * 4;
      src[i] = base + of_lane(at, row) + ((lane % CPV) ^ sw) * 8;
    }
    __builtin_amdgcn_sched_barrier(0);   // (the exchanges first, all at once)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_lds16(src[i], dst + i * 1024);
  };
  auto row_chunk = [&](const uint8_t* area, int row, int c) {
    const int chunk = 8 * (c >> 2) + 4 * (c >> 1 & 1) + 2 * hi + (c & 1);
    return *(const u32x4*)(area + row * 2 * D + (chunk ^ (row & 7)) * 16);
  };
  using n16 = std::integral_constant<int, 16>;
  using n32 = std::integral_constant<int, 32>;
  using yes = std::integral_constant<bool, true>;
  using no = std::integral_constant<bool, false>;
  auto load_q = [&](uint32_t dst) {
    load_rows(n32{}, no{}, (const T*)a.q, n * a.sq_n + t * a.sq_t + h * a.sq_h, dst);
  };
  auto take_q = [&](const uint8_t* area) {
#pragma unroll
    for (int c = 0; c < 4 * KS; ++c) qr[c] = row_chunk(area, col, c);
  };
  const bool has_suffix = a.Tk > 0 && split == 0 && (SHARED || wave == 3);
  int vlo = 0, vhi = -1, keys = 0;                   // keys the row sees, keys of the wave
  const int w0 = min(row0, a.R - 1) / a.by_T / a.by_G;
  const int64_t n0 = (int64_t)b * a.W + w0;
  if (has_suffix) {
    vlo = (w - w0) * a.Tk;
    vhi = vlo + a.Tk - a.T + t;
    keys = vhi + 1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) keys = max(keys, __shfl_xor(keys, o, 64));
    keys = __builtin_amdgcn_readfirstlane(keys);
  }
  auto suffix_load = [&](uint32_t dst, int f0) {
    const int f = min(f0 + (lane & 15), keys - 1), beam = f / a.by_Tk, token = f - beam * a.Tk;
    load_rows(n16{}, no{}, (const T*)a.sk,
              (n0 + beam) * a.ssk_n + (int64_t)token * a.ssk_t + kh * a.ssk_h, dst);
    load_rows(n16{}, yes{}, (const T*)a.sv,
              (n0 + beam) * a.ssv_n + (int64_t)token * a.ssv_t + kh * a.ssv_h, dst + 32 * D);
  };
  // q and the suffix, where a V tile and a K tile will go
  auto load_first = [&]() {
    load_q(lds0 + (SHARED ? 4 + wave : 2 * wave + 1) * S::tile);
    if (has_suffix) suffix_load(lds0 + (SHARED ? wave : 2 * wave) * S::tile, 0);
  };
  load_first();

  // ---- this wave's tiles of the prefix: first + stride * k, k < count.  (With one
  // range the first pages do not wait for the length.)
  int first_page = 0;
  const int* table = a.tables + (int64_t)b * a.width;
  if (a.splits == 1)
    first_page = table[min((((SHARED ? 0 : wave) + (SHARED ? 1 : 4) * (lane >> 1)) * 2 + (lane & 1))
                               >> (a.lblock - 5), a.width - 1)];
  const int len = max(min(a.lengths[b], a.width << a.lblock), 0);
  const int tiles = (len + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.by_splits;
  const int begin = min(split * per, tiles), end = min(begin + per, tiles);
  const int first = begin + (SHARED ? 0 : wave), stride = SHARED ? 1 : 4;
  const int count = __builtin_amdgcn_readfirstlane(
      SHARED ? end - begin : max((end - first + stride - 1) / stride, 0));

  // Pages: lane i of a chunk of 32 tiles describes half tile i: the offset of its
  // codes, and keys held (0: no page) | K's scale byte << 8 | V's << 16
  uint32_t code_lo = 0, code_hi = 0;
  int meta = 0;
  auto half_at = [&](int chunk) {
    return (first + stride * (32 * chunk + (lane >> 1))) * kKeys + (lane & 1) * 32;
  };
  auto page_at = [&](int chunk) {
    return table[min(half_at(chunk) >> a.lblock, a.width - 1)];
  };
  auto describe = [&](int chunk, int id) {
    const int pos = half_at(chunk);
    meta = 127 << 8 | 127 << 16;
    if (32 * chunk + (lane >> 1) < count && pos < len && id >= 0 && id < a.pages) {
      const int64_t ph = (int64_t)id * a.HK + kh;
      const int64_t code = ((ph << a.lblock) + (pos & ((1 << a.lblock) - 1))) * D;
      code_lo = (uint32_t)code;
      code_hi = (uint32_t)(code >> 32);
      meta = min(len - pos, 32) | (int)a.ksc[ph] << 8 | (int)a.vsc[ph] << 16;
    }
  };
  if (a.splits > 1) first_page = page_at(0);

  // ---- loads of a tile.  Instruction i of a K or V tile brings keys i * RPI +
  // lane / CPR; at place lane % CPR of a key goes the chunk that the swizzle puts
  // there.  Keys past those held arrive as zeros.
  constexpr int IPH = S::LT / 2;                 // instructions per half tile
  const int d_row = lane / S::CPR, d_pc = lane % S::CPR;
  auto source = [&](const uint8_t* codes, uint32_t lo, uint32_t hi32, int held) {
    const uint64_t p = (uint64_t)(uintptr_t)codes + ((uint64_t)hi32 << 32 | lo);
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)p),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) & 0xffffu,
                 (uint32_t)__builtin_amdgcn_readfirstlane(held * D), 0x00020000u};
  };
  // (the offset field adds (i % 4) KB to the source and the destination)
  auto off_of = [&](int kv, int i) {
    const int row = i * S::RPI + d_row;
    return (uint32_t)((row & 31) * D - i % 4 * 1024 +
                      (d_pc ^ (kv ? S::swv(row) : S::swk(row))) * 16);
  };

  // LDS offsets of the fragments
  uint32_t k_off[KS][2];   // K: key col of a half, chunks 4 s + hi and 4 s + 2 + hi
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      k_off[s][c] = col * D + ((4 * s + 2 * c + hi) ^ S::swk(col)) * 16;
  // V: key 8 (e / 4) + 4 hi + e % 4, e = (lane % 16) / 2; d = 32 dt + 16 (lane / 16 % 2) +
  // 8 (lane % 2)
  const int v_e = (lane & 15) >> 1;
  const int v_row = 8 * (v_e >> 2) + 4 * hi + (v_e & 3);
  uint32_t v_off[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    v_off[dt] = v_row * D + (lane & 1) * 8 + (((2 * dt + (lane >> 4 & 1)) ^ S::swv(v_row)) * 16);
  auto read_k = [&](const uint8_t* ks, int hf, int s) {
    const i32x4 x = *(const i32x4*)(ks + k_off[s][0] + hf * 32 * D);
    const i32x4 y = *(const i32x4*)(ks + k_off[s][1] + hf * 32 * D);
    return i32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };
  // 4 transpose reads of 8 keys (within 16 lanes, lane i receives byte i % 8 of
  // the 8-byte pieces that lanes 2e + i / 8 address, e < 8)
  auto read_v = [&](const uint8_t* vs, int dt) {
    typedef __attribute__((address_space(3))) i32x2* piece_t;
    const uint32_t at = (uint32_t)(uintptr_t)(lds_t*)vs + v_off[dt];
    i32x8 f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((piece_t)(at + 16 * c * D));
      f[2 * c] = x[0];
      f[2 * c + 1] = x[1];
    }
    return f;
  };

  // ---- the row's state, over the walk
  float m = -INFINITY, m_true, l;
  bool over, spoilt = false;
  f32x16 O[DT];
  i32x8 qf[NP][KS];        // q in e4m3 pieces against the row's power of two
  int qs[NP];
  auto split_q = [&]() {
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < 4 * KS; ++c) {
      float x[8];
      widen8(kind, qr[c], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
    }
    amax = max_xor32(amax);
    // (held where the last piece's scale is the smallest e8m0; what a piece cannot
    // hold there, 2^-137, is below every bf16 and fp16 number)
    const int E = max((int)(__float_as_uint(amax) >> 23) - 127 - 7, 4 * (NP - 1) - 127);
    const float inv = pow2i(-E) * a.qmul;
#pragma unroll
    for (int c = 0; c < 4 * KS; ++c) {
      float x[8];
      widen8(kind, qr[c], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= inv;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        qf[p][c >> 2][2 * (c & 3)] = piece4(x, x);
        qf[p][c >> 2][2 * (c & 3) + 1] = piece4(x + 4, x + 4);
        if (p + 1 < NP)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= 16.f;
      }
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) qs[p] = E - 4 * p + 127;
  };

  // ---- the beams' own suffixes.  The suffix keys of the wave's beams, in order,
  // are its key rows: of group after group of 16, S^T = K Q^T over all of them,
  // masked to each row's beam and to the tokens before its own, then O^T += V^T
  // P^T, both from LDS (area: 64 * D bytes of the wave's own).  A value that is not
  // finite would reach the rows that do not see it as 0 * inf, so a group that
  // holds one is multiplied without it, and the rows that do see it add it at the
  // end.  (In the private form the last wave does it, which has the fewest tiles.)
  // (the first group is there)
  auto suffix = [&](uint8_t* area, uint32_t area_at) {
    const float mul = a.qmul * a.sl2;
    constexpr float kUp = std::is_same<T, bf16_t>::value ? kMaxUp : 14.f;
    const uint8_t* values = area + 32 * D;
    const int gi = lane & 15, s_row = 4 * hi + (gi >> 2);
    const int s_d = (lane >> 4 & 1) * 16 + (gi & 3) * 4;
    const int s_sw = D == 64 ? (s_row >> 1 & 1) * 4 : (s_row & 3) * 4;
    const uint32_t base = area_at + 32 * D + s_row * D * 2 + (s_d & 7) * 2;
#pragma unroll 1
    for (int f0 = 0; f0 < keys; f0 += 16) {
      if (f0 > 0) {
        suffix_load(area_at, f0);
        wait_vm(0);
      }
      f32x16 st = f32x16{};
#pragma unroll
      for (int c = 0; c < 4 * KS; ++c)
        st = mfma_wide(kind, row_chunk(area, col & 15, c), qr[c], st);
      // (key rows 16 to 31 repeat the first ones)
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int f = f0 + 8 * (j >> 2) + 4 * hi + (j & 3);
        st[j] = f >= vlo && f <= vhi ? st[j] * mul : -INFINITY;
        top = fmaxf(top, st[j]);
      }
      top = max_xor32(top);
      m_true = fmaxf(m_true, top);
      if (m == -INFINITY) m = top;
      over |= top > m + kUp;
      const float ref = m == -INFINITY ? 0.f : m;
      u32x4 p;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float x = __builtin_amdgcn_exp2f(st[j] - ref);
        const float y = __builtin_amdgcn_exp2f(st[j + 1] - ref);
        sum += x + y;
        p[j >> 1] = pack2(kind, x, y);
      }
      l += add_xor32(sum);
      // (each lane looks at what its own loads brought)
      uint32_t top_exp = 0;
#pragma unroll
      for (int i = 0; i < 16 / RPV; ++i) {
        const u32x4 x = *(const u32x4*)(values + i * 1024 + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) top_exp = max_u16x2(top_exp, x[e] & kExponents<T>);
      }
      const uint32_t full = kExponents<T> & 0xffffu;
      const bool bad = __ballot((top_exp & 0xffffu) == full || top_exp >> 16 == full) != 0;
      if (bad) {
#pragma unroll 1
        for (int i = 0; i < 16 / RPV; ++i) {
          uint16_t* x = (uint16_t*)(values + i * 1024 + lane * 16);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((x[e] & full) == full) x[e] = 0;
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);
      }
      spoilt |= bad;
      if constexpr (std::is_same<T, bf16_t>::value) {   // a row that sees a big value
        if (__ballot((top_exp & 0xffffu) >= kBigValue || top_exp >> 16 >= kBigValue) != 0) {
          const int last = min(vhi - f0, 15);
          uint32_t seen = 0;
#pragma unroll 1
          for (int i = max(vlo - f0, 0); i <= last; ++i)
#pragma unroll 1
            for (int e = 0; e < D / 2; ++e)
              seen = max_u16x2(seen, ((const uint32_t*)(values + i * 2 * D))[e] & kExponents<T>);
          over |= (seen & 0xffffu) >= kBigValue || seen >> 16 >= kBigValue;
        }
      }
#pragma unroll
      for (int d2 = 0; d2 < DT / 2; ++d2) {
        u32x4 x, y;
        read_wide2<D>(base + ((((64 * d2 + s_d) >> 3) ^ s_sw) * 16),
                      base + ((((64 * d2 + 32 + s_d) >> 3) ^ s_sw) * 16), x, y);
        O[2 * d2] = mfma_wide(kind, x, p, O[2 * d2]);
        O[2 * d2 + 1] = mfma_wide(kind, y, p, O[2 * d2 + 1]);
      }
    }
  };

  // ---- the scores st of a tile (of halves holding held[] keys) to weights
  auto scores = [&](const uint8_t* ks, int meta0, int meta1, f32x16* st) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      st[hf] = f32x16{};
      const int sk = (hf ? meta1 : meta0) >> 8 & 0xff;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const i32x8 kf = read_k(ks, hf, s);
#pragma unroll
        for (int p = 0; p < NP; ++p) st[hf] = mfma_scaled(kf, qf[p][s], st[hf], sk, qs[p]);
      }
    }
  };
  auto mask = [&](int meta0, int meta1, f32x16* st) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int held = (hf ? meta1 : meta0) & 0xff;
      if (held < 32) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          st[hf][j] = 8 * (j >> 2) + 4 * hi + (j & 3) < held ? st[hf][j] : -INFINITY;
      }
    }
  };
  // The work on a tile's scores in slices: 8 of maxima, 1 of references, 24 of
  // weights.  A half's weights are 2^(s - ref - e + 8), e the least whole number
  // that keeps them at most 2^8, and their pieces' scales 2^(e - 8): what two
  // (three) pieces leave of a weight is at most 2^-8 (2^-12) of it, or 2^-17 of
  // the half's largest.
  float top[2], nm[2], sum[2], y4[4], climb;   // climb: climb_of the tile's larger V scale
  int e_of[2];
  auto slice = [&](auto c_c, const f32x16* cur, i32x8* pc, int& pcs) {
    constexpr int c = decltype(c_c)::value;
    if constexpr (c < 8) {
      constexpr int hf = c / 4, q4 = c % 4;
      const float x = max3(cur[hf][4 * q4 + 1], cur[hf][4 * q4 + 2], cur[hf][4 * q4 + 3]);
      top[hf] = max3(q4 == 0 ? x : top[hf], cur[hf][4 * q4], x);
    } else if constexpr (c == 8) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) top[hf] = max_xor32(top[hf]) * a.sl2;
      const float both = fmaxf(top[0], top[1]);
      m_true = fmaxf(m_true, both);
      m = m == -INFINITY ? both : m;
      over |= both > m + climb;
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const float e = fmaxf(ceilf(top[hf] - ref), -100.f);
        e_of[hf] = (int)fminf(e, 100.f);
        nm[hf] = 8.f - (float)e_of[hf] - ref;
        sum[hf] = 0.f;
      }
      pcs = (hi ? e_of[1] : e_of[0]) - 8 + 127;
    } else {
      constexpr int q = (c - 9) / 3, part = (c - 9) % 3, hf = q / 4, j4 = q % 4;
      if constexpr (part < 2) {
#pragma unroll
        for (int i = 2 * part; i < 2 * part + 2; ++i) {
          y4[i] = __builtin_amdgcn_exp2f(fmaf(cur[hf][4 * j4 + i], a.sl2, nm[hf]));
          sum[hf] += y4[i];
        }
        asm volatile("" ::"v"(sum[hf]));   // (here, not where it is used)
      } else {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int word = piece4(y4, y4);
          asm volatile("" ::"v"(word));
          pc[p][4 * hf + j4] = word;
        }
      }
    }
  };
  auto add_sums = [&]() {
    l += add_xor32(sum[0]) * pow2i(e_of[0] - 8) + add_xor32(sum[1]) * pow2i(e_of[1] - 8);
  };
  constexpr int SL = 33;

  const int64_t out_at = n * a.so_n + t * a.so_t + h * a.so_h;
  const int64_t gate_at = n * a.sg_n + t * a.sg_t + h * a.sg_h;
  const int rows = min(32, a.R - row0);          // (none or fewer for waves past the end)
  const bool gated = a.gate != nullptr && a.splits == 1;
  constexpr int STEPS = 32 / RPV;                // SHARED: RPV rows a step, 8 elements a lane
  const int sub = lane / CPV, d0 = lane % CPV * 8;
  u32x4 gv[STEPS];

#pragma unroll 1
  for (int pass = 0;; ++pass) {
    l = 0.f;
    m_true = -INFINITY;
    over = false;
#pragma unroll
    for (int i = 0; i < DT; ++i) O[i] = f32x16{};
    if constexpr (SHARED) {
      // Two rings of 4 tiles, K's and then V's.  Step k forms the scores of tile
      // k + 1 and adds tile k - 1 to the output while the vector unit turns tile
      // k's scores into weights: the three are independent, so products and
      // vector work overlap.  K(k) and V(k - 2) have been used by then, and K(k +
      // 4) and V(k + 2) are loaded into their places, three steps before their
      // use; wave w loads the w-th quarter of each, which lies in half w / 2.
      // Tiles past the last are loaded as zeros, which keeps the counts of loads
      // in flight the same.
      constexpr int LW = S::LT / 4;
      uint32_t k_src[LW], v_src[LW];
#pragma unroll
      for (int i = 0; i < LW; ++i) {
        k_src[i] = off_of(0, wave * LW + i) + (LW < 4 ? (wave * LW + i) % 4 * 1024 : 0);
        v_src[i] = off_of(1, wave * LW + i) + (LW < 4 ? (wave * LW + i) % 4 * 1024 : 0);
      }
      auto issue = [&](int kv, int k, u32x4 rsrc) {
        const uint32_t dst = lds0 + (4 * kv + (k & 3)) * S::tile + wave * LW * 1024;
        static_for<LW>([&](auto i_c) {
          constexpr int i = decltype(i_c)::value;
          if constexpr (LW == 4) load_lds16<i * 1024>(rsrc, kv ? v_src[i] : k_src[i], dst);
          else load_lds16<0>(rsrc, kv ? v_src[i] : k_src[i], dst + i * 1024);
        });
      };
      int ring[6][2];                       // meta of the halves of tiles k - 1 .. k + 4
      uint32_t own_lo[3], own_hi[3], own_held[3];   // this wave's half of tiles k + 2 .. k + 4
      auto read_half = [&](int x, int k) {
        const int at = 2 * (k & 31);
        own_lo[x] = __builtin_amdgcn_readlane(code_lo, at + (wave >> 1));
        own_hi[x] = __builtin_amdgcn_readlane(code_hi, at + (wave >> 1));
        own_held[x] = __builtin_amdgcn_readlane(meta, at + (wave >> 1)) & 0xff;
      };
      auto read_ring = [&](int x, int k) {
        ring[x][0] = __builtin_amdgcn_readlane(meta, 2 * (k & 31));
        ring[x][1] = __builtin_amdgcn_readlane(meta, 2 * (k & 31) + 1);
      };
      if (pass > 0) load_first();
      describe(0, first_page);
      wait_vm(0);
      take_q(smem + (4 + wave) * S::tile);
      if (has_suffix) suffix(smem + wave * S::tile, lds0 + wave * S::tile);
      __builtin_amdgcn_s_waitcnt(0xc07f);     // (q is read)
      tile_barrier();
      ring[0][0] = ring[0][1] = 127 << 8 | 127 << 16;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        read_ring(k + 1, k);
        read_half(k < 2 ? 2 : k - 2, k);
        issue(0, k, source(a.kc, own_lo[k < 2 ? 2 : k - 2], own_hi[k < 2 ? 2 : k - 2],
                           own_held[k < 2 ? 2 : k - 2]));
      }
      issue(1, -1, source(a.vc, 0, 0, 0));
      read_half(2, 0);
      issue(1, 0, source(a.vc, own_lo[2], own_hi[2], own_held[2]));
      read_half(2, 1);
      issue(1, 1, source(a.vc, own_lo[2], own_hi[2], own_held[2]));
      split_q();
      // scores and weights of tile k in set k % 2
      f32x16 st[2][2];
      i32x8 pf[2][NP];
      int ps[2];                              // the scale byte of this lane's block of weights
#pragma unroll
      for (int p = 0; p < NP; ++p) pf[1][p] = i32x8{};
      ps[1] = 127;
      wait_vm(6 * LW);                        // K(0)
      tile_barrier();
      scores(smem, ring[1][0], ring[1][1], st[0]);

      auto step = [&](auto x_c, int k) {
        constexpr int x = decltype(x_c)::value, z = 1 - x;
        if (k >= 2) wait_vm(4 * LW);          // K(k + 1) and V(k - 1)
        else wait_vm(2 * LW);
        tile_barrier();
        const uint8_t* ks = smem + (k + 1 & 3) * S::tile;
        const uint8_t* vs = smem + (4 + (k - 1 & 3)) * S::tile;
        constexpr int NF = 4 * KS, MF = NF * NP;
        i32x8 fr[3];
        auto fetch = [&](auto f_c) {
          constexpr int f = decltype(f_c)::value;
          if constexpr (f < 2 * KS) fr[f % 3] = read_k(ks, f / KS, f % KS);
          else if constexpr (f < NF) fr[f % 3] = read_v(vs, f - 2 * KS);
        };
        fetch(std::integral_constant<int, 0>{});
        fetch(std::integral_constant<int, 1>{});
        if ((k + 4 & 31) == 0) describe((k + 4) >> 5, page_at((k + 4) >> 5));
        read_ring(5, k + 4);
        read_half(2, k + 4);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int held = ring[1][hf] & 0xff;
          if (held < 32) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              f32x4 bound;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                bound[i] = 2 * j + 4 * hi + i < held ? INFINITY : -INFINITY;
              float x0 = st[x][hf][j], x1 = st[x][hf][j + 1], x2 = st[x][hf][j + 2],
                    x3 = st[x][hf][j + 3];
              min_acc(x0, x1, x2, x3, bound);
              st[x][hf][j] = x0;
              st[x][hf][j + 1] = x1;
              st[x][hf][j + 2] = x2;
              st[x][hf][j + 3] = x3;
            }
          }
        }
        const int sk[2] = {ring[2][0] >> 8 & 0xff, ring[2][1] >> 8 & 0xff};
        const int sv = (hi ? ring[0][1] : ring[0][0]) >> 16 & 0xff;
        climb = climb_of(max(ring[1][0], ring[1][1]) >> 16);
        __builtin_amdgcn_sched_barrier(0);
        static_for<MF>([&](auto i_c) {
          constexpr int i = decltype(i_c)::value, f = i / NP, p = i % NP;
          if constexpr (p == 0) fetch(std::integral_constant<int, f + 2>{});
          if constexpr (f < 2 * KS) {
            constexpr int hf = f / KS, s = f % KS;
            if constexpr (s == 0 && p == 0)
              st[z][hf] = mfma_scaled(fr[f % 3], qf[p][s], f32x16{}, sk[hf], qs[p]);
            else
              st[z][hf] = mfma_scaled(fr[f % 3], qf[p][s], st[z][hf], sk[hf], qs[p]);
          } else {
            constexpr int dt = f - 2 * KS;
            O[dt] = mfma_scaled(fr[f % 3], pf[z][p], O[dt], sv, ps[z]);
          }
          // K(k + 4) is loaded half way, V(k + 2) three quarters on
          if constexpr (i == MF / 2)
            issue(0, k + 4, source(a.kc, own_lo[2], own_hi[2], own_held[2]));
          if constexpr (i == 3 * MF / 4)
            issue(1, k + 2, source(a.vc, own_lo[0], own_hi[0], own_held[0]));
          constexpr int c0 = i * SL / MF, c1 = (i + 1) * SL / MF;
          static_for<c1 - c0>([&](auto n_c) {
            slice(std::integral_constant<int, c0 + decltype(n_c)::value>{}, st[x], pf[x], ps[x]);
          });
          __builtin_amdgcn_sched_barrier(0);
        });
        // (the products above stay here, not where their results are used)
        asm volatile("" ::"a"(st[z][0]), "a"(st[z][1]));
        add_sums();
#pragma unroll
        for (int i = 0; i < 5; ++i) {
          ring[i][0] = ring[i + 1][0];
          ring[i][1] = ring[i + 1][1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          own_lo[i] = own_lo[i + 1];
          own_hi[i] = own_hi[i + 1];
          own_held[i] = own_held[i + 1];
        }
      };
      using set0 = std::integral_constant<int, 0>;
      using set1 = std::integral_constant<int, 1>;
#pragma unroll 1
      for (int k = 0; k < count; k += 2) {
        step(set0{}, k);
        if (k + 1 == count) {                 // (the last tile's weights to set 1)
#pragma unroll
          for (int p = 0; p < NP; ++p) pf[1][p] = pf[0][p];
          ps[1] = ps[0];
          break;
        }
        step(set1{}, k + 1);
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) gv[s] = u32x4{};
      if (gated) {                            // (on their way during the last tile)
        const T* src[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
          src[s] = (const T*)a.gate + of_lane(gate_at, s * RPV + sub) + d0;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) gv[s] = *(const u32x4*)src[s];
        __builtin_amdgcn_sched_barrier(0);
      }
      // the last tile's output
      const bool any = __ballot(over) != 0;
      if (lane == 0) sm_over[wave] = any;
      wait_vm(0);
      __syncthreads();
      if (count > 0) {
        const uint8_t* vs = smem + (4 + (count - 1 & 3)) * S::tile;
        const int sv = (hi ? ring[0][1] : ring[0][0]) >> 16 & 0xff;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const i32x8 f = read_v(vs, dt);
#pragma unroll
          for (int p = 0; p < NP; ++p) O[dt] = mfma_scaled(f, pf[1][p], O[dt], sv, ps[1]);
        }
      }
      if (pass == 1 || (sm_over[0] | sm_over[1] | sm_over[2] | sm_over[3]) == 0) break;
      __syncthreads();
    } else {
      uint8_t* mine = smem + wave * S::slot;
      const uint32_t mine_at = lds0 + wave * S::slot;
      auto issue = [&](int kv, int k) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int at = 2 * (k & 31) + hf;
          const u32x4 rsrc = source(kv ? a.vc : a.kc, __builtin_amdgcn_readlane(code_lo, at),
                                    __builtin_amdgcn_readlane(code_hi, at),
                                    __builtin_amdgcn_readlane(meta, at) & 0xff);
          const uint32_t dst = mine_at + kv * S::tile + hf * IPH * 1024;
          static_for<IPH>([&](auto i_c) {
            constexpr int i = decltype(i_c)::value;
            load_lds16<i % 4 * 1024>(rsrc, off_of(kv, i), dst + i / 4 * 4096);
          });
        }
      };
      if (pass > 0) load_first();
      describe(0, first_page);
      if (!has_suffix) issue(0, 0);
      if (has_suffix) wait_vm(0);
      else wait_vm(S::LT);
      take_q(mine + S::tile);
      i32x8 pf[NP];
      int ps;
      if (has_suffix) {
        suffix(mine, mine_at);
        issue(0, 0);
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);     // (q is read)
      __builtin_amdgcn_sched_barrier(0);
      issue(1, 0);
      split_q();
#pragma unroll 1
      for (int k = 0; k < count; ++k) {
        const int m0 = __builtin_amdgcn_readlane(meta, 2 * (k & 31));
        const int m1 = __builtin_amdgcn_readlane(meta, 2 * (k & 31) + 1);
        wait_vm(S::LT);              // K of tile k is there, V may be on its way
        f32x16 st[2];
        scores(mine, m0, m1, st);
        // the next tile's K goes where this one's was, once its reads are done
        // (the products above have taken them)
        if ((k + 1 & 31) == 0) describe((k + 1) >> 5, page_at((k + 1) >> 5));
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
        issue(0, k + 1);
        mask(m0, m1, st);
        climb = climb_of(max(m0, m1) >> 16);
        static_for<SL>([&](auto c_c) { slice(c_c, st, pf, ps); });
        add_sums();
        wait_vm(S::LT);
        const int sv = (hi ? m1 : m0) >> 16 & 0xff;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const i32x8 f = read_v(mine + S::tile, dt);
#pragma unroll
          for (int p = 0; p < NP; ++p) O[dt] = mfma_scaled(f, pf[p], O[dt], sv, ps);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_sched_barrier(0);
        issue(1, k + 1);
      }
      wait_vm(0);
      if (pass == 1 || __ballot(over) == 0) break;
    }
    m = over ? m_true + kRoom<T> : m;
    first_page = page_at(0);
  }

  float* ep = (float*)smem + wave * 32 * S::EpiLd;
  auto rows_to_lds = [&]() {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *(f32x4*)(ep + col * S::EpiLd + 32 * dt + 8 * q4 + 4 * hi) =
            f32x4{O[dt][4 * q4], O[dt][4 * q4 + 1], O[dt][4 * q4 + 2], O[dt][4 * q4 + 3]};
    if (spoilt) {   // values that are not finite to the rows that see them
      const int64_t v_at = n * a.ssv_n + kh * a.ssv_h;
#pragma unroll 1
      for (int i = 0; i < 32; ++i) {
        const T* vr = (const T*)a.sv + of_lane(v_at, i);
        const int last = a.Tk - a.T + __shfl(t, i, 64);
#pragma unroll 1
        for (int e = lane; e < (last + 1) * D; e += 64) {
          const float x = Elem<T>::to_f(vr[(int64_t)(e / D) * a.ssv_t + e % D]);
          if (!(fabsf(x) < INFINITY)) ep[i * S::EpiLd + e % D] += x;
        }
      }
    }
  };
  if constexpr (SHARED) {
    // ---- the wave's rows through LDS, RPV rows at a time, 8 elements a lane: whole
    // rows of gates in and of results out
    __syncthreads();                // the rings are free
    rows_to_lds();
    if (a.splits > 1) {
      const int64_t at = ((int64_t)split * a.B * a.HK + bk) * a.R + row0;
      if (hi == 0 && col < rows) {
        a.part_ml[2 * (at + col)] = m;
        a.part_ml[2 * (at + col) + 1] = l;
      }
#pragma unroll 4
      for (int s = 0; s < STEPS; ++s) {
        const int i = s * RPV + sub;
        if (i < rows) {
          float* o = a.part_o + (at + i) * D + d0;
          *(f32x4*)o = *(const f32x4*)(ep + i * S::EpiLd + d0);
          *(f32x4*)(o + 4) = *(const f32x4*)(ep + i * S::EpiLd + d0 + 4);
        }
      }
      return;
    }
    T* to[STEPS];
    float inv[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      to[s] = (T*)a.out + of_lane(out_at, s * RPV + sub) + d0;
      inv[s] = __shfl(l, s * RPV + sub, 64);
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x4 x[2][2];
    auto fetch = [&](int s) {
      const float* o = ep + (s * RPV + sub) * S::EpiLd + d0;
      x[s & 1][0] = *(const f32x4*)o;
      x[s & 1][1] = *(const f32x4*)(o + 4);
    };
    fetch(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s + 1 < STEPS) fetch(s + 1);
      const float f = inv[s] == 0.f ? 0.f : __builtin_amdgcn_rcpf(inv[s]);
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[s & 1][i >> 2][i & 3] * f;
      if (gated) gate8(kind, gv[s], y);
      if (s * RPV + sub < rows)
        *(u32x4*)to[s] = u32x4{pack2(kind, y[0], y[1]), pack2(kind, y[2], y[3]),
                               pack2(kind, y[4], y[5]), pack2(kind, y[6], y[7])};
    }
    return;
  }

  // ---- O^T through LDS, joined over the waves that hold the same rows, then stored
  // (or left as a partial result).  A wave takes 256 / D rows at a time, 4 elements
  // a lane.
  constexpr int LPR = D / 4, RPS = 64 / LPR;     // lanes per row, rows per step
  constexpr int TURNS = (32 / RPS + 3) / 4;
  const int psub = lane / LPR, pd0 = lane % LPR * 4;
  auto first_row = [&](int s) { return (4 * s + wave) * RPS; };
  // the value of the row that this lane stores in step s
  auto of_row = [&](int64_t v, int s) {
    if constexpr (RPS == 1) {
      const int i = first_row(s);
      return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, i) |
                       (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32);
    } else {
      return of_lane(v, first_row(s) + psub);
    }
  };
  wait_vm(0);
  __syncthreads();
  rows_to_lds();
  if (hi == 0) {
    sm_m[wave][col] = m;
    sm_l[wave][col] = l;
  }
  __syncthreads();
#pragma unroll 1
  for (int s = 0; s < TURNS && first_row(s) < rows; ++s) {
    const int i = first_row(s) + psub;
    const int64_t to = of_row(out_at, s), gate_to = of_row(gate_at, s);
    u32x2 gate = u32x2{};
    if (gated) gate = *(const u32x2*)((const T*)a.gate + gate_to + pd0);
    const float mm = fmaxf(fmaxf(sm_m[0][i], sm_m[1][i]), fmaxf(sm_m[2][i], sm_m[3][i]));
    float ll = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float mx = sm_m[x][i];
      const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - mm);
      ll = fmaf(f, sm_l[x][i], ll);
      const f32x4 y = *(const f32x4*)((float*)smem + (x * 32 + i) * S::EpiLd + pd0);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, y[e], o[e]);
    }
    if (i < rows) {
      if (a.splits > 1) {
        const int64_t at = ((int64_t)split * a.B * a.HK + bk) * a.R + row0 + i;
        *(f32x4*)(a.part_o + at * D + pd0) = f32x4{o[0], o[1], o[2], o[3]};
        if (pd0 == 0) {
          a.part_ml[2 * at] = mm;
          a.part_ml[2 * at + 1] = ll;
        }
      } else {
        store_row4<T>((T*)a.out + to + pd0, o, ll == 0.f ? 0.f : 1.f / ll, gated, gate);
      }
    }
  }
}

// Joins the ranges of a split prefix: a wave takes 256 / D rows, 4 elements a
// lane.  Bound by the partial results, which L2 and the memory-side cache mostly
// hold: 3 ranges of 9600 rows of 256 (29 MB read) in 8.2 us, 3.6 TB/s; 4 to 5 us where they
// are few.
template <typename T, int D>
__global__ __launch_bounds__(256) void block_attn_join_kernel(BlockAttnArgs a) {
  constexpr int LPR = D / 4, RPB = 256 / LPR;
  const int64_t rows = (int64_t)a.B * a.HK * a.R;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  const int d0 = threadIdx.x % LPR * 4;
  if (row >= rows) return;
  const int bk = (int)(row / a.R), rr = (int)(row - (int64_t)bk * a.R);
  const int b = bk / a.by_HK, kh = bk - b * a.HK;
  const int rt = rr / a.by_T, t = rr - rt * a.T, w = rt / a.by_G, g = rt - w * a.G;
  const int64_t n = (int64_t)b * a.W + w;
  const int h = kh * a.G + g;
  u32x2 gate = u32x2{};
  if (a.gate)
    gate = *(const u32x2*)((const T*)a.gate + n * a.sg_n + t * a.sg_t + h * a.sg_h + d0);
  // 8 ranges' loads at a time (those past the last repeat it, at no weight)
  const float* ml = a.part_ml + 2 * row;
  const float* po = a.part_o + row * D + d0;
  float mm = -INFINITY, o[4] = {0.f, 0.f, 0.f, 0.f}, ll = 0.f;
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    f32x4 x[8];
    float ms[8], ls[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t s = min(s0 + i, a.splits - 1) * rows;
      ms[i] = ml[2 * s];
      ls[i] = ml[2 * s + 1];
      x[i] = *(const f32x4*)(po + s * D);
    }
    float top = mm;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, ms[i]);
    const float keep = mm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mm - top);
    mm = top;
    ll *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= keep;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool none = ms[i] == -INFINITY || s0 + i >= a.splits;
      const float f = none ? 0.f : __builtin_amdgcn_exp2f(ms[i] - mm);
      ll = fmaf(f, ls[i], ll);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = none ? o[e] : fmaf(f, x[i][e], o[e]);
    }
  }
  store_row4<T>((T*)a.out + n * a.so_n + t * a.so_t + h * a.so_h + d0, o,
                ll == 0.f ? 0.f : 1.f / ll, a.gate != nullptr, gate);
}

// The launch of a call: whether the waves share tiles, and the ranges the
// prefix is split into, whichever a count of nanoseconds finds cheapest.
// 256 workgroups (one a CU) run as a round; a round costs 30 D to start and end,
// and for each step of its walk
//   private: 600 + 6 D (four tiles for 32 rows; each wave waits for its own),
//   shared:  800 + 3 D (one tile for 128 rows), and 2000 a call, its rings' filling
// and a split costs 2000 for the second kernel and 0.3 a KB of partial results.
// Fitted to 3507 measured (form, ranges) of 306 calls, bf16 and fp16, D 64 to 256, 1 to
// 100 requests, 256 to 20000 keys, 4 to 1024 rows and one suffix key: what it takes is
// 0.6% slower than the best measured choice in the mean and 12% at worst.  It counts
// the tokens that the tables can hold, as the lengths are on the GPU, and neither the
// suffix nor the pieces.  (A limit in rows alone,
// shared from 65 on, lost 7 to 25% in the mean and up to 2.6 times.)  Both sides, us,
// bf16, 2 KV heads:
//                                    private  shared
//   D 256,  64 requests,  256 keys,   64 rows   18.4    23.4
//                                     96 rows   33.4    23.8
//                                   1024 rows  232.5    98.0
//   D 256,   1 request,  8192 keys,  128 rows   23.0    28.5
//                                   1024 rows   39.4    46.0
//   D 128,   8 requests, 4096 keys, 1024 rows   58.0    63.8
//   D 128, 100 requests,  640 keys,   96 rows   27.9    25.5
// Of the choices that a grid holds: fewer than 2^32 work-items, so fewer than 2^24
// workgroups of 256 (splits 0: there is none).
struct Plan {
  bool shared;
  int nqblk, splits;
};

Plan plan_of(int B, int HK, int R, int D, int keys) {
  Plan p = {};
  const int tiles = (int)kad_cdiv(keys, kKeys);
  const double most = (1 << 24) - 1;
  double best = INFINITY;
  for (int form = 0; form < 2; ++form) {
    const bool shared = form == 1;
    const int nqblk = (int)kad_cdiv(R, shared ? 128 : 32), step = shared ? 1 : 4;
    const double per_step = shared ? 800 + 3 * D : 600 + 6 * D;
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (s > 1 && tiles < s * step) break;
      const int walk = ((tiles + s - 1) / s + step - 1) / step;
      const double blocks = (double)B * HK * nqblk * s;
      if (blocks > most || (s > 1 && (double)B * HK * R / (1024 / D) > most)) break;
      const double rounds = std::ceil(blocks / 256);
      double cost = rounds * (30 * D + walk * per_step) + (shared ? 2000 : 0);
      if (s > 1) cost += 2000 + 0.0003 * s * B * HK * R * D * 4;
      if (cost < best) {
        best = cost;
        p = Plan{shared, nqblk, s};
      }
    }
  }
  return p;
}

// a KV head's rows in 32 bits and all rows in 64 (doubles hold any product)
bool rows_fit(int B, int W, int T, int H, int HK) {
  const double R = (double)W * T * (H / HK);
  return R <= 0x7fffffff - 256 && B * (double)HK * R / 4 <= 0x7fffffff;
}

int64_t workspace_of(const Plan& p, int B, int HK, int R, int D) {
  return p.splits > 1 ? (int64_t)p.splits * B * HK * R * (D + 2) * 4 : 0;
}

template <typename T, int D>
int launch(const BlockAttnArgs& a, bool shared, hipStream_t stream) {
  constexpr int lds = Shape<D>::lds;
  const void* f = shared ? (const void*)block_attn_kernel<T, D, true>
                         : (const void*)block_attn_kernel<T, D, false>;
  if (lds > 64 * 1024 &&
      hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
    kad_set_error("block_attn_kernel: %d bytes of LDS refused", lds);
    return KAD_ERR_HIP;
  }
  const dim3 grid((unsigned)((int64_t)a.B * a.HK * a.splits * a.nqblk));
  if (shared)
    hipLaunchKernelGGL((block_attn_kernel<T, D, true>), grid, dim3(256), lds, stream, a);
  else
    hipLaunchKernelGGL((block_attn_kernel<T, D, false>), grid, dim3(256), lds, stream, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((block_attn_join_kernel<T, D>),
                       dim3((unsigned)kad_cdiv((int64_t)a.B * a.HK * a.R, 1024 / D)), dim3(256),
                       0, stream, a);
  return kad_launch_status("block_attn_kernel");
}

template <typename T>
int launch_d(const BlockAttnArgs& a, int D, bool shared, hipStream_t stream) {
  if (D == 64) return launch<T, 64>(a, shared, stream);
  if (D == 128) return launch<T, 128>(a, shared, stream);
  return launch<T, 256>(a, shared, stream);
}

bool aligned(const void* p, int64_t s0, int64_t s1, int64_t s2, int elements) {
  return ((uintptr_t)p % (2 * elements)) == 0 && s0 % elements == 0 && s1 % elements == 0 &&
         s2 % elements == 0;
}

}  // namespace

extern "C" int kad_block_prefix_attention_workspace_bytes(int B, int W, int T, int H, int HK,
                                                          int D, int width, int block,
                                                          int64_t* bytes) {
  KAD_REQUIRE(bytes, "null pointer argument");
  KAD_REQUIRE(B > 0 && W > 0 && T > 0 && H > 0 && HK > 0 && H % HK == 0 && width > 0,
              "empty dimensions");
  KAD_REQUIRE(D == 64 || D == 128 || D == 256, "head dim %d is not 64, 128 or 256", D);
  KAD_REQUIRE(block > 0 && (int64_t)width * block <= 1 << 30, "tables of %d columns of %d tokens",
              width, block);
  KAD_REQUIRE(rows_fit(B, W, T, H, HK), "too many rows for a launch");
  const int R = W * T * (H / HK);
  const Plan p = plan_of(B, HK, R, D, width * block);
  KAD_REQUIRE(p.splits > 0, "too many rows for a launch");
  *bytes = workspace_of(p, B, HK, R, D);
  return KAD_OK;
}

extern "C" int kad_block_prefix_attention(
    const void* q, int64_t sq_n, int64_t sq_t, int64_t sq_h, const void* k_codes,
    const void* v_codes, const void* k_scale, const void* v_scale, int pages,
    const int32_t* tables, int width, const int32_t* lengths, const void* suffix_k,
    int64_t ssk_n, int64_t ssk_t, int64_t ssk_h, const void* suffix_v, int64_t ssv_n,
    int64_t ssv_t, int64_t ssv_h, const void* gate, int64_t sg_n, int64_t sg_t, int64_t sg_h,
    void* out, int64_t so_n, int64_t so_t, int64_t so_h, void* workspace,
    int64_t workspace_bytes, int B, int W, int T, int Tk, int H, int HK, int D, int block,
    int dtype, float scale, kad_stream_t stream) {
  KAD_REQUIRE(B > 0 && W > 0 && T > 0 && H > 0 && HK > 0 && width > 0 && pages > 0,
              "empty dimensions");
  KAD_REQUIRE(H % HK == 0, "%d heads over %d KV heads", H, HK);
  KAD_REQUIRE(Tk == 0 || Tk >= T, "a suffix of %d keys for %d queries", Tk, T);
  // (a wave numbers the suffix keys of up to 32 beams, and the elements of one beam's
  // values, in 32 bits)
  KAD_REQUIRE(Tk <= 1 << 22, "a suffix of %d keys", Tk);
  KAD_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && tables && lengths && out &&
                  (Tk == 0 || (suffix_k && suffix_v)),
              "null pointer argument");
  KAD_REQUIRE(D == 64 || D == 128 || D == 256, "head dim %d is not 64, 128 or 256", D);
  KAD_REQUIRE(block == 32 || block == 64 || block == 128 || block == 256,
              "block size %d is not 32, 64, 128 or 256", block);
  KAD_REQUIRE(aligned(k_codes, 0, 0, 0, 8) && aligned(v_codes, 0, 0, 0, 8) &&
                  aligned(q, sq_n, sq_t, sq_h, 8),
              "codes and query rows must be 16-byte aligned");
  KAD_REQUIRE(Tk == 0 || (aligned(suffix_k, ssk_n, ssk_t, ssk_h, 8) &&
                          aligned(suffix_v, ssv_n, ssv_t, ssv_h, 8)),
              "suffix rows must be 16-byte aligned");
  KAD_REQUIRE(aligned(out, so_n, so_t, so_h, 8) && (!gate || aligned(gate, sg_n, sg_t, sg_h, 8)),
              "gate and output rows must be 16-byte aligned");
  if (dtype != KAD_DTYPE_BF16 && dtype != KAD_DTYPE_F16)
    KAD_UNSUPPORTED("dtype code %d: queries are bf16 or fp16", dtype);
  KAD_REQUIRE((int64_t)width * block <= 1 << 30, "tables of %d columns of %d tokens", width, block);
  KAD_REQUIRE(rows_fit(B, W, T, H, HK), "too many rows for a launch");
  const int R = W * T * (H / HK);
  const Plan p = plan_of(B, HK, R, D, width * block);
  KAD_REQUIRE(p.splits > 0, "too many rows for a launch");
  const int64_t need = workspace_of(p, B, HK, R, D);
  KAD_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
              "a workspace of %lld bytes at a 16-byte boundary is needed", (long long)need);
  BlockAttnArgs a = {};
  a.q = q; a.sq_n = sq_n; a.sq_t = sq_t; a.sq_h = sq_h;
  a.kc = (const uint8_t*)k_codes; a.vc = (const uint8_t*)v_codes;
  a.ksc = (const uint8_t*)k_scale; a.vsc = (const uint8_t*)v_scale;
  a.tables = tables; a.lengths = lengths;
  a.sk = suffix_k; a.ssk_n = ssk_n; a.ssk_t = ssk_t; a.ssk_h = ssk_h;
  a.sv = suffix_v; a.ssv_n = ssv_n; a.ssv_t = ssv_t; a.ssv_h = ssv_h;
  a.gate = gate; a.sg_n = sg_n; a.sg_t = sg_t; a.sg_h = sg_h;
  a.out = out; a.so_n = so_n; a.so_t = so_t; a.so_h = so_h;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + (int64_t)p.splits * B * HK * R * D;
  a.pages = pages; a.width = width; a.B = B; a.W = W; a.T = T; a.Tk = Tk; a.H = H; a.HK = HK;
  a.lblock = block == 32 ? 5 : block == 64 ? 6 : block == 128 ? 7 : 8;
  a.splits = p.splits; a.nqblk = p.nqblk; a.R = R; a.G = H / HK;
  a.by_splits = divide_by(a.splits); a.by_nqblk = divide_by(a.nqblk);
  a.by_HK = divide_by(HK); a.by_G = divide_by(a.G); a.by_T = divide_by(T);
  a.by_Tk = divide_by(Tk > 0 ? Tk : 1);
  const float log2e = 1.4426950408889634f;
  a.qmul = scale > 0.f ? 1.f : scale < 0.f ? -1.f : scale == 0.f ? 0.f : scale;
  a.sl2 = scale == 0.f ? log2e : fabsf(scale) * log2e;
  return dtype == KAD_DTYPE_BF16 ? launch_d<bf16_t>(a, D, p.shared, (hipStream_t)stream)
                                 : launch_d<_Float16>(a, D, p.shared, (hipStream_t)stream);
}
