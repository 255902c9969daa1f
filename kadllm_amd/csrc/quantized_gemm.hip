// Products with 4-bit weights (quantized_weight.hip's layout):
//   linear  y = x W^T (+ r)
//   gated   h = silu(x G^T) * (x U^T), both projections in one kernel
// and the feed-forward block y = h D^T (+ r) of the two.
//
// The weight's values are exact in bf16 and go to v_mfma_f32_16x16x32_bf16 as they
// are; what x has more bits than bf16 goes as further products: x is the sum of
// bf16 pieces, one for bf16, two for fp16 (11 bits) and three for fp32 (24 bits),
// each the leading bits of what is left, so the sum is x itself.  Sums are fp32 and
// are rounded once, with the residual added.  The gated product h is rounded to one
// bf16 piece for bf16 x (2^-8, as the model's own activation), else to as many
// pieces as x has: 2^-15 for fp16, whose range h may leave, and 2^-22 for fp32.

#include "quantized_common.h"

namespace {

using namespace kad_q4;

template <typename T> constexpr int kPieces = sizeof(T) == 4 ? 3 : 2;
template <> constexpr int kPieces<bf16_t> = 1;

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

// Rows of x as bf16 pieces [P][M][KP], zeros past column K.  8 elements a thread.
template <typename T>
__global__ __launch_bounds__(256) void split_rows_kernel(const T* __restrict__ x, int64_t ldx,
                                                         bf16_t* __restrict__ out, int M, int K,
                                                         int KP) {
  constexpr int P = kPieces<T>;
  const int per_row = KP / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = i / per_row;
  if (m >= M) return;
  const int k = (int)(i - m * per_row) * 8;
  uint32_t w[P][4];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float f = k + e < K ? Elem<T>::to_f(x[m * ldx + k + e]) : 0.f;
    bf16_t p[P];
    split<P>(f, p);
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
  const bf16_t* x;           // pieces of the rows: (p, m, k) at x[p * xp + m * ldx + k]
  int64_t ldx, xp;
  const uint8_t* codes[2];   // the weight, or gate and up
  const uint8_t* scales[2];
  const void* r;             // residual (linear; may be null)
  int64_t ldr;
  void* y;                   // linear: rows of T; gated: pieces, (p, m, n) as for x
  int64_t ldy, yp;
  int M, N, KB;
  int cols;                  // columns that are written: N, or (gated) N padded to 128
  int vec;                   // 4 neighbours of y (and r) may go as one access
};

// a word of 8 codes times its group's scale, as an MFMA operand
__device__ __forceinline__ bf16x8 operand(uint32_t codes, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T>
__device__ __forceinline__ float silu_of(float g) {
  if constexpr (sizeof(T) == 4) return g / (1.0f + expf(-g));
  else return silu_f(g);
}

// Outputs (m, n .. n + 3) from their sums: s[0], or the gate's and the up's.
template <typename T, bool GATED>
__device__ __forceinline__ void finish(const Args& a, int m, int n, const f32x4* s) {
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
    const T* r = (const T*)a.r + (a.r ? m * a.ldr + n : 0);
    if (a.vec) {
      typedef T vec4 __attribute__((ext_vector_type(4)));
      f32x4 f = s[0];
      if (a.r) {
        const vec4 v = *(const vec4*)r;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] += Elem<T>::to_f(v[i]);
      }
      vec4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = Elem<T>::from_f(f[i]);
      *(vec4*)y = o;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) y[i] = Elem<T>::from_f(a.r ? s[0][i] + Elem<T>::to_f(r[i]) : s[0][i]);
    }
  }
}

// One workgroup: 16 rows of x and 16 of the weight(s), K split over its 4 waves, whose
// sums meet in LDS.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void q4_kernel(Args a) {
  constexpr int P = kPieces<T>, W = GATED ? 2 : 1, KS = 4;
  __shared__ f32x4 part[KS][W][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
  const int nt = blockIdx.x, m0 = blockIdx.y * 16;
  const int NB = (a.N + 15) / 16, nb = min(nt, NB - 1), K4 = (a.KB + 3) / 4;
  f32x4 acc[W];
#pragma unroll
  for (int w = 0; w < W; ++w) acc[w] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bf16_t* x = a.x + (int64_t)min(m0 + fr, a.M - 1) * a.ldx + fq * 32;
  for (int kb = wave; kb < a.KB; kb += KS) {
    u32x4 c[W];
    float scale[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      c[w] = *(const u32x4*)(a.codes[w] + (((int64_t)nb * a.KB + kb) * 64 + lane) * 16);
      const uint32_t s =
          a.scales[w][(((int64_t)nb * K4 + (kb >> 2)) * 64 + lane) * 4 + (kb & 3)];
      scale[w] = __uint_as_float(s << 23);
    }
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bf16x8 xf = as_bf16x8(*(const u32x4*)(x + p * a.xp + kb * 128 + j * 8));
#pragma unroll
        for (int w = 0; w < W; ++w) acc[w] = mfma16x16x32(operand(c[w][j], scale[w]), xf, acc[w]);
      }
  }
#pragma unroll
  for (int w = 0; w < W; ++w) part[wave][w][lane] = acc[w];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int w = 0; w < W; ++w)
      for (int i = 1; i < KS; ++i) acc[w] += part[i][w][lane];
    finish<T, GATED>(a, m0 + fr, nt * 16 + fq * 4, acc);
  }
}

int64_t pad128(int64_t k) { return kad_cdiv(k, 128) * 128; }

template <typename T>
bool in_place(const void* x, int64_t ldx, int K) {
  return kPieces<T> == 1 && K % 128 == 0 && (uintptr_t)x % 16 == 0 && ldx % 8 == 0;
}

// bytes of the rows' pieces; 0 where the rows can be read as they are
template <typename T>
int64_t piece_bytes(const void* x, int64_t ldx, int M, int K) {
  return in_place<T>(x, ldx, K) ? 0 : kPieces<T> * (int64_t)M * pad128(K) * 2;
}

// a.x, a.ldx, a.xp for the rows, split into `ws` where they cannot be read in place
template <typename T>
void rows_of(Args& a, const void* x, int64_t ldx, void* ws, int M, int K, hipStream_t s) {
  if (in_place<T>(x, ldx, K)) {
    a.x = (const bf16_t*)x, a.ldx = ldx, a.xp = 0;
    return;
  }
  const int KP = (int)pad128(K);
  a.x = (const bf16_t*)ws, a.ldx = KP, a.xp = (int64_t)M * KP;
  hipLaunchKernelGGL((split_rows_kernel<T>), dim3((unsigned)kad_cdiv((int64_t)M * (KP / 8), 256)),
                     dim3(256), 0, s, (const T*)x, ldx, (bf16_t*)ws, M, K, KP);
}

template <typename T, bool GATED>
void launch(const Args& a, hipStream_t s) {
  const dim3 grid((unsigned)kad_cdiv(a.cols, 16), (unsigned)kad_cdiv(a.M, 16));
  hipLaunchKernelGGL((q4_kernel<T, GATED>), grid, dim3(256), 0, s, a);
}

struct Weight {
  const void *codes, *scales;
};

template <typename T>
void linear(Args a, Weight w, const void* r, int64_t ldr, void* y, int64_t ldy, int M, int N,
            int K, hipStream_t s) {
  a.codes[0] = a.codes[1] = (const uint8_t*)w.codes;
  a.scales[0] = a.scales[1] = (const uint8_t*)w.scales;
  a.r = r, a.ldr = ldr, a.y = y, a.ldy = ldy, a.yp = 0;
  a.M = M, a.N = N, a.KB = (int)kad_cdiv(K, 128), a.cols = N;
  const int bytes = 4 * (int)sizeof(T);
  a.vec = N % 4 == 0 && (uintptr_t)y % bytes == 0 && ldy % 4 == 0 &&
          (!r || ((uintptr_t)r % bytes == 0 && ldr % 4 == 0));
  launch<T, false>(a, s);
}

template <typename T>
void gated(Args a, Weight g, Weight u, bf16_t* h, int M, int F, int K, hipStream_t s) {
  a.codes[0] = (const uint8_t*)g.codes, a.codes[1] = (const uint8_t*)u.codes;
  a.scales[0] = (const uint8_t*)g.scales, a.scales[1] = (const uint8_t*)u.scales;
  a.r = nullptr, a.ldr = 0, a.y = h, a.ldy = pad128(F), a.yp = M * pad128(F);
  a.M = M, a.N = F, a.KB = (int)kad_cdiv(K, 128), a.cols = (int)pad128(F), a.vec = 1;
  launch<T, true>(a, s);
}

int check_sizes(int M, int N, int K) {
  KAD_REQUIRE(M > 0 && N > 0 && K > 0, "empty dimensions");
  KAD_REQUIRE(K <= kMaxK, "rows of %d columns", K);
  // (a grid holds fewer than 2^32 work-items a dimension)
  KAD_REQUIRE(kad_cdiv(M, 16) <= 65535 && N <= kMaxN, "a product of %d x %d outputs", M, N);
  return KAD_OK;
}

int check_weight(Weight w) {
  KAD_REQUIRE(w.codes && w.scales, "null pointer argument");
  KAD_REQUIRE((uintptr_t)w.codes % 16 == 0 && (uintptr_t)w.scales % 16 == 0,
              "codes and scales must be 16-byte aligned");
  return KAD_OK;
}

#define KAD_TRY(call)                    \
  do {                                   \
    if (const int rc = (call)) return rc; \
  } while (0)

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
    *bytes = piece_bytes<decltype(t)>(x, ldx, M, K);
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
    Args a{};
    rows_of<T>(a, x, ldx, workspace, M, K, (hipStream_t)stream);
    linear<T>(a, {codes, scales}, residual, ldr, y, ldy, M, N, K, (hipStream_t)stream);
    return kad_launch_status("q4_kernel");
  });
}

extern "C" int kad_quantized_gated_ffn_workspace_bytes(const void* x, int64_t ldx, int dtype,
                                                       int M, int H, int F, int64_t* bytes) {
  KAD_REQUIRE(bytes, "null pointer argument");
  KAD_TRY(check_sizes(M, F, H));
  KAD_TRY(check_sizes(M, H, F));
  return for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    *bytes = piece_bytes<T>(x, ldx, M, H) + kPieces<T> * (int64_t)M * pad128(F) * 2;
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
    Args a{};
    rows_of<T>(a, x, ldx, workspace, M, H, s);
    bf16_t* h = (bf16_t*)((char*)workspace + piece_bytes<T>(x, ldx, M, H));
    gated<T>(a, g, u, h, M, F, H, s);
    a.x = h, a.ldx = pad128(F), a.xp = M * pad128(F);
    linear<T>(a, d, residual, ldr, y, ldy, M, H, F, s);
    return kad_launch_status("q4_kernel");
  });
}
