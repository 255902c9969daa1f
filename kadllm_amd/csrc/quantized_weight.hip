// Weights in 4 bits: quantising them and reading them back.
//
// A weight [N, K] is held in groups of 32 neighbours of a row: e2m1 codes (0,
// 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) and one e8m0 scale, the power of
// two 2^(byte - 127).  A code has two significant bits, so code * scale is exact in
// bf16, and what the products of quantized_gemm.hip multiply by is the value itself.
//
// Rows are padded to 16 and columns to 128 with zero codes, and laid out as the
// MFMA's operand takes them: codes [N/16][K/128][64 lanes][4 words], word j of lane l
// the 8 codes of row l % 16, columns 32 j + 8 (l / 16) .. +7 (the first column in the lowest
// bits), so a wave loads 1 KB in one piece and word j is the lane's part of the j-th
// product of 32 columns; scales [N/16][K/128][16 rows][4 groups], a word a lane.

#include "quantized_common.h"

namespace {

using namespace kad_q4;

// The scale's byte of a group whose largest magnitude is amax: the smallest e in
// [-100, 125] with amax <= 7 * 2^e.  Up to 7 the rounding of the largest element is
// off by at most 2^e, half the step between 4 and 6; 125 keeps 6 * 2^e finite.
// amax = 1.m * 2^x and 7 = 1.75 * 2^2.  255 (NaN) where amax is not finite, and 2^0 for a
// group of zeros (which the products take for a value like others').
__device__ __forceinline__ uint32_t scale_byte(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits >= 0x7f800000u) return 255u;
  if (bits == 0u) return 127u;
  const int e = (int)(bits >> 23) - 127 - 2 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(min(max(e, -100), 125) + 127);
}

// the larger, and a NaN where either is one
__device__ __forceinline__ float max_nan(float a, float b) {
  return (__float_as_uint(a) > __float_as_uint(b)) ? a : b;  // (non-negative or NaN)
}

// One workgroup takes 4 blocks of 16 rows and 128 columns, in a row of blocks' order: a wave
// 4 rows, 16 lanes a row, so that a load instruction reads 4 whole runs of 16 x 8 elements.
// A group is 4 lanes.  Everything is loaded before the first use.  Memory bounds it: 248320 x
// 1024 from bf16, 0.64 GB, 114 us (5.6 TB/s; 144 us from memory that no cache holds), 3584 x
// 1024 4.6 us, 3370 x 3437, where a row's lines are shared with the next, 7.9 us (3.7 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* __restrict__ w, int64_t ldw,
                                                              uint8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, int N,
                                                              int K, int KB) {
  const int lane = threadIdx.x & 63, r = (threadIdx.x >> 6) * 4 + (lane >> 4), c = lane & 15;
  const int NB = (N + 15) / 16;
  int nb[4], kb[4], left[4];
  const T* row[4];
  T v[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = blockIdx.x * 4 + j;
    nb[j] = (int)(b / (uint32_t)KB), kb[j] = (int)(b - (uint32_t)nb[j] * (uint32_t)KB);
    const int n = nb[j] * 16 + r;
    row[j] = w + min(n, N - 1) * ldw;
    left[j] = n < N ? K - (kb[j] * 128 + c * 8) : 0;
  }
  // one access, wherever it begins, and on no condition of the lane's, so that the four go
  // out together; lanes at the row's end read its last 8, and their own below
  if (K >= 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_memcpy(v[j], row[j] + min(kb[j] * 128 + c * 8, K - 8), sizeof(v[j]));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (left[j] < 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = i < left[j] ? row[j][K - left[j] + i] : T(0);
    }
  const int at = ((c & 3) * 16 + r) * 16 + (c >> 2) * 4;  // of the codes' word in its block
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float f[8], amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = Elem<T>::to_f(v[j][i]);
      amax = max_nan(amax, fabsf(f[i]));
    }
    amax = max_nan(amax, __shfl_xor(amax, 1, 64));
    amax = max_nan(amax, __shfl_xor(amax, 2, 64));
    const uint32_t s = scale_byte(amax);
    if (nb[j] < NB) {
      const int64_t block = (int64_t)nb[j] * KB + kb[j];
      uint32_t code = 0;
      const float scale = __uint_as_float(s << 23);
      if (s != 255u) {
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[0], f[1], scale, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[2], f[3], scale, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[4], f[5], scale, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[6], f[7], scale, 3);
      }
      *(uint32_t*)(codes + block * 1024 + at) = code;
      if ((c & 3) == 0) scales[block * 64 + r * 4 + (c >> 2)] = (uint8_t)s;
    }
  }
}

// The same split the other way (111 us, 5.8 TB/s; 4.3 us; 7.6 us, 3.8 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void dequantize_weight_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
    int64_t ldo, int N, int K, int KB) {
  const int lane = threadIdx.x & 63, r = (threadIdx.x >> 6) * 4 + (lane >> 4), c = lane & 15;
  const int NB = (N + 15) / 16;
  const int at = ((c & 3) * 16 + r) * 16 + (c >> 2) * 4;
  int nb[4], kb[4];
  uint32_t code[4], byte[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t b = blockIdx.x * 4 + j;
    nb[j] = (int)(b / (uint32_t)KB), kb[j] = (int)(b - (uint32_t)nb[j] * (uint32_t)KB);
    const int64_t block = (int64_t)min(nb[j], NB - 1) * KB + kb[j];
    code[j] = *(const uint32_t*)(codes + block * 1024 + at);
    byte[j] = scales[block * 64 + r * 4 + (c >> 2)];
  }
  T y[4][8], *dst[4];
  int left[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = nb[j] * 16 + r, k = kb[j] * 128 + c * 8;
    dst[j] = out + n * ldo + k;
    left[j] = n < N ? K - k : 0;
    const float scale = scale_value(byte[j]);
    float f[8];
    codes_to_float(code[j], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[j][i] = Elem<T>::from_f(f[i] * scale);
    if (left[j] >= 8) __builtin_memcpy(dst[j], y[j], sizeof(y[j]));  // (wherever it begins)
  }
  // the rows' ends (beside the whole 8 the compiler would split those for what both store)
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (left[j] < 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left[j]) dst[j][i] = y[j][i];
    }
}

int check(const void* w, const void* codes, const void* scales, int N, int K, int64_t ld) {
  KAD_REQUIRE(N > 0 && K > 0, "empty dimensions");
  KAD_REQUIRE(w && codes && scales, "null pointer argument");
  KAD_REQUIRE(ld >= K, "rows of %d columns at stride %lld", K, (long long)ld);
  KAD_REQUIRE(K <= kMaxK && N <= kMaxN, "a weight of %d rows of %d columns", N, K);
  KAD_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0,
              "codes and scales must be 16-byte aligned");
  // (a grid holds fewer than 2^32 work-items a dimension: 256 for 4 blocks)
  KAD_REQUIRE(kad_cdiv(N, 16) * kad_cdiv(K, 128) <= (1ll << 26) - 4, "too large a weight");
  return KAD_OK;
}

template <typename T>
void launch_quantize(const void* w, int64_t ldw, void* codes, void* scales, int N, int K,
                     hipStream_t s) {
  const int KB = (int)kad_cdiv(K, 128);
  const dim3 grid((unsigned)kad_cdiv(kad_cdiv(N, 16) * KB, 4));
  hipLaunchKernelGGL(quantize_weight_kernel<T>, grid, dim3(256), 0, s, (const T*)w, ldw,
                     (uint8_t*)codes, (uint8_t*)scales, N, K, KB);
}

template <typename T>
void launch_dequantize(const void* codes, const void* scales, void* out, int64_t ldo, int N, int K,
                       hipStream_t s) {
  const int KB = (int)kad_cdiv(K, 128);
  const dim3 grid((unsigned)kad_cdiv(kad_cdiv(N, 16) * KB, 4));
  hipLaunchKernelGGL(dequantize_weight_kernel<T>, grid, dim3(256), 0, s, (const uint8_t*)codes,
                     (const uint8_t*)scales, (T*)out, ldo, N, K, KB);
}

}  // namespace

extern "C" int kad_quantize_weight(const void* w, int64_t ldw, int dtype, void* codes,
                                   void* scales, int N, int K, kad_stream_t stream) {
  if (const int rc = check(w, codes, scales, N, K, ldw)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == KAD_DTYPE_BF16) launch_quantize<bf16_t>(w, ldw, codes, scales, N, K, s);
  else if (dtype == KAD_DTYPE_F16) launch_quantize<_Float16>(w, ldw, codes, scales, N, K, s);
  else if (dtype == KAD_DTYPE_F32) launch_quantize<float>(w, ldw, codes, scales, N, K, s);
  else KAD_UNSUPPORTED("dtype code %d", dtype);
  return kad_launch_status("quantize_weight_kernel");
}

extern "C" int kad_dequantize_weight(const void* codes, const void* scales, void* out, int64_t ldo,
                                     int dtype, int N, int K, kad_stream_t stream) {
  if (const int rc = check(out, codes, scales, N, K, ldo)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == KAD_DTYPE_BF16) launch_dequantize<bf16_t>(codes, scales, out, ldo, N, K, s);
  else if (dtype == KAD_DTYPE_F16) launch_dequantize<_Float16>(codes, scales, out, ldo, N, K, s);
  else if (dtype == KAD_DTYPE_F32) launch_dequantize<float>(codes, scales, out, ldo, N, K, s);
  else KAD_UNSUPPORTED("dtype code %d", dtype);
  return kad_launch_status("dequantize_weight_kernel");
}
