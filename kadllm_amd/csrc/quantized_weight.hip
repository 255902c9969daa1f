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

// 8 neighbours of a row as floats; zeros past the row's end
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int left, float* f) {
  if (VEC && left >= 8) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const f32x4 x = *(const f32x4*)(p + 4 * v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * v + i] = x[i];
      }
    } else {
      typedef T vec8 __attribute__((ext_vector_type(8)));
      const vec8 x = *(const vec8*)p;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to_f(x[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < left ? Elem<T>::to_f(p[i]) : 0.f;
  }
}

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

// One workgroup takes 16 rows and 512 columns: a wave 4 rows, 16 lanes a row and
// block of 128, so that a load instruction reads 4 whole runs of 16 x 8 elements.  A
// group is 4 lanes.  Everything is loaded before the first use.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* __restrict__ w, int64_t ldw,
                                                              uint8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, int N,
                                                              int K, int KB) {
  const int lane = threadIdx.x & 63, r = (threadIdx.x >> 6) * 4 + (lane >> 4), c = lane & 15;
  const int K4 = (KB + 3) / 4;
  const int64_t nb = blockIdx.x / K4;
  const int k4 = (int)(blockIdx.x - nb * K4);
  const int64_t row = nb * 16 + r;
  float f[4][8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = (k4 * 4 + j) * 128 + c * 8;
    if (row < N && k < K) {
      load8<T, VEC>(w + row * ldw + k, K - k, f[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
    }
  }
  const int at = ((c & 3) * 16 + r) * 16 + (c >> 2) * 4;  // of the codes' word in its block
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int kb = k4 * 4 + j;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(f[j][i]));
    amax = max_nan(amax, __shfl_xor(amax, 1, 64));
    amax = max_nan(amax, __shfl_xor(amax, 2, 64));
    const uint32_t s = scale_byte(amax);
    if (kb < KB) {
      uint32_t code = 0;
      const float scale = __uint_as_float(s << 23);
      if (s != 255u) {
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[j][0], f[j][1], scale, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[j][2], f[j][3], scale, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[j][4], f[j][5], scale, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, f[j][6], f[j][7], scale, 3);
      }
      *(uint32_t*)(codes + (nb * KB + kb) * 1024 + at) = code;
      if ((c & 3) == 0) scales[(nb * KB + kb) * 64 + r * 4 + (c >> 2)] = (uint8_t)s;
    }
  }
}

// The same split the other way.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dequantize_weight_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
    int64_t ldo, int N, int K, int KB) {
  const int lane = threadIdx.x & 63, r = (threadIdx.x >> 6) * 4 + (lane >> 4), c = lane & 15;
  const int K4 = (KB + 3) / 4;
  const int64_t nb = blockIdx.x / K4;
  const int k4 = (int)(blockIdx.x - nb * K4);
  const int64_t row = nb * 16 + r;
  if (row >= N) return;
  const int at = ((c & 3) * 16 + r) * 16 + (c >> 2) * 4;
  uint32_t code[4], byte[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int kb = min(k4 * 4 + j, KB - 1);
    code[j] = *(const uint32_t*)(codes + (nb * KB + kb) * 1024 + at);
    byte[j] = scales[(nb * KB + kb) * 64 + r * 4 + (c >> 2)];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = (k4 * 4 + j) * 128 + c * 8;
    if (k >= K) continue;
    const float scale = scale_value(byte[j]);
    float f[8];
    codes_to_float(code[j], f);
    T* dst = out + row * ldo + k;
    T y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = Elem<T>::from_f(f[i] * scale);
    if (VEC && K - k >= 8) {
      u32x4 v[sizeof(T) / 2];
      __builtin_memcpy(v, y, sizeof(y));
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((u32x4*)dst)[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < K - k) dst[i] = y[i];
    }
  }
}

template <typename T>
bool rows16(const T* p, int64_t ld) {
  return (uintptr_t)p % 16 == 0 && ld * (int64_t)sizeof(T) % 16 == 0;
}

int check(const void* w, const void* codes, const void* scales, int N, int K, int64_t ld) {
  KAD_REQUIRE(N > 0 && K > 0, "empty dimensions");
  KAD_REQUIRE(w && codes && scales, "null pointer argument");
  KAD_REQUIRE(ld >= K, "rows of %d columns at stride %lld", K, (long long)ld);
  KAD_REQUIRE(K <= kMaxK, "rows of %d columns", K);
  KAD_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)scales % 16 == 0,
              "codes and scales must be 16-byte aligned");
  // (a grid holds fewer than 2^32 work-items a dimension)
  KAD_REQUIRE(kad_cdiv(N, 16) * kad_cdiv(K, 512) < (1ll << 32) / 256, "too large a weight");
  return KAD_OK;
}

template <typename T>
void launch_quantize(const void* w, int64_t ldw, void* codes, void* scales, int N, int K,
                     hipStream_t s) {
  const dim3 grid((unsigned)(kad_cdiv(N, 16) * kad_cdiv(K, 512)));
  const int KB = (int)kad_cdiv(K, 128);
  if (rows16((const T*)w, ldw))
    hipLaunchKernelGGL((quantize_weight_kernel<T, true>), grid, dim3(256), 0, s, (const T*)w, ldw,
                       (uint8_t*)codes, (uint8_t*)scales, N, K, KB);
  else
    hipLaunchKernelGGL((quantize_weight_kernel<T, false>), grid, dim3(256), 0, s, (const T*)w, ldw,
                       (uint8_t*)codes, (uint8_t*)scales, N, K, KB);
}

template <typename T>
void launch_dequantize(const void* codes, const void* scales, void* out, int64_t ldo, int N, int K,
                       hipStream_t s) {
  const dim3 grid((unsigned)(kad_cdiv(N, 16) * kad_cdiv(K, 512)));
  const int KB = (int)kad_cdiv(K, 128);
  if (rows16((const T*)out, ldo))
    hipLaunchKernelGGL((dequantize_weight_kernel<T, true>), grid, dim3(256), 0, s,
                       (const uint8_t*)codes, (const uint8_t*)scales, (T*)out, ldo, N, K, KB);
  else
    hipLaunchKernelGGL((dequantize_weight_kernel<T, false>), grid, dim3(256), 0, s,
                       (const uint8_t*)codes, (const uint8_t*)scales, (T*)out, ldo, N, K, KB);
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
