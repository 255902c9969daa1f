// The 8-bit prefix cache: pages of a batch's requests, and keys and values into them.
//
// A cache is a pool of pages.  A page holds `block` tokens of one layer:
// codes [HK, block, D] in e4m3 (OCP) and one scale per KV head in e8m0, the
// power of two 2^(byte - 127).  A token's value is code * scale.  Powers of
// two cost an e4m3 value no precision (its significand is untouched) and make
// both a change of scale and the product in the attention's scaled MFMAs
// exact.  The pool's codes are [pages, HK, block, D], so that the rows of a
// page and head are one contiguous piece.

#include "kad_common.h"

// ---------------------------------------------------------------------------
// Block tables.  Request b has `starts[b]` tokens in pages that it holds
// already and `lengths[b]` after this call; it gets
//   need[b] = ceil(lengths / block) - ceil(starts / block)
// pages, taken from `free` in request order behind the `taken` that earlier calls got:
// entry j of its row is
//   old[b][j]                                      j <  ceil(starts / block)
//   free[taken + sum of need before b + j - held]  j <  ceil(lengths / block)
//   -1                                             otherwise, or when `free` is used up.
// One workgroup a request, which adds up what the requests before it need by
// itself: B / 2 lengths on average out of L2, and no second launch or wait between
// workgroups.  Bound by latency: 3.0 us for 32 requests of 1024 tokens, 5.3 us for
// 1000 of 32768 that grow (3.1 MB).

__device__ __forceinline__ int pages_of(int tokens, int block) {
  return (int)(((int64_t)max(tokens, 0) + block - 1) / block);
}

__global__ __launch_bounds__(256) void block_tables_kernel(
    const int* __restrict__ lengths, const int* __restrict__ starts, const int* __restrict__ old,
    int old_width, const int* __restrict__ free_blocks, int num_free,
    const int* __restrict__ taken, int* __restrict__ tables, int width, int* __restrict__ used,
    int B, int block, int max_length) {
  __shared__ int64_t part[4];
  const int tid = threadIdx.x, b = blockIdx.x;
  // pages that the requests before b need (the sum can pass 32 bits, where the
  // lengths do not fit the list anyway)
  int64_t before = 0;
  for (int i = tid; i < b; i += 256) {
    const int held = starts ? pages_of(min(starts[i], max_length), block) : 0;
    before += max(pages_of(min(lengths[i], max_length), block) - held, 0);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
  if ((tid & 63) == 0) part[tid >> 6] = before;
  const int held = starts ? pages_of(min(starts[b], max_length), block) : 0;
  const int total = max(pages_of(min(lengths[b], max_length), block), held);
  __syncthreads();
  before = part[0] + part[1] + part[2] + part[3] + (taken ? max(*taken, 0) : 0);
  for (int j = tid; j < width; j += 256) {
    int page = -1;
    if (j < held) {
      if (old && j < old_width) page = old[(int64_t)b * old_width + j];
    } else if (j < total && before + (j - held) < num_free) {
      page = free_blocks[before + (j - held)];
    }
    tables[(int64_t)b * width + j] = page;
  }
  if (b == B - 1 && tid == 0)
    *used = (int)min(before + total - held, (int64_t)0x7fffffff);
}

extern "C" int kad_prefix_block_tables_ex(const int32_t* lengths, const int32_t* starts,
                                          const int32_t* old_tables, int old_width,
                                          const int32_t* free_blocks, int num_free,
                                          const int32_t* taken, int32_t* tables, int width,
                                          int32_t* used, int B, int block, int max_length,
                                          kad_stream_t stream) {
  KAD_REQUIRE(B > 0 && width > 0 && old_width >= 0 && num_free >= 0,
              "block tables need requests and columns");
  KAD_REQUIRE(block > 0 && max_length > 0 && kad_cdiv(max_length, block) <= width,
              "tables of %d columns of %d tokens do not hold %d", width, block, max_length);
  KAD_REQUIRE(lengths && tables && used && (free_blocks || num_free == 0),
              "null pointer argument");
  KAD_REQUIRE(max_length <= 1 << 30, "requests of %d tokens", max_length);
  // (each workgroup adds up the requests before its own, so the work grows with B^2)
  KAD_REQUIRE(B <= 1 << 20, "block tables of %d requests", B);
  KAD_REQUIRE(!old_tables || starts, "held tables need the tokens held");
  hipLaunchKernelGGL(block_tables_kernel, dim3((unsigned)B), dim3(256), 0, (hipStream_t)stream,
                     lengths, starts, old_tables, old_width, free_blocks, num_free, taken, tables,
                     width, used, B, block, max_length);
  return kad_launch_status("block_tables_kernel");
}

extern "C" int kad_prefix_block_tables(const int32_t* lengths, const int32_t* starts,
                                       const int32_t* old_tables, int old_width,
                                       const int32_t* free_blocks, int num_free, int32_t* tables,
                                       int width, int32_t* used, int B, int block, int max_length,
                                       kad_stream_t stream) {
  return kad_prefix_block_tables_ex(lengths, starts, old_tables, old_width, free_blocks, num_free,
                                    nullptr, tables, width, used, B, block, max_length, stream);
}

// ---------------------------------------------------------------------------
// Writing.  Token i of request b goes to position starts[b] + i while that is
// below lengths[b].  A workgroup owns one touched page of one request and
// head, so the page's scale has one writer:
//   e_need = the smallest e >= -100 with amax <= 448 * 2^e over the finite new values
//   e      = e_need, or max(e_need, the page's) when it holds earlier tokens
//   code   = e4m3(x * 2^-e), to nearest even; infinities and NaN become NaN
// and the earlier tokens' codes are rounded again when the scale has grown.  A page
// of earlier tokens whose scale is not a number (byte 255) stays one: new codes are
// NaN too.
// Rows past lengths[b] are left as they were.
constexpr int kMinExp = -100;

__device__ __forceinline__ int scale_exp(float amax) {
  // amax = 1.m * 2^x; 448 = 1.75 * 2^8
  const uint32_t bits = __float_as_uint(amax);
  const int x = (int)(bits >> 23) - 127;
  const int e = x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kMinExp);  // zeros and subnormals of fp32 give x = -127
}
__device__ __forceinline__ float pow2f(int e) {  // 2^e, -127 <= e <= 127
  return __uint_as_float(e > -127 ? (uint32_t)(e + 127) << 23 : 1u << 22);
}

struct WriteArgs {
  const void* x[2];       // k, v
  int64_t s_b[2], s_t[2], s_h[2];
  const int* tables;
  const int* lengths;
  const int* starts;
  uint8_t* codes[2];
  uint8_t* scale[2];
  int width, pages, B, N, HK, D, block, touched;
};

// 16 elements of a row as floats
__device__ __forceinline__ void load16(const bf16_t* p, float* f) {
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const u32x4 x = *(const u32x4*)(p + 8 * v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[8 * v + 2 * i] = __uint_as_float(x[i] << 16);
      f[8 * v + 2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void load16(const _Float16* p, float* f) {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const f16x8 x = *(const f16x8*)(p + 8 * v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[8 * v + i] = (float)x[i];
  }
}
__device__ __forceinline__ void load16(const float* p, float* f) {
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const f32x4 x = *(const f32x4*)(p + 4 * v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[4 * v + i] = x[i];
  }
}
__device__ __forceinline__ void store16(uint8_t* p, const float* f, float scale) {
  u32x4 c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i] * scale, f[4 * i + 1] * scale, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2] * scale, f[4 * i + 3] * scale, w, true);
    c[i] = (uint32_t)w;
  }
  *(u32x4*)p = c;
}

// A page and head is block * D / 16 pieces of 16 elements.  Each of up to 1024
// threads keeps 4 of them in registers between the maximum and the rounding, so
// the input is read once and the codes are written once, 16 bytes a lane.
// Bound by HBM: 32 requests of 1024 tokens (bf16, 2 KV heads of 256; 101 MB) in 19.4 us,
// 5.2 TB/s, and 8 of up to 20000 (fp16, 8 heads of 128; 492 MB) in 98 to 100 us, 4.9 to
// 5.0 TB/s, the rate of a large copy (5.18).  The 32 in fp32 (168 MB, part of it from the
// memory-side cache in repeated calls): 25 us.  One token for each of 256 requests: 5.7 us.
// VEC: rows of the input start at 16-byte boundaries (else element by element).
constexpr int kPieces = 4;

template <typename T, bool VEC>
__global__ __launch_bounds__(1024) void write_blocks_kernel(WriteArgs a) {
  __shared__ float part[16];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int u = blockIdx.x % a.touched, b = blockIdx.x / a.touched;
  const int h = blockIdx.y, kv = blockIdx.z;
  const int start = a.starts ? max(a.starts[b], 0) : 0;
  const int64_t stop64 = min((int64_t)start + a.N, (int64_t)a.width * a.block);
  // one past the last new position; at least 0, so that no difference below wraps
  const int stop = max(min(a.lengths[b], (int)stop64), 0);
  const int blk = start / a.block + u;
  if (blk >= a.width) return;
  const int lo = max(start - blk * a.block, 0), hi = min(stop - blk * a.block, a.block);
  if (hi <= lo) return;                               // rows [lo, hi) of the page are new
  const int page = a.tables[(int64_t)b * a.width + blk];
  if (page < 0 || page >= a.pages) return;
  const T* x = (const T*)a.x[kv] + (int64_t)b * a.s_b[kv] + (int64_t)h * a.s_h[kv] +
               ((int64_t)blk * a.block - start) * a.s_t[kv];
  uint8_t* codes = a.codes[kv] + ((int64_t)page * a.HK + h) * a.block * a.D;
  uint8_t* scale = a.scale[kv] + (int64_t)page * a.HK + h;
  const int ppr = a.D / 16;                           // pieces per row
  float f[kPieces][16];
  float amax = 0.f;
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    const int i = tid + p * threads, row = i / ppr, d = i % ppr * 16;
#pragma unroll
    for (int e = 0; e < 16; ++e) f[p][e] = 0.f;
    if (row >= lo && row < hi) {
      const T* src = x + row * a.s_t[kv] + d;
      if constexpr (VEC) {
        load16(src, f[p]);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) f[p][e] = Elem<T>::to_f(src[e]);
      }
    }
  }
  // (fmaxf leaves NaN out; an infinity, seen by one compare, is left out in a
  // second pass over the registers)
#pragma unroll
  for (int p = 0; p < kPieces; ++p)
#pragma unroll
    for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(f[p][e]));
  if (amax == INFINITY) {
    amax = 0.f;
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (fabsf(f[p][e]) < INFINITY) amax = fmaxf(amax, fabsf(f[p][e]));
  }
  amax = wave_max(amax);
  if ((tid & 63) == 0) part[tid >> 6] = amax;
  __syncthreads();
  for (int i = 0; i < threads / 64; ++i) amax = fmaxf(amax, part[i]);
  int e = scale_exp(amax);
  if (lo > 0) {
    const int before = (int)*scale - 127;             // (128: not a number)
    if (e > before) {                                 // the earlier rows to the new scale
      const float m = pow2f(max(before - e, -126));
      for (int i = tid; i < lo * ppr; i += threads) {
        const u32x4 c = *(const u32x4*)(codes + 16 * i);
        float g[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          g[4 * j] = __builtin_amdgcn_cvt_f32_fp8((int)c[j], 0);
          g[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8((int)c[j], 1);
          g[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8((int)c[j], 2);
          g[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8((int)c[j], 3);
        }
        store16(codes + 16 * i, g, m);
      }
    }
    e = max(e, before);
  }
  const float inv = e <= 127 ? pow2f(-e) : NAN;
#pragma unroll
  for (int p = 0; p < kPieces; ++p) {
    const int i = tid + p * threads, row = i / ppr;
    if (row >= lo && row < hi) store16(codes + 16 * i, f[p], inv);
  }
  __syncthreads();                                    // every thread has read the old scale
  if (tid == 0) *scale = (uint8_t)(e + 127);
}

// 4 pieces a thread, whole waves
static int write_threads(int block, int D) { return max(64, block * D / (16 * kPieces)); }

template <typename T>
static void launch_write(const WriteArgs& a, bool vec, hipStream_t stream) {
  const dim3 grid((unsigned)(a.touched * a.B), (unsigned)a.HK, 2);
  const int threads = write_threads(a.block, a.D);
  if (vec)
    hipLaunchKernelGGL((write_blocks_kernel<T, true>), grid, dim3(threads), 0, stream, a);
  else
    hipLaunchKernelGGL((write_blocks_kernel<T, false>), grid, dim3(threads), 0, stream, a);
}

extern "C" int kad_write_prefix_blocks(
    const void* k, int64_t sk_b, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_b,
    int64_t sv_t, int64_t sv_h, int dtype, const int32_t* tables, int width,
    const int32_t* lengths, const int32_t* starts, void* k_codes, void* v_codes, void* k_scale,
    void* v_scale, int pages, int B, int N, int HK, int D, int block, kad_stream_t stream) {
  KAD_REQUIRE(B > 0 && N > 0 && HK > 0 && width > 0 && pages > 0, "empty dimensions");
  KAD_REQUIRE(k && v && tables && lengths && k_codes && v_codes && k_scale && v_scale,
              "null pointer argument");
  KAD_REQUIRE(D == 64 || D == 128 || D == 256, "head dim %d is not 64, 128 or 256", D);
  KAD_REQUIRE(block == 32 || block == 64 || block == 128 || block == 256,
              "block size %d is not 32, 64, 128 or 256", block);
  WriteArgs a = {{k, v}, {sk_b, sv_b}, {sk_t, sv_t}, {sk_h, sv_h}, tables, lengths, starts,
                 {(uint8_t*)k_codes, (uint8_t*)v_codes}, {(uint8_t*)k_scale, (uint8_t*)v_scale},
                 width, pages, B, N, HK, D, block, 0};
  // N tokens reach into at most this many pages of a request
  a.touched = (int)(starts ? ((int64_t)N + block - 2) / block + 1 : kad_cdiv(N, block));
  if (a.touched > width) a.touched = width;
  // (a grid holds fewer than 2^32 work-items a dimension)
  KAD_REQUIRE((int64_t)a.touched * B < (1ll << 32) / write_threads(block, D) && HK <= 65535,
              "too many pages for a launch");
  KAD_REQUIRE((int64_t)width * block <= 1 << 30, "tables of %d columns of %d tokens", width, block);
  KAD_REQUIRE(((uintptr_t)k_codes % 16) == 0 && ((uintptr_t)v_codes % 16) == 0,
              "codes must be 16-byte aligned");
  const int item = dtype == KAD_DTYPE_F32 ? 4 : 2;
  auto rows16 = [&](const void* p, int64_t b, int64_t t, int64_t h) {
    return (uintptr_t)p % 16 == 0 && b * item % 16 == 0 && t * item % 16 == 0 &&
           h * item % 16 == 0;
  };
  const bool vec = rows16(k, sk_b, sk_t, sk_h) && rows16(v, sv_b, sv_t, sv_h);
  if (dtype == KAD_DTYPE_BF16) launch_write<bf16_t>(a, vec, (hipStream_t)stream);
  else if (dtype == KAD_DTYPE_F16) launch_write<_Float16>(a, vec, (hipStream_t)stream);
  else if (dtype == KAD_DTYPE_F32) launch_write<float>(a, vec, (hipStream_t)stream);
  else KAD_UNSUPPORTED("dtype code %d", dtype);
  return kad_launch_status("write_blocks_kernel");
}
