// Attention of beams over a request's prefix in the 8-bit cache, then over
// their own causal suffix: for a query row (beam n of request b, token t,
// head h, KV head kh = h / (H / HK))
//   s_j = scale * q . k_j   over the request's cached keys, j < lengths[b],
//                           and the beam's suffix keys j <= Tk - T + t
//   out = sum_j softmax(s)_j v_j, times sigmoid(gate) where one is given
// with k_j, v_j = code * scale of the page and KV head that holds token j.  A
// row that sees no key gives zeros.

#include "kad_common.h"

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
  int pages, width, W, T, Tk, H, HK, block;
  int64_t rows;
  float scale;
};

// One wave per query row, lane l holding D / 64 of its elements; the softmax
// runs over the keys one at a time.
template <typename T, int D>
__global__ __launch_bounds__(256) void block_attn_row_kernel(BlockAttnArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int h = (int)(row % a.H), t = (int)(row / a.H % a.T);
  const int64_t n = row / a.H / a.T;
  const int b = (int)(n / a.W), kh = h / (a.H / a.HK);
  float q[E], o[E];
  for (int i = 0; i < E; ++i) {
    q[i] = a.scale * Elem<T>::to_f(
        ((const T*)a.q)[n * a.sq_n + t * a.sq_t + h * a.sq_h + lane * E + i]);
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  auto take = [&](const float* k, const float* v) {
    float s = 0.f;
    for (int i = 0; i < E; ++i) s = fmaf(q[i], k[i], s);
    s = wave_sum(s);
    const float top = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - top), p = expf(s - top);
    for (int i = 0; i < E; ++i) o[i] = fmaf(p, v[i], o[i] * keep);
    l = l * keep + p;
    m = top;
  };
  const int len = min(a.lengths[b], a.width * a.block);
  for (int j = 0; j < len; ++j) {
    const int page = a.tables[(int64_t)b * a.width + j / a.block];
    if (page < 0 || page >= a.pages) continue;
    const int64_t ph = (int64_t)page * a.HK + kh;
    const int64_t at = (ph * a.block + j % a.block) * D + lane * E;
    const float ks = ldexpf(1.f, (int)a.ksc[ph] - 127), vs = ldexpf(1.f, (int)a.vsc[ph] - 127);
    float k[E], v[E];
    for (int i = 0; i < E; ++i) {
      k[i] = __builtin_amdgcn_cvt_f32_fp8((int)a.kc[at + i], 0) * ks;
      v[i] = __builtin_amdgcn_cvt_f32_fp8((int)a.vc[at + i], 0) * vs;
    }
    take(k, v);
  }
  for (int j = 0; j <= a.Tk - a.T + t && j < a.Tk; ++j) {
    float k[E], v[E];
    for (int i = 0; i < E; ++i) {
      const int d = lane * E + i;
      k[i] = Elem<T>::to_f(((const T*)a.sk)[n * a.ssk_n + j * a.ssk_t + kh * a.ssk_h + d]);
      v[i] = Elem<T>::to_f(((const T*)a.sv)[n * a.ssv_n + j * a.ssv_t + kh * a.ssv_h + d]);
    }
    take(k, v);
  }
  for (int i = 0; i < E; ++i) {
    float y = l > 0.f || l != l ? o[i] / l : 0.f;
    if (a.gate)
      y *= sigmoid_f(Elem<T>::to_f(
          ((const T*)a.gate)[n * a.sg_n + t * a.sg_t + h * a.sg_h + lane * E + i]));
    ((T*)a.out)[n * a.so_n + t * a.so_t + h * a.so_h + lane * E + i] = Elem<T>::from_f(y);
  }
}

template <typename T>
static void launch_rows(const BlockAttnArgs& a, int D, hipStream_t stream) {
  const dim3 grid((unsigned)kad_cdiv(a.rows, 4));
  if (D == 64) hipLaunchKernelGGL((block_attn_row_kernel<T, 64>), grid, dim3(256), 0, stream, a);
  else if (D == 128)
    hipLaunchKernelGGL((block_attn_row_kernel<T, 128>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((block_attn_row_kernel<T, 256>), grid, dim3(256), 0, stream, a);
}

extern "C" int kad_block_prefix_attention(
    const void* q, int64_t sq_n, int64_t sq_t, int64_t sq_h, const void* k_codes,
    const void* v_codes, const void* k_scale, const void* v_scale, int pages,
    const int32_t* tables, int width, const int32_t* lengths, const void* suffix_k,
    int64_t ssk_n, int64_t ssk_t, int64_t ssk_h, const void* suffix_v, int64_t ssv_n,
    int64_t ssv_t, int64_t ssv_h, const void* gate, int64_t sg_n, int64_t sg_t, int64_t sg_h,
    void* out, int64_t so_n, int64_t so_t, int64_t so_h, int B, int W, int T, int Tk, int H,
    int HK, int D, int block, int dtype, float scale, kad_stream_t stream) {
  KAD_REQUIRE(B > 0 && W > 0 && T > 0 && H > 0 && HK > 0 && width > 0 && pages > 0,
              "empty dimensions");
  KAD_REQUIRE(H % HK == 0, "%d heads over %d KV heads", H, HK);
  KAD_REQUIRE(Tk == 0 || Tk >= T, "a suffix of %d keys for %d queries", Tk, T);
  KAD_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && tables && lengths && out &&
                  (Tk == 0 || (suffix_k && suffix_v)),
              "null pointer argument");
  KAD_REQUIRE(D == 64 || D == 128 || D == 256, "head dim %d is not 64, 128 or 256", D);
  KAD_REQUIRE(block == 32 || block == 64 || block == 128 || block == 256,
              "block size %d is not 32, 64, 128 or 256", block);
  KAD_REQUIRE((int64_t)width * block <= 0x7fffffff, "tables of %d columns", width);
  BlockAttnArgs a = {q, sq_n, sq_t, sq_h, (const uint8_t*)k_codes, (const uint8_t*)v_codes,
                     (const uint8_t*)k_scale, (const uint8_t*)v_scale, tables, lengths, suffix_k,
                     ssk_n, ssk_t, ssk_h, suffix_v, ssv_n, ssv_t, ssv_h, gate, sg_n, sg_t, sg_h,
                     out, so_n, so_t, so_h, pages, width, W, T, Tk, H, HK, block,
                     (int64_t)B * W * T * H, scale};
  KAD_REQUIRE(kad_cdiv(a.rows, 4) <= 0x7fffffff, "too many rows for a launch");
  if (dtype == KAD_DTYPE_BF16) launch_rows<bf16_t>(a, D, (hipStream_t)stream);
  else if (dtype == KAD_DTYPE_F16) launch_rows<_Float16>(a, D, (hipStream_t)stream);
  else KAD_UNSUPPORTED("dtype code %d: queries are bf16 or fp16", dtype);
  return kad_launch_status("block_attn_row_kernel");
}
