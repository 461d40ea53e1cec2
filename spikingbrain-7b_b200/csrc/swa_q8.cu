// Sliding-window attention over the 8-bit paged K/V cache (format: kv_q8.cuh), one query token per sequence or runs of
// them:
//     s_j = scale * 2^ek_j * sum_d q_d ck_jd        o = sum_j softmax(s)_j * 2^ev_j * cv_jd        lse = log sum_j exp(s_j)
// over the visible tokens j of the query's sequence, ck / cv being the codes and ek / ev the exponents of a row.
//
// One CTA per (query token, kv head), on the CUDA cores in fp32: 128 keys at a time, a thread per key for the scores and a
// thread per dim for the sums, with a running maximum and sum per query head.
#include "kv_q8.cuh"

namespace sbk {
namespace attn_q8 {

constexpr int kD = 128, kTile = 128, kMaxG = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kNegBig = -1.0e30f;

struct Params {
  const __nv_bfloat16* q; int64_t q_stride;
  const uint8_t* k_cache; const uint8_t* v_cache; const uint8_t* k_scale; const uint8_t* v_scale;
  int64_t cache_block_stride, scale_block_stride;
  const int32_t* block_tables; int max_blocks;
  const int32_t* seq_lens;                                    // decode
  const int32_t* query_start_loc; const int32_t* context_lens; // runs
  int n_seqs, H, kvh; int64_t num_blocks; int block_size, window_left; float scale_log2;
  void* out; int64_t out_stride; float* lse_out; int32_t* status;
};

template <typename TO> __device__ __forceinline__ void put(TO* p, float x);
template <> __device__ __forceinline__ void put<float>(float* p, float x) { *p = x; }
template <> __device__ __forceinline__ void put<__nv_bfloat16>(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// grid (queries of a sequence, kv heads, sequences)
template <typename TO>
__global__ void __launch_bounds__(kTile) attend_kernel(const Params P) {
  __shared__ float q_s[kMaxG][kD];
  __shared__ float p_s[kMaxG][kTile];
  __shared__ int64_t row_s[kTile];       // byte offset of a key's row in the caches, or -1
  __shared__ float vs_s[kTile];
  __shared__ float red[kMaxG][4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = blockIdx.y, s = blockIdx.z, G = P.H / P.kvh;
  int64_t row;
  int hi;                                 // keys before hi are visible
  if (P.seq_lens) {
    row = s;
    hi = P.seq_lens[s];
  } else {
    const int a = P.query_start_loc[s], n = P.query_start_loc[s + 1] - a;
    if ((int)blockIdx.x >= n) return;
    row = a + blockIdx.x;
    hi = P.context_lens[s] + (int)blockIdx.x + 1;
  }
  const int lo = first_visible(hi, 1, P.window_left);
  for (int i = tid; i < G * kD; i += kTile)
    q_s[i / kD][i % kD] = __bfloat162float(P.q[row * P.q_stride + (int64_t)hk * G * kD + i]);
  float m[kMaxG], l[kMaxG], o[kMaxG];
#pragma unroll
  for (int g = 0; g < kMaxG; ++g) { m[g] = -INFINITY; l[g] = 0.f; o[g] = 0.f; }
  for (int j0 = lo; j0 < hi; j0 += kTile) {
    const int j = j0 + tid;
    int64_t at = -1;
    float ks = 0.f, vs = 0.f;
    if (j < hi) {
      const int lb = j / P.block_size, off = j - lb * P.block_size;
      const int32_t pb = lb < P.max_blocks ? P.block_tables[(int64_t)s * P.max_blocks + lb] : -1;
      if (pb < 0 || pb >= P.num_blocks) {
        raise_status(P.status, SBK_ST_BAD_BLOCK);
      } else {
        at = (int64_t)pb * P.cache_block_stride + ((int64_t)off * P.kvh + hk) * kD;
        const int64_t sa = (int64_t)pb * P.scale_block_stride + (int64_t)hk * P.block_size + off;
        ks = q8::byte_scale(P.k_scale[sa]);
        vs = q8::byte_scale(P.v_scale[sa]);
      }
    }
    __syncthreads();                      // the tile before has been read
    row_s[tid] = at;
    vs_s[tid] = vs;
    __syncthreads();
    float sc[kMaxG];
#pragma unroll
    for (int g = 0; g < kMaxG; ++g) sc[g] = 0.f;
    if (at >= 0) {
      for (int d = 0; d < kD; d += 2) {
        const float2 k2 = q8::e4m3x2_to_float2(*reinterpret_cast<const uint16_t*>(P.k_cache + at + d));
#pragma unroll
        for (int g = 0; g < kMaxG; ++g)
          if (g < G) sc[g] += q_s[g][d] * k2.x + q_s[g][d + 1] * k2.y;
      }
    }
#pragma unroll
    for (int g = 0; g < kMaxG; ++g) {
      sc[g] = at >= 0 ? sc[g] * (ks * P.scale_log2) : -INFINITY;
      float top = sc[g];
      for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      if (lane == 0) red[g][warp] = top;
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < kMaxG; ++g) {
      const float mn = fmaxf(m[g], fmaxf(fmaxf(red[g][0], red[g][1]), fmaxf(red[g][2], red[g][3])));
      const float ms = fmaxf(mn, kNegBig), alpha = exp2f(m[g] - ms);
      m[g] = mn;
      l[g] *= alpha;
      o[g] *= alpha;
      p_s[g][tid] = at >= 0 ? exp2f(sc[g] - ms) : 0.f;
    }
    __syncthreads();
    for (int i = 0; i < kTile; ++i) {
      if (row_s[i] < 0) continue;
      const float v = q8::e4m3x2_to_float2(P.v_cache[row_s[i] + tid]).x * vs_s[i];
#pragma unroll
      for (int g = 0; g < kMaxG; ++g) {
        if (g >= G) break;
        l[g] += p_s[g][i];
        o[g] += p_s[g][i] * v;
      }
    }
  }
#pragma unroll
  for (int g = 0; g < kMaxG; ++g) {
    if (g >= G) break;
    const int h = hk * G + g;
    put<TO>(reinterpret_cast<TO*>(P.out) + row * P.out_stride + (int64_t)h * kD + tid, l[g] != 0.f ? o[g] / l[g] : 0.f);
    if (P.lse_out && tid == 0) P.lse_out[row * P.H + h] = l[g] != 0.f ? (m[g] + log2f(l[g])) * kLn2 : -INFINITY;
  }
}

static int check(const char* who, const Params& P, int D, int n_q, int out_dtype) {
  if (P.n_seqs < 0 || n_q < 0 || P.H <= 0 || P.kvh <= 0 || P.H % P.kvh != 0 || P.max_blocks <= 0 || P.num_blocks < 0) {
    set_error("%s: bad sizes n=%d H=%d kvh=%d max_blocks=%d", who, P.n_seqs, P.H, P.kvh, P.max_blocks);
    return SBK_E_ARG;
  }
  if (D != kD || P.H / P.kvh > kMaxG || !(P.kvh == 1 || P.kvh == 2 || P.kvh == 4)) {
    set_error("%s: unsupported shape D=%d H/kvh=%d kvh=%d (need D=128, group<=8, kvh in 1,2,4)", who, D, P.H / P.kvh, P.kvh);
    return SBK_E_ARG;
  }
  if (P.block_size <= 0 || P.block_size % 16 != 0) {
    set_error("%s: block_size=%d must be a positive multiple of 16", who, P.block_size);
    return SBK_E_ARG;
  }
  if (out_dtype != SBK_BF16 && out_dtype != SBK_F32) {
    set_error("%s: out_dtype=%d unsupported", who, out_dtype);
    return SBK_E_ARG;
  }
  if (P.n_seqs == 0 || n_q == 0) return SBK_OK;
  if (!P.q || !P.k_cache || !P.v_cache || !P.k_scale || !P.v_scale || !P.block_tables || !P.out) {
    set_error("%s: null pointer", who);
    return SBK_E_ARG;
  }
  if (!aligned16(P.k_cache) || !aligned16(P.v_cache) || !aligned16(P.k_scale) || !aligned16(P.v_scale) ||
      P.cache_block_stride % 16 || P.scale_block_stride % 16 || (reinterpret_cast<uintptr_t>(P.q) & 3u) || (P.q_stride & 1)) {
    set_error("%s: caches, scales and their block strides must be 16-byte multiples and q 4-byte aligned", who);
    return SBK_E_ALIGN;
  }
  if (P.cache_block_stride < (int64_t)P.kvh * D * P.block_size || P.scale_block_stride < (int64_t)P.kvh * P.block_size) {
    set_error("%s: a block stride is smaller than the block it spans", who);
    return SBK_E_ARG;
  }
  return SBK_OK;
}

}  // namespace attn_q8
}  // namespace sbk

extern "C" int sbk_swa_prefill_q8(const void* q, int64_t q_tok_stride, const void* k_cache, const void* v_cache,
                                  const void* k_scale, const void* v_scale, const int32_t* block_tables, int max_blocks,
                                  const int32_t* query_start_loc, const int32_t* context_lens, int n_seqs,
                                  int max_query_len, int H, int kvh, int D, int64_t num_blocks, int block_size,
                                  int64_t cache_block_stride_bytes, int64_t scale_block_stride_bytes, int window_left,
                                  float scale, void* out, int64_t out_tok_stride, int32_t* status, void* stream) {
  using namespace sbk;
  using namespace sbk::attn_q8;
  Params P = {};
  P.q = (const __nv_bfloat16*)q; P.q_stride = q_tok_stride;
  P.k_cache = (const uint8_t*)k_cache; P.v_cache = (const uint8_t*)v_cache; P.k_scale = (const uint8_t*)k_scale;
  P.v_scale = (const uint8_t*)v_scale; P.cache_block_stride = cache_block_stride_bytes;
  P.scale_block_stride = scale_block_stride_bytes; P.block_tables = block_tables; P.max_blocks = max_blocks;
  P.query_start_loc = query_start_loc; P.context_lens = context_lens; P.n_seqs = n_seqs; P.H = H; P.kvh = kvh;
  P.num_blocks = num_blocks; P.block_size = block_size; P.window_left = window_left; P.scale_log2 = scale * kLog2e;
  P.out = out; P.out_stride = out_tok_stride; P.status = status;
  const int rc = check("sbk_swa_prefill_q8", P, D, max_query_len, SBK_BF16);
  if (rc != SBK_OK || n_seqs == 0 || max_query_len == 0) return rc;
  if (!query_start_loc || !context_lens) {
    set_error("sbk_swa_prefill_q8: null pointer");
    return SBK_E_ARG;
  }
  if (n_seqs > 65535) {
    set_error("sbk_swa_prefill_q8: n_seqs=%d exceeds 65535", n_seqs);
    return SBK_E_ARG;
  }
  attend_kernel<__nv_bfloat16><<<dim3(max_query_len, kvh, n_seqs), kTile, 0, (cudaStream_t)stream>>>(P);
  return check_launch("sbk_swa_prefill_q8");
}
