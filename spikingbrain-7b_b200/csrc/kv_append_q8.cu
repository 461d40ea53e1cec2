// Writing the 8-bit K/V cache and reading it back: the quantising append (with the rotary embedding folded in on request)
// and the gather of a window as dense tensors. Formats and rounding: kv_q8.cuh.
//
// A row is the unit of work throughout: D values of one token and head, held by neighbouring lanes, so that its largest
// magnitude takes a few shuffles and no row knows of another.
//   rotation (NeoX form, the halves of the first rot_dim values turn together), in fp32 with every product and sum
//   rounded once to fp32 and no rounding to the input type before the quantisation:
//     x'[i] = x[i] cos[i] - x[i+h] sin[i],   x'[i+h] = x[i+h] cos[i] + x[i] sin[i],   h = rot_dim / 2
//   HBM-bound in prompts (reads T * (2 kvh + H) * D elements, writes the rotated queries and 2 kvh (D + 1) bytes a token),
//   latency-bound in decode steps.
#include "kv_q8.cuh"
#include "sbk_tcgen05.cuh"

namespace sbk {
namespace q8 {

using namespace tc5;                  // packed fp32 pairs

template <typename T> struct Vec8;   // eight elements of a row
template <> struct Vec8<__nv_bfloat16> {
  static __device__ __forceinline__ void load(const uint8_t* p, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(uint8_t* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                              pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
};
template <> struct Vec8<float> {
  static __device__ __forceinline__ void load(const uint8_t* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  static __device__ __forceinline__ void store(uint8_t* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};

struct AppendParams {
  uint8_t* query; int H; int64_t q_token_stride;              // rotated in place, or NULL
  uint8_t* key; const uint8_t* value; int64_t kv_token_stride; int key_in_place;
  uint8_t* k_cache; uint8_t* v_cache; int64_t cache_block_stride;
  uint8_t* k_scale; uint8_t* v_scale; int64_t scale_block_stride;
  const int64_t* slot_mapping; int64_t num_slots; int block_size;
  const int64_t* positions; const uint8_t* cos_sin; int64_t max_position; int rot_dim;
  int T, kvh;
  uint32_t n_rows;                                            // T * (2 kvh + H)
  int32_t* block_tables; int max_blocks; const int32_t* seq_lens; const int32_t* query_start_loc;
  int B, window_left; int32_t* retired_out; int max_retired; int32_t* status;
};

constexpr int kAppendThreads = 128;

// V = D / 8 vectors per row, V / 2 lanes, two vectors each: a rotated pair (j, j + half) lies in one lane, so the rotation needs
// no exchange and its cosines are read once for both. Rows of a token: kvh of K, kvh of V, H of the query. CTAs past the
// last row retire blocks. Bound by the latency of position -> cosines and slot -> cache (a third of the DRAM
// rate; the issue slots are 72 % busy), so by the rows in flight: twelve CTAs of 128 threads per SM. Measured on 8192 tokens,
// 28 + 4 heads of 128 (142 MB, 22 us at the copy rate): 29 us; 31 us at the 47 registers the compiler takes when it may; 58 us
// with one vector per lane and the partner's values by shuffles; 48 us with four query heads per lane group (fewer address
// and table reads, a quarter of the threads).
template <typename T, int V, bool ROPE>
__global__ void __launch_bounds__(kAppendThreads, 12) kv_append_q8_kernel(const AppendParams p, int row_ctas) {
  constexpr int D = 8 * V, LPR = V / 2, kRows = kAppendThreads / LPR, ES = (int)sizeof(T);
  if ((int)blockIdx.x >= row_ctas) {
    retire_rows(((int)blockIdx.x - row_ctas) * kAppendThreads + threadIdx.x, p.block_tables, p.max_blocks, p.seq_lens,
                p.query_start_loc, p.B, p.window_left, p.block_size, p.retired_out, p.max_retired, p.status);
    return;
  }
  const int l = threadIdx.x % LPR;
  const uint32_t row = blockIdx.x * kRows + threadIdx.x / LPR, per_tok = 2 * p.kvh + (ROPE ? p.H : 0);
  const bool live = row < p.n_rows;
  const int t = live ? (int)(row / per_tok) : 0;
  const int r = live ? (int)(row - (uint32_t)t * per_tok) : 0;
  const bool is_k = r < p.kvh, is_v = !is_k && r < 2 * p.kvh, is_q = ROPE && !is_k && !is_v;
  const int head = is_k ? r : (is_v ? r - p.kvh : r - 2 * p.kvh);
  uint8_t* src = is_k ? p.key : (is_v ? const_cast<uint8_t*>(p.value) : p.query);
  src += (int64_t)t * (is_q ? p.q_token_stride : p.kv_token_stride) + (int64_t)head * D * ES;
  // this lane's vectors: the halves of a rotated pair, or two neighbours beyond the rotated part
  const int hv = ROPE ? p.rot_dim >> 4 : 0;
  const bool inside = l < hv;
  const int va = inside ? l : 2 * l, vb = inside ? l + hv : va + 1;
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
  if (live) {                                    // (on their way while the slot and the position are read)
    Vec8<T>::load(src + 8 * va * ES, a);
    Vec8<T>::load(src + 8 * vb * ES, b);
  }
  // whether (and where) the row goes into the cache
  int64_t slot = live && !is_q ? p.slot_mapping[t] : -1;
  bool skip = !live;
  int64_t pos = 0;
  if (ROPE && live) {
    pos = p.positions[t];
    if (pos < 0 || pos >= p.max_position) {      // nothing of this token is written
      if (r == 0 && l == 0) raise_status(p.status, SBK_ST_BAD_POSITION);
      skip = true;
    }
  }
  if (!skip && slot >= p.num_slots) {
    if (r == 0 && l == 0) raise_status(p.status, SBK_ST_BAD_SLOT);
    slot = -1;
  }
  const bool turn = ROPE && !is_v;
  const bool work = !skip && (turn || slot >= 0);
  if (work && turn) {
    if (inside) {
      float c[8], s[8];
      const uint8_t* tab = p.cos_sin + (pos * p.rot_dim + 8 * l) * ES;
      Vec8<T>::load(tab, c);
      Vec8<T>::load(tab + (p.rot_dim >> 1) * ES, s);
      // products and sums of two values at a time, each rounded once as ever
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const f32x2 x = pack2(a[i], a[i + 1]), y = pack2(b[i], b[i + 1]), cc = pack2(c[i], c[i + 1]), ss = pack2(s[i], s[i + 1]);
        unpack2(ffma2(fmul2(y, ss), pack2(-1.f, -1.f), fmul2(x, cc)), a[i], a[i + 1]);
        unpack2(fadd2(fmul2(y, cc), fmul2(x, ss)), b[i], b[i + 1]);
      }
    }
    if (is_q || p.key_in_place) {
      Vec8<T>::store(src + 8 * va * ES, a);
      Vec8<T>::store(src + 8 * vb * ES, b);
    }
  }
  if (__all_sync(0xffffffffu, slot < 0 || skip)) return;       // a warp of query rows ends here
  // ---- the row's exponent: largest finite magnitude over its lanes ----
  float top = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    odd |= !finite(a[i]) || !finite(b[i]);
    top = fmaxf(top, fmaxf(finite(a[i]) ? fabsf(a[i]) : 0.f, finite(b[i]) ? fabsf(b[i]) : 0.f));
  }
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (skip || slot < 0) return;
  const int e = row_exponent(top);
  const float inv = pow2i(-e);
#pragma unroll
  for (int i = 0; i < 8; ++i) { a[i] *= inv; b[i] *= inv; }
  if (odd) {                                                    // infinities become NaN like NaN itself
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = finite(a[i]) ? a[i] : __uint_as_float(0x7fffffffu);
      b[i] = finite(b[i]) ? b[i] : __uint_as_float(0x7fffffffu);
    }
  }
  auto codes = [](const float (&x)[8]) {
    return make_uint2(pack_e4m3x2(x[0], x[1]) | (pack_e4m3x2(x[2], x[3]) << 16),
                      pack_e4m3x2(x[4], x[5]) | (pack_e4m3x2(x[6], x[7]) << 16));
  };
  const int64_t blk = slot <= 0x7fffffff ? (int64_t)((uint32_t)slot / (uint32_t)p.block_size) : slot / p.block_size;
  const int off = (int)(slot - blk * p.block_size);
  uint8_t* dst = (is_k ? p.k_cache : p.v_cache) + blk * p.cache_block_stride + ((int64_t)off * p.kvh + head) * D;
  *reinterpret_cast<uint2*>(dst + 8 * va) = codes(a);
  *reinterpret_cast<uint2*>(dst + 8 * vb) = codes(b);
  if (l == 0) ((is_k ? p.k_scale : p.v_scale) + blk * p.scale_block_stride)[(int64_t)head * p.block_size + off] = (uint8_t)(e + 127);
}

// Dense read-back of the visible window: out[b, h, i, :] = value of token t0 + i, head h. D / 8 lanes per row.
template <typename TO, int LPR>
__global__ void __launch_bounds__(256)
kv_gather_q8_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache,
                    const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                    const int32_t* __restrict__ block_tables, int max_blocks, const int32_t* __restrict__ seq_lens,
                    int kvh, int64_t num_blocks, int block_size, int64_t cache_block_stride, int64_t scale_block_stride,
                    int window_left, uint8_t* __restrict__ k_out, uint8_t* __restrict__ v_out, int n_out,
                    int32_t* status) {
  constexpr int D = 8 * LPR;
  const int b = blockIdx.y;
  const int L = seq_lens[b];
  const int t0 = first_visible(L, 1, window_left);
  const int n_vis = L - t0;
  const int l = threadIdx.x % LPR;
  const int32_t* row = block_tables + (int64_t)b * max_blocks;
  const int64_t n_rows = (int64_t)kvh * n_out;
  for (int64_t i0 = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR; i0 < n_rows; i0 += (int64_t)gridDim.x * (256 / LPR)) {
    const int h = (int)(i0 / n_out);
    const int i = (int)(i0 - (int64_t)h * n_out);
    float kx[8], vx[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) kx[j] = vx[j] = 0.f;
    if (i < n_vis) {
      const int t = t0 + i;
      const int lb = t / block_size;
      const int32_t pb = lb < max_blocks ? row[lb] : -1;
      if (pb < 0 || pb >= num_blocks) {
        if (l == 0) raise_status(status, SBK_ST_BAD_BLOCK);
      } else {
        const int off = t - lb * block_size;
        const int64_t at = (int64_t)pb * cache_block_stride + ((int64_t)off * kvh + h) * D + 8 * l;
        const int64_t sa = (int64_t)pb * scale_block_stride + (int64_t)h * block_size + off;
        const uint2 kw = *reinterpret_cast<const uint2*>(k_cache + at), vw = *reinterpret_cast<const uint2*>(v_cache + at);
        const float ks = byte_scale(k_scale[sa]), vs = byte_scale(v_scale[sa]);
        const uint32_t ku[2] = {kw.x, kw.y}, vu[2] = {vw.x, vw.y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 kf = e4m3x2_to_float2(ku[j >> 1] >> (16 * (j & 1)));
          const float2 vf = e4m3x2_to_float2(vu[j >> 1] >> (16 * (j & 1)));
          kx[2 * j] = kf.x * ks; kx[2 * j + 1] = kf.y * ks;
          vx[2 * j] = vf.x * vs; vx[2 * j + 1] = vf.y * vs;
        }
      }
    }
    const int64_t o = (((int64_t)b * n_rows + i0) * D + 8 * l) * (int)sizeof(TO);
    Vec8<TO>::store(k_out + o, kx);
    Vec8<TO>::store(v_out + o, vx);
  }
}

static int check_geometry(const char* who, int kvh, int D, int64_t num_blocks, int block_size, const void* k_cache,
                          const void* v_cache, const void* k_scale, const void* v_scale, int64_t cache_block_stride,
                          int64_t scale_block_stride) {
  if (kvh <= 0 || num_blocks < 0 || !(D == 64 || D == 128 || D == 256)) {
    set_error("%s: bad sizes kvh=%d D=%d num_blocks=%lld (need D of 64, 128 or 256)", who, kvh, D, (long long)num_blocks);
    return SBK_E_ARG;
  }
  if (block_size <= 0 || block_size % 16 != 0) {
    set_error("%s: block_size=%d must be a positive multiple of 16", who, block_size);
    return SBK_E_ARG;
  }
  if (!k_cache || !v_cache || !k_scale || !v_scale) {
    set_error("%s: null cache or scale pointer", who);
    return SBK_E_ARG;
  }
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scale) || !aligned16(v_scale) || cache_block_stride % 16 ||
      scale_block_stride % 16) {
    set_error("%s: cache and scale pointers and their block strides must be multiples of 16 bytes", who);
    return SBK_E_ALIGN;
  }
  if (cache_block_stride < (int64_t)kvh * D * block_size || scale_block_stride < (int64_t)kvh * block_size) {
    set_error("%s: a block stride is smaller than the block it spans", who);
    return SBK_E_ARG;
  }
  return SBK_OK;
}

static int append(const char* who, AppendParams& p, int dtype, int D, int64_t num_blocks, bool rope, cudaStream_t st) {
  if (p.T < 0 || p.B < 0 || p.H < 0) {
    set_error("%s: negative size T=%d B=%d H=%d", who, p.T, p.B, p.H);
    return SBK_E_ARG;
  }
  if (dtype != SBK_BF16 && dtype != SBK_F32) {
    set_error("%s: dtype=%d unsupported", who, dtype);
    return SBK_E_ARG;
  }
  const int es = dtype == SBK_BF16 ? 2 : 4;
  if (p.T > 0) {
    const int rc = check_geometry(who, p.kvh, D, num_blocks, p.block_size, p.k_cache, p.v_cache, p.k_scale, p.v_scale,
                                  p.cache_block_stride, p.scale_block_stride);
    if (rc != SBK_OK) return rc;
    if (!p.key || !p.value || !p.slot_mapping) {
      set_error("%s: null pointer with T=%d", who, p.T);
      return SBK_E_ARG;
    }
    if (!aligned16(p.key) || !aligned16(p.value) || p.kv_token_stride % 16) {
      set_error("%s: key / value and their token stride must be multiples of 16 bytes", who);
      return SBK_E_ALIGN;
    }
    if (p.kv_token_stride < (int64_t)p.kvh * D * es) {
      set_error("%s: token stride smaller than the row it spans", who);
      return SBK_E_ARG;
    }
  }
  if (rope && p.T > 0) {
    if (!p.positions || !p.cos_sin || p.max_position <= 0 || p.rot_dim <= 0 || p.rot_dim > D || p.rot_dim % 16) {
      set_error("%s: needs positions and a cos/sin table with rot_dim a multiple of 16, at most D (got %d)", who, p.rot_dim);
      return SBK_E_ARG;
    }
    if (!aligned16(p.cos_sin) || (p.query && (!aligned16(p.query) || p.q_token_stride % 16))) {
      set_error("%s: the cos/sin table, query and its token stride must be multiples of 16 bytes", who);
      return SBK_E_ALIGN;
    }
    if (p.query && (p.H <= 0 || p.q_token_stride < (int64_t)p.H * D * es)) {
      set_error("%s: query needs H > 0 and a token stride that spans its heads", who);
      return SBK_E_ARG;
    }
  }
  if (!p.query) p.H = 0;
  const bool retire = p.block_tables != nullptr && p.B > 0;
  if (retire && (!p.seq_lens || p.max_blocks <= 0 || p.block_size <= 0 || (p.retired_out && p.max_retired <= 0))) {
    set_error("%s: retirement needs seq_lens, max_blocks > 0 and max_retired > 0", who);
    return SBK_E_ARG;
  }
  const int64_t n_rows = p.T > 0 ? (int64_t)p.T * (2 * p.kvh + (rope ? p.H : 0)) : 0;
  if (n_rows > 2147483647LL) {
    set_error("%s: %lld rows in one call, at most 2^31 - 1", who, (long long)n_rows);
    return SBK_E_ARG;
  }
  p.n_rows = (uint32_t)n_rows;
  const int per_cta = p.T > 0 ? kAppendThreads / (D / 16) : 1;
  const int64_t row_ctas = (n_rows + per_cta - 1) / per_cta;
  const int64_t grid = row_ctas + (retire ? (p.B + kAppendThreads - 1) / kAppendThreads : 0);
  if (!retire) p.block_tables = nullptr;
  if (grid == 0) return SBK_OK;
#define SBK_LAUNCH_APPEND(TT, V)                                                                               \
  do {                                                                                                         \
    if (rope) kv_append_q8_kernel<TT, V, true><<<(unsigned)grid, kAppendThreads, 0, st>>>(p, (int)row_ctas);  \
    else kv_append_q8_kernel<TT, V, false><<<(unsigned)grid, kAppendThreads, 0, st>>>(p, (int)row_ctas);      \
  } while (0)
#define SBK_APPEND_D(TT)                              \
  switch (D) {                                        \
    case 64: SBK_LAUNCH_APPEND(TT, 8); break;         \
    case 256: SBK_LAUNCH_APPEND(TT, 32); break;       \
    default: SBK_LAUNCH_APPEND(TT, 16); break;        \
  }
  if (dtype == SBK_BF16) { SBK_APPEND_D(__nv_bfloat16) } else { SBK_APPEND_D(float) }
#undef SBK_APPEND_D
#undef SBK_LAUNCH_APPEND
  return check_launch(who);
}

}  // namespace q8
}  // namespace sbk

extern "C" int sbk_kv_append_q8(const void* key, const void* value, int dtype, void* k_cache, void* v_cache,
                                void* k_scale, void* v_scale, const int64_t* slot_mapping, int T, int kvh, int D,
                                int64_t kv_token_stride_bytes, int64_t num_blocks, int block_size,
                                int64_t cache_block_stride_bytes, int64_t scale_block_stride_bytes,
                                int32_t* block_tables, int max_blocks, const int32_t* seq_lens,
                                const int32_t* query_start_loc, int B, int window_left, int32_t* retired_out,
                                int max_retired, int32_t* status, void* stream) {
  using namespace sbk::q8;
  AppendParams p = {};
  p.key = (uint8_t*)const_cast<void*>(key); p.value = (const uint8_t*)value; p.kv_token_stride = kv_token_stride_bytes;
  p.k_cache = (uint8_t*)k_cache; p.v_cache = (uint8_t*)v_cache; p.cache_block_stride = cache_block_stride_bytes;
  p.k_scale = (uint8_t*)k_scale; p.v_scale = (uint8_t*)v_scale; p.scale_block_stride = scale_block_stride_bytes;
  p.slot_mapping = slot_mapping; p.num_slots = num_blocks * block_size; p.block_size = block_size;
  p.T = T; p.kvh = kvh;
  p.block_tables = block_tables; p.max_blocks = max_blocks; p.seq_lens = seq_lens; p.query_start_loc = query_start_loc;
  p.B = B; p.window_left = window_left; p.retired_out = retired_out; p.max_retired = max_retired; p.status = status;
  return append("sbk_kv_append_q8", p, dtype, D, num_blocks, false, (cudaStream_t)stream);
}

extern "C" int sbk_rope_kv_append_q8(void* query, int H, int64_t q_token_stride_bytes, void* key, const void* value,
                                     int key_in_place, int dtype, void* k_cache, void* v_cache, void* k_scale,
                                     void* v_scale, const int64_t* slot_mapping, const int64_t* positions,
                                     const void* cos_sin_cache, int rot_dim, int64_t max_position, int T, int kvh, int D,
                                     int64_t kv_token_stride_bytes, int64_t num_blocks, int block_size,
                                     int64_t cache_block_stride_bytes, int64_t scale_block_stride_bytes,
                                     int32_t* block_tables, int max_blocks, const int32_t* seq_lens,
                                     const int32_t* query_start_loc, int B, int window_left, int32_t* retired_out,
                                     int max_retired, int32_t* status, void* stream) {
  using namespace sbk::q8;
  AppendParams p = {};
  p.query = (uint8_t*)query; p.H = H; p.q_token_stride = q_token_stride_bytes;
  p.key = (uint8_t*)key; p.value = (const uint8_t*)value; p.kv_token_stride = kv_token_stride_bytes;
  p.key_in_place = key_in_place;
  p.k_cache = (uint8_t*)k_cache; p.v_cache = (uint8_t*)v_cache; p.cache_block_stride = cache_block_stride_bytes;
  p.k_scale = (uint8_t*)k_scale; p.v_scale = (uint8_t*)v_scale; p.scale_block_stride = scale_block_stride_bytes;
  p.slot_mapping = slot_mapping; p.num_slots = num_blocks * block_size; p.block_size = block_size;
  p.positions = positions; p.cos_sin = (const uint8_t*)cos_sin_cache; p.max_position = max_position; p.rot_dim = rot_dim;
  p.T = T; p.kvh = kvh;
  p.block_tables = block_tables; p.max_blocks = max_blocks; p.seq_lens = seq_lens; p.query_start_loc = query_start_loc;
  p.B = B; p.window_left = window_left; p.retired_out = retired_out; p.max_retired = max_retired; p.status = status;
  return append("sbk_rope_kv_append_q8", p, dtype, D, num_blocks, true, (cudaStream_t)stream);
}

extern "C" int sbk_kv_gather_q8(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                                const int32_t* block_tables, int max_blocks, const int32_t* seq_lens, int B, int kvh,
                                int D, int64_t num_blocks, int block_size, int64_t cache_block_stride_bytes,
                                int64_t scale_block_stride_bytes, int window_left, void* k_out, void* v_out,
                                int out_dtype, int n_out, int32_t* status, void* stream) {
  using namespace sbk;
  using namespace sbk::q8;
  if (B < 0 || n_out < 0 || max_blocks <= 0) {
    set_error("sbk_kv_gather_q8: bad sizes B=%d n_out=%d max_blocks=%d", B, n_out, max_blocks);
    return SBK_E_ARG;
  }
  if (out_dtype != SBK_BF16 && out_dtype != SBK_F32) {
    set_error("sbk_kv_gather_q8: out_dtype=%d unsupported", out_dtype);
    return SBK_E_ARG;
  }
  if (B == 0 || n_out == 0) return SBK_OK;
  const int rc = check_geometry("sbk_kv_gather_q8", kvh, D, num_blocks, block_size, k_cache, v_cache, k_scale, v_scale,
                                cache_block_stride_bytes, scale_block_stride_bytes);
  if (rc != SBK_OK) return rc;
  if (!block_tables || !seq_lens || !k_out || !v_out) {
    set_error("sbk_kv_gather_q8: null pointer");
    return SBK_E_ARG;
  }
  if (!aligned16(k_out) || !aligned16(v_out)) {
    set_error("sbk_kv_gather_q8: outputs must be 16-byte aligned");
    return SBK_E_ALIGN;
  }
  if (B > 65535) {
    set_error("sbk_kv_gather_q8: B=%d exceeds 65535", B);
    return SBK_E_ARG;
  }
  const int per_cta = 256 / (D / 8);
  const int64_t ctas = ((int64_t)kvh * n_out + per_cta - 1) / per_cta;
  const dim3 grid((unsigned)(ctas < 4096 ? ctas : 4096), B);
#define SBK_LAUNCH_GATHER(TT, LPR)                                                                                  \
  kv_gather_q8_kernel<TT, LPR><<<grid, 256, 0, (cudaStream_t)stream>>>(                                             \
      (const uint8_t*)k_cache, (const uint8_t*)v_cache, (const uint8_t*)k_scale, (const uint8_t*)v_scale,           \
      block_tables, max_blocks, seq_lens, kvh, num_blocks, block_size, cache_block_stride_bytes,                    \
      scale_block_stride_bytes, window_left, (uint8_t*)k_out, (uint8_t*)v_out, n_out, status)
#define SBK_GATHER_D(TT)                         \
  switch (D) {                                   \
    case 64: SBK_LAUNCH_GATHER(TT, 8); break;    \
    case 256: SBK_LAUNCH_GATHER(TT, 32); break;  \
    default: SBK_LAUNCH_GATHER(TT, 16); break;   \
  }
  if (out_dtype == SBK_BF16) { SBK_GATHER_D(__nv_bfloat16) } else { SBK_GATHER_D(float) }
#undef SBK_GATHER_D
#undef SBK_LAUNCH_GATHER
  return check_launch("sbk_kv_gather_q8");
}
