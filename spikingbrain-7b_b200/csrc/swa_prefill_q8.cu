// Sliding-window attention for runs of query tokens over the 8-bit paged K/V cache (format: kv_q8.cuh), in two launches.
//
// 1. unpack: the keys that a run sees become dense bf16 rows, K and V [head][row][128], once. Every value of the cache is
//    a bf16 number, so nothing is rounded. A run's rows start at a multiple of 128 and its last 128 are filled up with
//    zeros. Each key serves (window / queries of a tile) query tiles, so expanding it in every CTA that reads it would repeat that work
//    a hundred times over in the kernel that is short of instructions; written out once it is (6 D + 2) kvh bytes a
//    token, under 2 % of the time of a long run. What must not meet a weight of zero is kept from the second step here: NaN codes of V
//    become a mark, tokens that the pool does not hold a bit of their tile, and a flag per tile says whether there are any.
// 2. attend: tcgen05, two query tiles per CTA taking turns, as in swa_prefill_tc2.cu: a CTA owns 2 x (128 / G) consecutive queries of a
//    run and one kv head as two MMA tiles A and B of 128 rows (row = query * G + head); both read the same K / V tiles in shared
//    memory; one thread owns one row, and while the warps of A work on their scores the tensor core computes for B:
//        tensor core:  S_A(0) S_B(0) | P_A(0).V S_A(1) | P_B(0).V S_B(1) | ...
//        warps 0-3  :  softmax A(0)  |                 | softmax A(1)    ...
//        warps 4-7  :                | softmax B(0)    |                 ...
//    Unlike there V is bf16 (a V row may have any exponent, which fp16 does not hold), and P goes in as a bf16 head and a bf16 remainder,
//    two products, so that it loses 2^-15 of itself (the head alone loses 2^-8, as much as the output's own rounding: mean relative
//    error 1.7e-3, over the 1e-3 that the framework's attention kernels keep). Nothing has to be converted, and a tile of
//    128 keys is one copy per 64 dims.
//    Tensor memory (512 columns): S_A / P_A [0,128), S_B / P_B [128,256), O_A [256,384), O_B [384,512). The softmax offset of a row
//    moves only when its maximum has grown by more than 2^8, so O is rescaled in tensor memory almost only on the first tile.
//    Roles (384 threads): warps 0-3 softmax / epilogue of tile A, 4-7 of tile B, 8 producer of the K ring, 9 of the V ring, 10 tensor
//    memory and MMA issue; 11 looks through the tiles' flags, and is there for its registers: the softmax warps hold a row's 128 scores
//    at once, with what the last four warps give up. Every wait is bounded.
// Measured, 28 + 4 heads of 128, window 4096, 8192 queries on 8192 cached tokens: 685 us, 704 TFLOP/s of useful products (4 H D
//    a visible pair), the tensor core at work 60 % of the time. With the heads of P alone it took 578: then a tile pair took about 4000
//    cycles per 128 keys, of which the tensor core worked 2050 (now 3070): the rest is the way from a tile's last P over the MMAs
//    still to be issued to its next scores, and the softmax (two warps per scheduler, 1900 cycles alone, 2700 when A's and B's
//    overlap). Tried and slower, with the heads alone (us, the first form of this kernel being 624): scores read twice instead of held
//    598 against 581; tiles of 64 keys with two S buffers each 711; two threads per row 592; part of the exponentials as a
//    polynomial 0 to 5 % more; P in halves 581; MMAs issued under `lane == 0` 618 against 598; a warp of its own to issue
//    each tile's MMAs 662.
#include <math.h>

#include "kv_q8.cuh"
#include "sbk_tcgen05.cuh"
#include "sbk_tma.cuh"
#include "swa_decode_q8.cuh"

namespace sbk {
namespace prefill_q8 {

using namespace tc5;

constexpr int kD = 128, kTile = 128;
constexpr int kPanelBytes = 128 * 128;           // [128 rows][128 B]: 64 bf16 of every row
constexpr int kOperandBytes = 2 * kPanelBytes;
constexpr int kStagesK = 2, kStagesV = 3;
constexpr int kQOff = 0, kKOff = 2 * kOperandBytes, kVOff = kKOff + kStagesK * kOperandBytes;
constexpr int kBarOff = kVOff + kStagesV * kOperandBytes;
constexpr int kSmemBytes = kBarOff + 256 + 1024;
constexpr int kSoftmaxWarps = 8, kThreads = 32 * (kSoftmaxWarps + 4);
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;   // registers of a thread after the block has started with 168
static_assert(32 * kSoftmaxWarps * kSoftmaxRegs + (kThreads - 32 * kSoftmaxWarps) * kOtherRegs <= kThreads * 168,
              "the registers of the warpgroups must fit what the block is launched with");
constexpr int kTmemCols = 512, kOCol = 256;
constexpr float kLog2e = 1.4426950408889634f, kNegBig = -1.0e30f;
constexpr int64_t kScratchTarget = (int64_t)1 << 28;   // 256 MiB of dense rows at a time, or one sequence's where that is more

struct Params {
  const __nv_bfloat16* q; int64_t q_tok_stride;
  const int32_t* query_start_loc; const int32_t* context_lens;
  int seq0;               // first sequence of this launch; its dense rows start at row 0
  int rows_per_seq;       // dense rows of a sequence, a multiple of 128
  int64_t width;          // tokens that a row of the block table has entries for
  int pairs;              // query tile pairs per sequence
  int pairs_per_head;     // of the sequences of this launch
  int split;              // pairs from here on are two CTAs' (of all heads, laid end to end)
  int max_query_len, H, G, bq, window_left; float scale_log2;   // >= 0: a negative scale's sign goes into q
  uint32_t q_sign;
  const uint16_t* v_rows; int64_t rows_total;    // the dense V rows, for what the tensor core must not see
  const uint4* gone; const uint32_t* tile_flags; // of every head and tile [kvh][rows_total / 128]: rows that the pool does not hold, flags
  __nv_bfloat16* out; int64_t out_tok_stride; int32_t* status;
};

// what a sequence's run sees: keys [first, first + n) of its token axis, of which the block table has entries for `there`
struct Keys { int first, n, there, n_q; };
__device__ __forceinline__ Keys keys_of(const int32_t* qsl, const int32_t* ctx_lens, int s, int window_left, int max_query_len,
                                        int64_t width) {
  Keys k;
  k.n_q = qsl[s + 1] - qsl[s];
  if (k.n_q > max_query_len) k.n_q = max_query_len;
  if (k.n_q < 0) k.n_q = 0;
  int ctx = ctx_lens[s];
  ctx = ctx < 0 ? 0 : (ctx > (1 << 30) ? (1 << 30) : ctx);
  k.first = window_left < 0 || ctx <= window_left ? 0 : ctx - window_left;
  k.n = k.n_q > 0 ? ctx - k.first + k.n_q : 0;
  k.there = k.n <= width - k.first ? k.n : (width > k.first ? (int)(width - k.first) : 0);
  return k;
}

// A NaN code of V stands in the dense rows as this bf16 number, which no code gives (it is below their smallest by a factor of 2^60)
// and which no sum notices: a weight of zero must not meet a NaN. The queries that see it get their NaN at the end.
constexpr uint32_t kNanMark = 1u;
enum : uint32_t { kTileNan = 1, kTileGone = 2 };     // flags of a tile: marked values in its V rows; rows that take no part (a bit each)
// NaN codes of four: 1 in every byte that is one
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7; }

// ---- 1. the visible keys of sequences seq0 ... as dense rows: a CTA per tile of 128 keys and head, 16 lanes per row, eight values each ----
__global__ void __launch_bounds__(256)
unpack_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const uint8_t* __restrict__ k_scale,
              const uint8_t* __restrict__ v_scale, const int32_t* __restrict__ block_tables, int max_blocks,
              const int32_t* __restrict__ query_start_loc, const int32_t* __restrict__ context_lens, int seq0, int kvh,
              int64_t num_blocks, int block_size, int64_t cache_block_stride, int64_t scale_block_stride, int window_left,
              int max_query_len, int rows_per_seq, int64_t rows_total, uint8_t* __restrict__ k_out, uint8_t* __restrict__ v_out,
              uint4* __restrict__ gone, uint32_t* __restrict__ tile_flags, int32_t* status) {
  const int s = seq0 + (int)blockIdx.y;
  const Keys ks = keys_of(query_start_loc, context_lens, s, window_left, max_query_len, (int64_t)max_blocks * block_size);
  if (ks.n > ks.there && blockIdx.x == 0 && threadIdx.x == 0) raise_status(status, SBK_ST_BAD_BLOCK);
  // consecutive CTAs take the heads of a tile: the rows of a token are contiguous in the cache
  const int tile = (int)blockIdx.x / kvh, h = (int)blockIdx.x - tile * kvh;
  if (ks.n_q == 0 || (tile > 0 && tile * kTile >= ks.there)) return;      // (a run that sees nothing still reads a tile of zeros)
  const int l = threadIdx.x & 15;
  const int32_t* table = block_tables + (int64_t)s * max_blocks;
  const int64_t row0 = (int64_t)blockIdx.y * rows_per_seq + tile * kTile;
  __shared__ uint32_t miss[4];
  if (threadIdx.x < 4) miss[threadIdx.x] = 0u;
  __syncthreads();
  bool any_nan = false;
#pragma unroll 4
  for (int i = threadIdx.x >> 4; i < kTile; i += 16) {
    const int r = tile * kTile + i;
    uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
    if (r < ks.there) {
      const int tok = ks.first + r, lb = tok / block_size, off = tok - lb * block_size;
      const int32_t pb = table[lb];
      if (pb < 0 || pb >= num_blocks) {
        if (l == 0) {
          raise_status(status, SBK_ST_BAD_BLOCK);
          atomicOr(&miss[i >> 5], 1u << (i & 31));
        }
      } else {
        const int64_t at = (int64_t)pb * cache_block_stride + ((int64_t)off * kvh + h) * kD + 8 * l;
        const int64_t sa = (int64_t)pb * scale_block_stride + (int64_t)h * block_size + off;
        const uint2 kc = *reinterpret_cast<const uint2*>(k_cache + at), vc = *reinterpret_cast<const uint2*>(v_cache + at);
        const float kf = q8::byte_scale(k_scale[sa]), vf = q8::byte_scale(v_scale[sa]);
        auto two = [](uint32_t w, float f) {
          const float2 x = q8::e4m3x2_to_float2(w);
          return pack_bf16x2(x.x * f, x.y * f);
        };
        kw = make_uint4(two(kc.x & 0xffffu, kf), two(kc.x >> 16, kf), two(kc.y & 0xffffu, kf), two(kc.y >> 16, kf));
        vw = make_uint4(two(vc.x & 0xffffu, vf), two(vc.x >> 16, vf), two(vc.y & 0xffffu, vf), two(vc.y >> 16, vf));
        const uint32_t nx = nan_bytes(vc.x), ny = nan_bytes(vc.y);
        if (__builtin_expect(nx | ny, 0)) {
          auto mark = [](uint32_t w, uint32_t n) {
            if (n & 1u) w = (w & 0xffff0000u) | kNanMark;
            if (n & 0x100u) w = (w & 0xffffu) | kNanMark << 16;
            return w;
          };
          vw = make_uint4(mark(vw.x, nx), mark(vw.y, nx >> 16), mark(vw.z, ny), mark(vw.w, ny >> 16));
          any_nan = true;
        }
      }
    }
    const int64_t o = (((int64_t)h * rows_total + row0 + i) * kD + 8 * l) * 2;
    *reinterpret_cast<uint4*>(k_out + o) = kw;
    *reinterpret_cast<uint4*>(v_out + o) = vw;
  }
  any_nan = __syncthreads_or(any_nan);
  if (threadIdx.x == 0) {
    const int64_t at = (h * rows_total + row0) / kTile;
    const uint4 m = make_uint4(miss[0], miss[1], miss[2], miss[3]);
    const bool any_gone = m.x | m.y | m.z | m.w;
    if (any_gone) gone[at] = m;
    tile_flags[at] = (any_nan ? kTileNan : 0u) | (any_gone ? kTileGone : 0u);
  }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

// one lane of a converged warp, always the same
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}

// Two weights as packed bf16 heads and packed bf16 remainders: the heads are cut off (one instruction for both), not rounded, so
// a remainder is under 2^-7 of the weight, and its rounding under 2^-15. (Rounded heads: 714 us against 702 on 8192 queries.)
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
  float ra, rb;
  unpack2(ffma2(pack2(__uint_as_float(__float_as_uint(a) & 0xffff0000u), __uint_as_float(__float_as_uint(b) & 0xffff0000u)),
                pack2(-1.f, -1.f), pack2(a, b)), ra, rb);
  lo = pack_bf16x2(ra, rb);
}

// ---- 2. attention of the runs over the dense rows ----
__global__ void __launch_bounds__(kThreads, 1)
attend_kernel(const Params P, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  // barriers: K ring full / empty, V ring full / empty; per tile: S ready, P ready (four quarters of the keys); Q staged; all done; tiles' flags read.
  // S and P of a tile take turns strictly, so one barrier each and phase t & 1.
  const uint32_t bar_kf = sbase + kBarOff, bar_ke = bar_kf + 8 * kStagesK;
  const uint32_t bar_vf = bar_ke + 8 * kStagesK, bar_ve = bar_vf + 8 * kStagesV;
  const uint32_t bar_s = bar_ve + 8 * kStagesV, bar_p = bar_s + 16, bar_q = bar_p + 64, bar_done = bar_q + 8, bar_info = bar_done + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + kBarOff + 192);
  volatile uint8_t* abort_flag = smem + kBarOff + 208;
  volatile uint8_t* info = smem + kBarOff + 209;               // what the flags of this pair's tiles hold

  // pairs of tiles [0, split) are a CTA's each, the others two CTAs'
  int item = blockIdx.x, tile = -1;
  if (item >= P.split) {
    tile = (item - P.split) & 1;
    item = P.split + ((item - P.split) >> 1);
  }
  const int hk = item / P.pairs_per_head, kBQ = P.bq, G = P.G;
  item -= hk * P.pairs_per_head;
  const int sl = item / P.pairs, s = P.seq0 + sl;
  // later queries see more keys: they are launched first, so the long items do not start last
  const int q0 = (P.pairs - 1 - (item - sl * P.pairs)) * 2 * kBQ + (tile == 1 ? kBQ : 0), most = tile < 0 ? 2 * kBQ : kBQ;
  const Keys ks = keys_of(P.query_start_loc, P.context_lens, s, P.window_left, P.max_query_len, P.width);
  if (q0 >= ks.n_q) return;            // whole CTA, before anything is allocated
  const int nq_pair = ks.n_q - q0 < most ? ks.n_q - q0 : most;
  const bool has_b = nq_pair > kBQ;
  const int qs = P.query_start_loc[s] + q0;                // row of the pair's first query
  // in dense rows (row 0 = key ks.first): the last key of the pair's first query, the first key it sees, one past the last key
  const int p0 = ks.n - ks.n_q + q0;
  const int lo = P.window_left < 0 || p0 <= P.window_left ? 0 : p0 - P.window_left;
  // one past the last key of the pair; where the table ends in front of the first one, a tile that is masked altogether
  const int key_end = p0 + nq_pair < ks.there ? p0 + nq_pair : ks.there;
  const int t_lo = key_end > lo ? lo / kTile : 0, n_tiles = key_end > lo ? (key_end - 1) / kTile - t_lo + 1 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStagesK; ++i) { mbar_init(bar_kf + 8 * i, 1); mbar_init(bar_ke + 8 * i, 1); }
    for (int i = 0; i < kStagesV; ++i) { mbar_init(bar_vf + 8 * i, 1); mbar_init(bar_ve + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) mbar_init(bar_s + 8 * i, 1);
    for (int i = 0; i < 8; ++i) mbar_init(bar_p + 8 * i, 4);      // one arrival per warp of the tile
    mbar_init(bar_q, kSoftmaxWarps);
    mbar_init(bar_done, 1);
    mbar_init(bar_info, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kSoftmaxWarps + 2) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
    tmem_relinquish();
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // everyone meets here, then the allocating warp returns the tensor memory
  auto finish = [&]() {
    if (*abort_flag) {
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);   // copies and MMAs in flight land
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps + 2) tmem_dealloc(tmem, kTmemCols);
  };
  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kSoftmaxWarps || warp == kSoftmaxWarps + 1) {
      // ===== producers: one warp per ring, a tile is two copies of [128 rows][64 dims] =====
      const int kind = warp - kSoftmaxWarps;
      const int stages = kind ? kStagesV : kStagesK;
      bool ok = true;
      for (int t = 0; ok && t < n_tiles; ++t) {
        const int slot = t % stages, use = t / stages;
        const uint32_t bar_e = (kind ? bar_ve : bar_ke) + 8 * slot, bar_f = (kind ? bar_vf : bar_kf) + 8 * slot;
        if (use > 0 && !mbar_wait_bounded(bar_e, (use - 1) & 1)) ok = false;
        if (*abort_flag) ok = false;
        if (!ok) break;
        if (lane == 0) {
          const uint32_t dst = sbase + (kind ? kVOff : kKOff) + slot * kOperandBytes;
          const CUtensorMap* map = kind ? &map_v : &map_k;
          const int row = sl * P.rows_per_seq + (t_lo + t) * kTile;
          mbar_arrive_expect_tx(bar_f, kOperandBytes);
          tma_load_3d(dst, map, 0, row, hk, bar_f);
          tma_load_3d(dst + kPanelBytes, map, 64, row, hk, bar_f);
        }
        __syncwarp();
      }
      if (!ok && lane == 0 && !*abort_flag) { raise_status(P.status, SBK_ST_WAIT_TIMEOUT); *abort_flag = 1; }
    } else if (warp == kSoftmaxWarps + 2) {
      // ================================= MMA issuer =================================
      // (an elected lane: behind `lane == 0` every MMA was issued some forty cycles later)
      const bool leader = elect_one();
      const uint32_t idesc_qk = instr_desc(0), idesc_pv = instr_desc(1);
      auto issue_s = [&](int X, int t) {     // S_X(t) = Q_X . K(t)^T
        if (leader) {
          const uint32_t q_addr = sbase + kQOff + X * kOperandBytes;
          const uint32_t k_addr = sbase + kKOff + (t % kStagesK) * kOperandBytes;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t off = (k >> 2) * kPanelBytes + (k & 3) * 32;
            umma_bf16(tmem + X * 128, smem_desc(q_addr + off, 16), smem_desc(k_addr + off, 16), idesc_qk, k > 0);
          }
          umma_commit(bar_s + 8 * X);
        }
        __syncwarp();
      };
      // O_X += P_X(t) . V(t) for a quarter of the keys: steps of 16 keys, whose P is 8 columns of packed pairs (heads) at the
      // beginning of the 32 columns its scores came from, and 8 of remainders 16 columns further
      auto issue_pv = [&](int X, int t, int quarter) {
        if (leader) {
          const uint32_t v_addr = sbase + kVOff + (t % kStagesV) * kOperandBytes;
#pragma unroll
          for (int k4 = 0; k4 < 2; ++k4) {
            const int k = 2 * quarter + k4;
            const uint32_t p_addr = tmem + X * 128 + 32 * quarter + 8 * k4;
            const uint64_t vd = smem_desc(v_addr + k * 2048, kPanelBytes);
            umma_bf16_ts(tmem + kOCol + X * 128, p_addr, vd, idesc_pv, (t > 0) || (k > 0));
            umma_bf16_ts(tmem + kOCol + X * 128, p_addr + 16, vd, idesc_pv, 1u);
          }
        }
        __syncwarp();
      };
      auto commit = [&](uint32_t bar) {
        if (leader) umma_commit(bar);
        __syncwarp();
      };
      auto k_full = [&](int t) { return mbar_wait_bounded(bar_kf + 8 * (t % kStagesK), (t / kStagesK) & 1) && !*abort_flag; };
      bool ok = mbar_wait_bounded(bar_q, 0) && k_full(0);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        if (has_b) issue_s(1, 0);
        commit(bar_ke);
      }
      for (int t = 0; ok && t < n_tiles; ++t) {
        const int vslot = t % kStagesV;
        const bool more = t + 1 < n_tiles;
        for (int X = 0; ok && X < (has_b ? 2 : 1); ++X) {
          const bool last = X == (has_b ? 1 : 0);
          // P_X(t), 32 keys at a time: the product of a quarter runs while the threads work on the next; behind the last one
          // S_X(t + 1) may take the place of P_X(t)
          ok = mbar_wait_bounded(bar_vf + 8 * vslot, (t / kStagesV) & 1);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            ok = ok && mbar_wait_bounded(bar_p + 32 * X + 8 * c, t & 1) && !*abort_flag;
            if (!ok) break;
            tc_fence_after();
            issue_pv(X, t, c);
          }
          if (!ok) break;
          if (last) commit(bar_ve + 8 * vslot);
          if (more) {
            if (X == 0) {
              ok = k_full(t + 1);
              if (!ok) break;
              tc_fence_after();
            }
            issue_s(X, t + 1);
            if (last) commit(bar_ke + 8 * ((t + 1) % kStagesK));
          }
        }
        if (*abort_flag) ok = false;
      }
      if (ok) commit(bar_done);
      if (!ok && lane == 0 && !*abort_flag) { raise_status(P.status, SBK_ST_WAIT_TIMEOUT); *abort_flag = 1; }
    } else {
      const uint32_t* flags = P.tile_flags + ((int64_t)hk * P.rows_total + (int64_t)sl * P.rows_per_seq) / kTile + t_lo;
      uint32_t any = 0u;
      for (int t = lane; t < n_tiles; t += 32) any |= flags[t];
      any = __reduce_or_sync(0xffffffffu, any);
      if (lane == 0) {
        *info = (uint8_t)any;
        mbar_arrive(bar_info);
      }
    }
    finish();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ====================== softmax / epilogue: one thread per row ======================
    const int X = warp >> 2;
    const int r = (warp & 3) * 32 + lane;        // row of the MMA tile = tensor-memory lane
    const int ql = r / G, slot_h = r - ql * G;   // rows past bq * G land on ql == bq: never a query of the tile
    const int nq_tile = X ? nq_pair - kBQ : (nq_pair < kBQ ? nq_pair : kBQ);
    const bool row_ok = ql < nq_tile;
    const int64_t q_row = qs + X * kBQ + ql;
    const int p_row = p0 + X * kBQ + ql;         // the row's last visible key
    const int lo_row = P.window_left < 0 || p_row <= P.window_left ? 0 : p_row - P.window_left;
    {
      const uint4* qp = reinterpret_cast<const uint4*>(P.q + q_row * P.q_tok_stride + (int64_t)(hk * G + slot_h) * kD);
      uint4 v[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        v[c] = row_ok ? qp[c] : make_uint4(0, 0, 0, 0);
        v[c].x ^= P.q_sign; v[c].y ^= P.q_sign; v[c].z ^= P.q_sign; v[c].w ^= P.q_sign;
      }
#pragma unroll
      for (int c = 0; c < 16; ++c)
        *reinterpret_cast<uint4*>(smem + kQOff + X * kOperandBytes + (c >> 3) * kPanelBytes + swz(r, c & 7)) = v[c];
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q);
    }
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = t_lane + X * 128, o_col = t_lane + kOCol + X * 128;
    float m_run = -INFINITY, mr = -INFINITY, l_run = 0.f;
    bool ok = mbar_wait_bounded(bar_info, 0);
    if (X == 0 || has_b) {
      for (int t = 0; ok && t < n_tiles; ++t) {
        ok = mbar_wait_bounded(bar_s + 8 * X, t & 1);
        if (!ok || *abort_flag) break;
        tc_fence_after();
        const int tb = (t_lo + t) * kTile;
        int v_lo = lo_row - tb, v_hi = (p_row < ks.there ? p_row + 1 : ks.there) - tb;   // columns this row may see: [v_lo, v_hi)
        v_lo = v_lo < 0 ? 0 : v_lo;
        v_hi = v_hi > kTile ? kTile : v_hi;
        const bool holes = *info & kTileGone;
        const bool full = __all_sync(0xffffffffu, v_lo == 0 && v_hi == kTile && !holes);   // the warp takes one path
        // ---- the row's scores and their maximum ----
        uint32_t sr4[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32_issue(s_col + 32 * c, sr4[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_fence(sr4[c]);
        float both;
        {
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if (full) {
#pragma unroll
            for (int i = 0; i < 32; i += 2)
#pragma unroll
              for (int c = 0; c < 4; ++c) mx[c] = fmax3(mx[c], __uint_as_float(sr4[c][i]), __uint_as_float(sr4[c][i + 1]));
          } else {
            // what the row does not see becomes -inf
            uint32_t hid[4] = {0u, 0u, 0u, 0u};
            if (holes) {
              const int64_t at = ((int64_t)hk * P.rows_total + (int64_t)sl * P.rows_per_seq) / kTile + t_lo + t;
              if (P.tile_flags[at] & kTileGone) {
                const uint4 g = P.gone[at];
                hid[0] = g.x; hid[1] = g.y; hid[2] = g.z; hid[3] = g.w;
              }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int a = v_lo - 32 * c, b = v_hi - 32 * c;
              if (a > 0) hid[c] |= a > 31 ? 0xffffffffu : (1u << a) - 1u;
              if (b < 32) hid[c] |= b <= 0 ? 0xffffffffu : 0xffffffffu << b;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                if (hid[c] >> i & 1u) sr4[c][i] = __float_as_uint(-INFINITY);
                mx[c] = fmaxf(mx[c], __uint_as_float(sr4[c][i]));
              }
            }
          }
          both = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        }
        const float cand = fmaxf(m_run, both * P.scale_log2);
        const bool move = cand > m_run + 8.f;   // also the first visible key of a row (m_run = -inf)
        const float mr_new = move ? both : mr;  // the offset as a score, and in the exponent's units
        const float m_s = move ? cand : fmaxf(m_run, kNegBig);
        const float alpha = !move ? 1.f : (mr == -INFINITY ? 0.f : fast_exp2((mr - mr_new) * P.scale_log2));
        if (move) m_run = cand;
        mr = mr_new;
        // One multiply-add per score where the offset is of ordinary size: all of a row's exponents are off by the rounding of the
        // offset, which cancels against l. Beyond 2^20 that rounding is no longer small against the exponent itself.
        const bool fast = full && __all_sync(0xffffffffu, fabsf(m_s) <= 1048576.f);
        // O moves with the offset. The products that wrote it are done: S_X(t) was issued behind P_X(t-1).V.
        if (__any_sync(0xffffffffu, t > 0 && alpha != 1.f)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t orr[32];
            tmem_ld32_issue(o_col + 32 * c, orr);
            tmem_ld_fence(orr);
#pragma unroll
            for (int i = 0; i < 32; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * alpha);
            tmem_st32(o_col + 32 * c, orr);
          }
        }
        // ---- probabilities in place of the scores, each quarter reported as soon as it is stored ----
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
        const f32x2 sc2 = pack2(P.scale_log2, P.scale_log2), nm2 = pack2(-m_s, -m_s);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t (&sr)[32] = sr4[2 * hf + cc];
            const int col0 = 64 * hf + 32 * cc;
            uint32_t ph[32];               // packed bf16 pairs, key 2e in the low half: [0, 16) heads, [16, 32) remainders
            if (fast) {
              f32x2 la = 0ull, lb = 0ull;
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                float x0, x1, x2, x3;
                unpack2(ffma2(pack2(__uint_as_float(sr[i]), __uint_as_float(sr[i + 1])), sc2, nm2), x0, x1);
                unpack2(ffma2(pack2(__uint_as_float(sr[i + 2]), __uint_as_float(sr[i + 3])), sc2, nm2), x2, x3);
                const float e0 = fast_exp2(x0), e1 = fast_exp2(x1), e2 = fast_exp2(x2), e3 = fast_exp2(x3);
                la = fadd2(la, pack2(e0, e1));
                lb = fadd2(lb, pack2(e2, e3));
                split2(e0, e1, ph[i >> 1], ph[16 + (i >> 1)]);
                split2(e2, e3, ph[(i >> 1) + 1], ph[17 + (i >> 1)]);
              }
              float a0, a1, b0, b1;
              unpack2(la, a0, a1);
              unpack2(lb, b0, b1);
              ls[0] += a0; ls[1] += a1; ls[2] += b0; ls[3] += b1;
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float pa = fast_exp2((__uint_as_float(sr[i]) - mr) * P.scale_log2);
                float pb = fast_exp2((__uint_as_float(sr[i + 1]) - mr) * P.scale_log2);
                if (__uint_as_float(sr[i]) == -INFINITY) pa = 0.f;
                if (__uint_as_float(sr[i + 1]) == -INFINITY) pb = 0.f;
                ls[i & 3] += pa;
                ls[(i + 1) & 3] += pb;
                split2(pa, pb, ph[i >> 1], ph[16 + (i >> 1)]);
              }
            }
            tmem_st32(s_col + col0, ph);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p + 32 * X + 16 * hf + 8 * cc);
          }
        }
        l_run = l_run * alpha + (ls[0] + ls[1]) + (ls[2] + ls[3]);
      }
      if (ok && !*abort_flag) {
        ok = mbar_wait_bounded(bar_done, 0);
        if (ok) {
          tc_fence_after();
          const float inv = l_run != 0.f ? 1.f / l_run : 0.f;
          uint4* op = reinterpret_cast<uint4*>(P.out + q_row * P.out_tok_stride + (int64_t)(hk * G + slot_h) * kD);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t orr[32];
            tmem_ld32_issue(o_col + 32 * c, orr);
            tmem_ld_fence(orr);
            if (row_ok) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                op[c * 4 + e] = make_uint4(
                    pack_bf16x2(__uint_as_float(orr[e * 8 + 0]) * inv, __uint_as_float(orr[e * 8 + 1]) * inv),
                    pack_bf16x2(__uint_as_float(orr[e * 8 + 2]) * inv, __uint_as_float(orr[e * 8 + 3]) * inv),
                    pack_bf16x2(__uint_as_float(orr[e * 8 + 4]) * inv, __uint_as_float(orr[e * 8 + 5]) * inv),
                    pack_bf16x2(__uint_as_float(orr[e * 8 + 6]) * inv, __uint_as_float(orr[e * 8 + 7]) * inv));
            }
          }
          if (__builtin_expect(*info & kTileNan, 0)) {
            // the marked dims of the keys that this row sees: dim 4 l + i is bit l of word i
            uint32_t bits[4] = {0u, 0u, 0u, 0u};
            const int64_t row0 = (int64_t)hk * P.rows_total + (int64_t)sl * P.rows_per_seq;
#pragma unroll 1
            for (int t = t_lo; t < t_lo + n_tiles; ++t) {
              if (!(P.tile_flags[row0 / kTile + t] & kTileNan)) continue;
              const int key0 = t * kTile;
              const uint16_t* rows = P.v_rows + (row0 + key0) * kD + 4 * lane;
#pragma unroll 1
              for (int j = 0; j < kTile; ++j) {
                const ushort4 v = *reinterpret_cast<const ushort4*>(rows + (int64_t)j * kD);
                const bool sees = key0 + j >= lo_row && key0 + j <= p_row;
                const uint32_t b[4] = {__ballot_sync(0xffffffffu, v.x == kNanMark), __ballot_sync(0xffffffffu, v.y == kNanMark),
                                       __ballot_sync(0xffffffffu, v.z == kNanMark), __ballot_sync(0xffffffffu, v.w == kNanMark)};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (sees) bits[i] |= b[i];
              }
            }
            if (row_ok) {
              uint16_t* o = reinterpret_cast<uint16_t*>(op);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                for (uint32_t b = bits[i]; b; b &= b - 1) o[4 * (__ffs(b) - 1) + i] = 0x7fffu;
            }
          }
        }
      }
    }
    if (!ok && lane == 0 && !*abort_flag) { raise_status(P.status, SBK_ST_WAIT_TIMEOUT); *abort_flag = 1; }
    finish();
  }
}

// Runs of at most kFew queries go through the kernel of the single tokens, which reads the cache once for four queries and
// expands nothing. Measured there against here, us, window 4096 on 8190 cached tokens: 256 runs of 16 1170 / 1348, of 17 1483 / 1348;
// 64 of 8 197 / 401, of 16 348 / 410, of 20 410 / 428, of 24 481 / 430. With fewer sequences the border lies higher, and what is in
// between loses here: 8 runs of 20 84 / 109, of 32 113 / 111; one of 20 51 / 94, of 128 74 / 92, of 300 125 / 96.
constexpr int kFew = 16;
static bool few_queries(int max_query_len, int kvh) { return max_query_len <= kFew && (kvh == 1 || kvh == 2 || kvh == 4); }

// dense rows of a sequence, and sequences that share one scratch
struct Layout { int64_t rows_per_seq; int group; };
static Layout layout_of(int n_seqs, int max_query_len, int max_blocks, int kvh, int block_size, int window_left) {
  Layout y;
  const int64_t width = (int64_t)max_blocks * block_size;
  int64_t n = width;
  if (window_left >= 0 && (int64_t)window_left + max_query_len < width) n = (int64_t)window_left + max_query_len;
  y.rows_per_seq = (n + kTile - 1) / kTile * kTile;
  const int64_t bytes = y.rows_per_seq * kvh * kD * 4;      // K and V in bf16
  int64_t g = kScratchTarget / bytes;
  if (g < 1) g = 1;
  y.group = (int)(g < n_seqs ? g : n_seqs);
  return y;
}
// the workspace: dense K rows, dense V rows, for every head and tile 16 bytes of missing rows and the flags
static size_t dense_bytes(const Layout& y, int kvh) { return (size_t)(y.rows_per_seq * y.group) * kvh * kD * 4; }
static size_t scratch_bytes(const Layout& y, int kvh) { return dense_bytes(y, kvh) + (size_t)(y.rows_per_seq / kTile * y.group) * kvh * 20; }

}  // namespace prefill_q8
}  // namespace sbk

extern "C" size_t sbk_swa_prefill_q8_workspace_bytes(int n_seqs, int max_query_len, int max_blocks, int kvh, int D, int block_size,
                                                     int window_left) {
  using namespace sbk::prefill_q8;
  if (n_seqs <= 0 || max_query_len <= 0 || max_blocks <= 0 || kvh <= 0 || D <= 0 || block_size <= 0) return 0;
  if (few_queries(max_query_len, kvh)) return sbk::decode_q8::workspace_bytes(8 * kvh, true);   // H is 8 * kvh at the most
  return scratch_bytes(layout_of(n_seqs, max_query_len, max_blocks, kvh, block_size, window_left), kvh);
}

extern "C" int sbk_swa_prefill_q8(const void* q, int64_t q_tok_stride, const void* k_cache, const void* v_cache,
                                  const void* k_scale, const void* v_scale, const int32_t* block_tables, int max_blocks,
                                  const int32_t* query_start_loc, const int32_t* context_lens, int n_seqs,
                                  int max_query_len, int H, int kvh, int D, int64_t num_blocks, int block_size,
                                  int64_t cache_block_stride_bytes, int64_t scale_block_stride_bytes, int window_left,
                                  float scale, void* out, int64_t out_tok_stride, void* workspace, size_t workspace_bytes,
                                  int32_t* status, void* stream) {
  using namespace sbk;
  using namespace sbk::prefill_q8;
  if (n_seqs < 0 || max_query_len < 0 || H <= 0 || kvh <= 0 || H % kvh != 0 || num_blocks < 0) {
    set_error("sbk_swa_prefill_q8: bad sizes n_seqs=%d max_query_len=%d H=%d kvh=%d", n_seqs, max_query_len, H, kvh);
    return SBK_E_ARG;
  }
  if (D != kD || H / kvh > 8) {
    set_error("sbk_swa_prefill_q8: unsupported shape D=%d H/kvh=%d (need D=128, at most 8 query heads per kv head)", D, H / kvh);
    return SBK_E_ARG;
  }
  if (block_size <= 0 || block_size % 16 != 0) {
    set_error("sbk_swa_prefill_q8: block_size=%d must be a positive multiple of 16", block_size);
    return SBK_E_ARG;
  }
  if (n_seqs == 0 || max_query_len == 0) return SBK_OK;
  if (max_blocks <= 0 || !q || !k_cache || !v_cache || !k_scale || !v_scale || !block_tables || !query_start_loc || !context_lens || !out) {
    set_error("sbk_swa_prefill_q8: null pointer or max_blocks=%d", max_blocks);
    return SBK_E_ARG;
  }
  if ((int64_t)max_blocks * block_size > decode_q8::kMaxWidth) {
    set_error("sbk_swa_prefill_q8: a table of %d blocks of %d tokens spans more than 2^30 tokens", max_blocks, block_size);
    return SBK_E_ARG;
  }
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scale) || !aligned16(v_scale) ||
      cache_block_stride_bytes % 16 || scale_block_stride_bytes % 16 || !aligned16(q) || !aligned16(out) || q_tok_stride % 8 ||
      out_tok_stride % 8) {
    set_error("sbk_swa_prefill_q8: caches, scales, their block strides, q, out and their token strides must be 16-byte multiples");
    return SBK_E_ALIGN;
  }
  if (cache_block_stride_bytes < (int64_t)kvh * D * block_size || scale_block_stride_bytes < (int64_t)kvh * block_size) {
    set_error("sbk_swa_prefill_q8: a block stride is smaller than the block it spans");
    return SBK_E_ARG;
  }
  if (out_tok_stride < (int64_t)H * D) {
    set_error("sbk_swa_prefill_q8: the rows of out overlap");
    return SBK_E_ARG;
  }
  const size_t need = sbk_swa_prefill_q8_workspace_bytes(n_seqs, max_query_len, max_blocks, kvh, D, block_size, window_left);
  if (!workspace || workspace_bytes < need) {
    set_error("sbk_swa_prefill_q8: workspace of %zu bytes given, %zu needed", workspace ? workspace_bytes : 0, need);
    return SBK_E_WORKSPACE;
  }
  if (!aligned16(workspace)) {
    set_error("sbk_swa_prefill_q8: workspace must be 16-byte aligned");
    return SBK_E_ALIGN;
  }
  if (few_queries(max_query_len, kvh)) {
    decode_q8::Call c = {};
    c.q = q; c.q_stride = q_tok_stride;
    c.k_cache = k_cache; c.v_cache = v_cache; c.k_scale = k_scale; c.v_scale = v_scale;
    c.cache_block_stride = cache_block_stride_bytes; c.scale_block_stride = scale_block_stride_bytes;
    c.block_tables = block_tables; c.max_blocks = max_blocks;
    c.query_start_loc = query_start_loc; c.context_lens = context_lens; c.max_query_len = max_query_len;
    c.n_seqs = n_seqs; c.H = H; c.kvh = kvh; c.num_blocks = num_blocks; c.block_size = block_size; c.window_left = window_left;
    c.scale = scale; c.out = out; c.out_dtype = SBK_BF16; c.out_stride = out_tok_stride;
    c.workspace = workspace; c.status = status;
    return decode_q8::stream_cache("sbk_swa_prefill_q8", c, (cudaStream_t)stream);
  }
  const Layout y = layout_of(n_seqs, max_query_len, max_blocks, kvh, block_size, window_left);
  const int64_t rows = y.rows_per_seq * y.group;
  const int bq = 128 / (H / kvh);
  const int pairs = (max_query_len + 2 * bq - 1) / (2 * bq);
  if (rows > 2147483647LL || (int64_t)y.group * pairs * kvh > 1 << 30 || y.group > 65535) {
    set_error("sbk_swa_prefill_q8: grid or scratch too large");
    return SBK_E_ARG;
  }
  const size_t half = dense_bytes(y, kvh) / 2;
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    if (!encode_rows_map(&maps[i], (uint8_t*)workspace + i * half, rows, kvh)) {
      set_error("sbk_swa_prefill_q8: cuTensorMapEncodeTiled rejected the scratch (%lld rows, %d heads)", (long long)rows, kvh);
      return SBK_E_ARG;
    }
  }
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attend_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) {
      set_error("sbk_swa_prefill_q8: cannot opt in to %d bytes of shared memory: %s", kSmemBytes, cudaGetErrorString(e));
      return SBK_E_LAUNCH;
    }
    // (a split of the registers that the launch does not bring would wait forever)
    cudaFuncAttributes fa;
    const cudaError_t ea = cudaFuncGetAttributes(&fa, attend_kernel);
    if (ea != cudaSuccess ||
        fa.numRegs * kThreads < 32 * kSoftmaxWarps * kSoftmaxRegs + (kThreads - 32 * kSoftmaxWarps) * kOtherRegs) {
      set_error("sbk_swa_prefill_q8: the kernel was built with %d registers per thread", ea == cudaSuccess ? fa.numRegs : -1);
      return SBK_E_LAUNCH;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int sms = decode_q8::device_sms();
  cudaStream_t st = (cudaStream_t)stream;
  Params P = {};
  P.q = (const __nv_bfloat16*)q; P.q_tok_stride = q_tok_stride;
  P.query_start_loc = query_start_loc; P.context_lens = context_lens;
  P.rows_per_seq = (int)y.rows_per_seq; P.width = (int64_t)max_blocks * block_size; P.pairs = pairs;
  P.max_query_len = max_query_len; P.H = H; P.G = H / kvh; P.bq = bq;
  P.window_left = window_left; P.scale_log2 = fabsf(scale) * kLog2e; P.q_sign = scale < 0.f ? 0x80008000u : 0u;
  P.out = (__nv_bfloat16*)out; P.out_tok_stride = out_tok_stride; P.status = status;
  uint4* const gone = reinterpret_cast<uint4*>((uint8_t*)workspace + 2 * half);
  uint32_t* const tile_flags = reinterpret_cast<uint32_t*>(gone + rows / kTile * kvh);
  P.v_rows = reinterpret_cast<const uint16_t*>((const uint8_t*)workspace + half); P.rows_total = rows;
  P.gone = gone; P.tile_flags = tile_flags;
  // groups of sequences share the scratch, one after the other on the stream
  for (int s0 = 0; s0 < n_seqs; s0 += y.group) {
    const int n = n_seqs - s0 < y.group ? n_seqs - s0 : y.group;
    unpack_kernel<<<dim3((unsigned)(y.rows_per_seq / kTile * kvh), n), 256, 0, st>>>(
        (const uint8_t*)k_cache, (const uint8_t*)v_cache, (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_tables,
        max_blocks, query_start_loc, context_lens, s0, kvh, num_blocks, block_size, cache_block_stride_bytes,
        scale_block_stride_bytes, window_left, max_query_len, P.rows_per_seq, rows, (uint8_t*)workspace,
        (uint8_t*)workspace + half, gone, tile_flags, status);
    int rc = check_launch("sbk_swa_prefill_q8");
    if (rc != SBK_OK) return rc;
    P.seq0 = s0;
    // What is left for the last, partly filled round of CTAs takes one tile to a CTA if the SMs have room for twice as many: half
    // the queries take less than a pair, though more than half of it. Against pairs throughout, us, 28 + 4 heads: 8192 queries 621 / 631,
    // 1500 184 / 195, 4 x 700 274 / 287.
    const int64_t total = (int64_t)n * pairs * kvh;
    const int rest = (int)(total % sms);
    P.pairs_per_head = n * pairs;
    P.split = (int)(2 * rest <= sms ? total - rest : total);
    attend_kernel<<<(unsigned)(2 * total - P.split), kThreads, kSmemBytes, st>>>(P, maps[0], maps[1]);
    rc = check_launch("sbk_swa_prefill_q8");
    if (rc != SBK_OK) return rc;
  }
  return SBK_OK;
}
