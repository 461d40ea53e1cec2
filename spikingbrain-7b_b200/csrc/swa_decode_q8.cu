// Sliding-window attention of one query token per sequence, or of a few, over the 8-bit paged K/V cache (format: kv_q8.cuh):
//     s_j = scale * 2^ek_j * sum_d q_d ck_jd      o = sum_j softmax(s)_j * 2^ev_j * cv_jd      lse = log sum_j exp(s_j)
// over the visible tokens j of a sequence, ck / cv being the e4m3 codes and ek / ev the exponents of a row.
//
// Single tokens are bound by HBM: 2 kvh (D + 1) bytes per visible token, at 14 flops a byte. 28 + 4 heads of 128, window 4096:
//   256 sequences of 8193 tokens 170 us (1.08 GB, 6.4 TB/s); 64 of 1025 ... 32769 54 us (4.9 TB/s; 11 us of it until the first
//   bytes come and from the last ones to the folded rows); 4 of 100003 ... 131072, no window, 87 us (5.8
//   TB/s).
// Runs of up to four queries to an item read the cache once for them, and are bound by the instructions around the products: 64 x 4
//   queries 115 us (2.4 TB/s; 0.35 instructions issued per cycle and scheduler, eight consumer warps an SM being all that the
//   accumulators leave room for; 109 before values that a query does not see were kept from it). Against those 109: two groups of
//   four warps with two queries each, every code converted twice, 124 us; the weights of all four queries before one vote on the offsets, not query by query, 122 us.
//
// Products. Both run on mma.sync m16n8k16 in fp16, the codes converted in registers on their way into the A operand (exact, two codes
//   per instruction), K and V taking the 16-row side and the query heads of a kv group (at most eight) the other:
//       S^T[16 tokens, 8 heads] = K . Q^T            O^T[16 dims, 8 heads] = V^T . W^T
//   q is scaled by the power of two that takes its largest value to (2^13.8, 2^14.8]: a bf16 number is an fp16 number then, down to 2^-30
//   of the largest (below, an element is off by 2^-38 of the largest at the most). Feeding the codes to the e4m3 MMA as they are, with query and
//   probabilities split into two 4-bit parts, takes three times the instructions: the compiler expands that MMA into
//   conversions of both operands and two fp16 ones (64 mixed sequences: 72 us against 64 in fp16, the rest alike).
// Softmax. The V scale belongs to the probability's exponent: with an offset m per head the normaliser sums p_j = 2^(s_j - m), and
//   the product takes w_j = p_j 2^(ev_j - r), rounded to fp16's eleven bits. m and r are not the running maxima: they move only
//   when a w would leave fp16 (or p grow past 2^40), to put the largest w of the item between 2^6 and 2^7; until the
//   next move w may grow to 2^15, and the smallest fp16 number is 2^-30 of the largest w at the most. So a step costs one
//   vote where maxima over the tokens would cost twelve shuffles. At the end O * 2^r / l.
// Fragments. The order of tokens inside a tile is free as long as K, the exponents and V agree on it, and so is the order of
//   dims inside a K = 16 step: a 4-byte word of a row is two adjacent pairs, which become columns 2t, 2t+1 and 2t+8, 2t+9 of the
//   fragment. Row r of a tile is token r (r < 8) or 8 + (r - 8 ^ 4): the rows of K (plain ldmatrix) and of V (the transposing
//   8-bit one) then come from eight different 16-byte columns of the 128-byte swizzle, eight rows at a time.
// Data movement. One producer warp walks the block table and issues a TMA tensor copy per 16 tokens (kvh * 2 KiB of K, the same of V)
//   into a ring of three 32 KiB stages; two CTAs per SM. The exponents, 16 bytes per head and 16 tokens, come beside them through
//   the load path (cp.async): as bulk copies they took four of five requests of the copy engine (256 sequences: 214 us against 184). A stage holds 32
//   tokens per consumer warp: warp w serves kv head w % kvh and the 32-token part w / kvh.
// Partition. The units (one stage of tokens each) of all sequences, laid end to end with a fixed charge per sequence, are cut
//   into one equal run per CTA. Only the first and the last sequence of a run can be cut, so a CTA writes at most two partial results
//   (m, l, O): the workspace is indexed by CTA, holds nothing between calls and needs no clearing. A second kernel, launched
//   ahead of the first one's end (programmatic dependent launch), folds the partials: no counters, no waits between CTAs.
#include "kv_q8.cuh"
#include "sbk_tcgen05.cuh"
#include "sbk_tma.cuh"
#include "swa_decode_q8.cuh"

namespace sbk {
namespace decode_q8 {

constexpr int kD = 128, kChunk = 16, kMaxG = 8;
constexpr int kMaxSeqs = 1024;        // items (sequences, or groups of queries of one) per launch: lengths and prefix in shared memory
constexpr int kMaxSms = 160;          // as many as the workspace is laid out for
constexpr int kTileBytes = 16384;     // K, or V, of a stage
constexpr int kScaleBytes = 256;      // exponents of a stage: 128 of K, 128 of V
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kMergeWarpBytes = kMaxG * kD * 4;
constexpr float kMostW = 32768.f, kMostP = 1.099511627776e12f;   // 2^15, 2^40: where the offsets of the softmax move
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kNegBig = -1.0e30f;
enum : int { kFirst = 1, kLast = 2, kEnd = 4, kGoneShift = 8 };   // from kGoneShift on: a bit for each 16 tokens that the pool does not hold

// row: the item's first query row; n_q: its queries; top: one past the last key of the last of them (the table may end before);
// part: partial slot of the item's result, or -1 (direct)
struct StageInfo { int row, n_q, top, tok_base, lo, hi, flags, part; };

// Four consumer warps and a producer, two CTAs per SM. Up to two queries to an item live in registers. Four do not: their
// fragments and the state of their softmax lie in shared memory, in place of a third stage, and the consumers take over the
// registers that three idle warps beside the producer give up (what the block is launched with is what the two warpgroups
// hold afterwards: 256 x 128 = 128 x 216 + 128 x 40).
template <int NQ>
struct Cfg {
  static constexpr bool kShare = NQ > 2;
  static constexpr int kWarps = 4, kConsumers = 32 * kWarps, kThreads = kShare ? 256 : 160;
  static constexpr int kConsumerRegs = 216, kProducerRegs = 40;
  static constexpr int kCtasPerSm = 2;
  static constexpr int kStages = kShare ? 2 : 3;
  // What starting and finishing an item is charged, in units. Measured: 1024 ragged sequences 121 us with 2, 123 with 4, 126
  // with 8; runs 64 x 4: 124 us with 2, 120 with 4, 113 with 8, 109 with 12, 111 with 16
  static constexpr int kItemCost = kShare ? 12 : 2;
  static constexpr int kScaleOff = kStages * kStageBytes;
  static constexpr int kQueryOff = kScaleOff + kStages * kScaleBytes;   // [warp][query][4][lane] 16 bytes: steps 2j and 2j + 1
  static constexpr int kStateOff = kQueryOff + (kShare ? kWarps * NQ * 2048 : 0);   // [warp][query][t] (m, m, 2^-r, 2^-r)
  static constexpr int kFactorOff = kStateOff + (kShare ? kWarps * NQ * 64 : 0);    // [warp][query][head] what a product is scaled by
  static constexpr int kNanOff = kFactorOff + (kShare ? kWarps * NQ * 32 : 0);      // [warp][query] dims of the output that are NaN, a bit each
  static constexpr int kInfoOff = kNanOff + (NQ > 1 ? kWarps * NQ * 16 : 0);
  static constexpr int kPreOff = kInfoOff + kStages * (int)sizeof(StageInfo);
  static constexpr int kLensOff = kPreOff + (kMaxSeqs + 4) * 4;
  static constexpr int kCntOff = kLensOff + kMaxSeqs * 4;
  static constexpr int kMlFloats = NQ > 1 ? 20 : 16;             // (m, l) of a warp's heads at the end of an item, the dims that are NaN
  static constexpr int kMlOff = kCntOff + kMaxSeqs;
  static constexpr int kBarOff = kMlOff + kWarps * kMlFloats * 4;
  static constexpr int kMiscOff = kBarOff + (2 * kStages + 1) * 8;
  static constexpr int kSmemBytes = kMiscOff + 64 + 1024;        // + slack to align the ring to 1 KiB
  static_assert(kSmemBytes * kCtasPerSm <= 230400, "the CTAs of an SM must fit its shared memory");
  static_assert(kWarps * kMergeWarpBytes <= kStageBytes, "the merge scratch lives inside one stage");
  static_assert(!kShare || kConsumers * kConsumerRegs + (kThreads - kConsumers) * kProducerRegs <= kThreads * 128,
                "the registers of the warpgroups must fit what the block is launched with");
};

struct Params {
  const __nv_bfloat16* q; int64_t q_stride;
  const uint8_t* k_scale; const uint8_t* v_scale; int64_t scale_block_stride;
  const int32_t* block_tables; int max_blocks;
  const int32_t* seq_lens;                                    // single tokens; NULL: runs, whose item v is queries
  const int32_t* query_start_loc; const int32_t* context_lens; // cap * (v % per_seq) ... of sequence v / per_seq
  int per_seq, max_query_len;
  int item0, B;         // items [item0, item0 + B) of the call
  int H; int64_t num_blocks; int block_size, window_left; float scale_log2;
  void* out; int64_t out_stride; float* lse_out;
  int4* cut;            // (first query row, first CTA, pieces, queries; pieces <= 1: not cut), an entry per item where there are
                        // fewer of them than CTAs, else per CTA: the item that begins in its run and goes on
  int cut_by_item;
  float* ws_o; float2* ws_ml;   // partials [2 * CTA + slot][query][H][D] and [..][H]: slot 0 an item that began before, 1 one that goes on
  int32_t* status; int tile_copy;
};

struct Span { int first, units; };    // units [first, first + units) of the token axis hold the visible tokens
// width: tokens that a row of the block table has entries for
template <int UNIT>
__device__ __forceinline__ Span span_of(int top, int n_q, int window_left, int64_t width) {
  Span s;
  s.first = s.units = 0;
  if (top <= 0) return s;
  const int t0 = first_visible(top, n_q, window_left), end = top < width ? top : (int)width;
  if (end <= t0) return s;
  s.first = t0 / UNIT;
  s.units = (end - 1) / UNIT - s.first + 1;
  return s;
}

// D(16x8,f32) += A(16x16,f16,row) * B(16x8,f16,col)
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// words of four codes of rows g (lo) and g + 8 (hi) -> an A fragment: each word holds columns 2t, 2t+1, then 2t+8, 2t+9
__device__ __forceinline__ void widen(uint32_t (&a)[4], uint32_t lo, uint32_t hi) {
  a[0] = q8::e4m3x2_to_f16x2(lo & 0xffffu); a[1] = q8::e4m3x2_to_f16x2(hi & 0xffffu);
  a[2] = q8::e4m3x2_to_f16x2(lo >> 16); a[3] = q8::e4m3x2_to_f16x2(hi >> 16);
}
// two 16 x 16 byte matrices, transposed: lane 4g + t gets column g (r0) and g + 8 (r1) of the first, rows 4t ... 4t+3, and the
// same of the second (r2, r3); lanes 0-15 name the rows of the first matrix, 16-31 those of the second
__device__ __forceinline__ void ldmatrix_b8_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes global -> shared through the load path, and the arrival of a lane's copies on a barrier
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}
__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// mbar_wait_bounded as one statement: as a loop of the language it cost runs of four 7 us of 115, by what the compiler made of the code
// around it
__device__ __forceinline__ uint32_t meet_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      " .reg .pred p, q;\n"
      " .reg .u32 n;\n"
      " mov.u32 n, 0;\n"
      "again:\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " add.u32 n, n, 1;\n"
      " setp.lt.and.u32 q, n, 0x1000000, !p;\n"
      " @q bra again;\n"
      " selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}

template <typename TO> __device__ __forceinline__ void store2(TO* p, float a, float b);
template <> __device__ __forceinline__ void store2<float>(float* p, float a, float b) { p[0] = a; p[1] = b; }
template <> __device__ __forceinline__ void store2<__nv_bfloat16>(__nv_bfloat16* p, float a, float b) {
  if ((reinterpret_cast<uintptr_t>(p) & 3u) == 0) {
    *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(a, b);
  } else {
    p[0] = __float2bfloat16_rn(a); p[1] = __float2bfloat16_rn(b);
  }
}
template <typename TO>
__device__ __forceinline__ void store4(TO* p, float4 v) { store2(p, v.x, v.y); store2(p + 2, v.z, v.w); }

// log-sum-exp of a row; l is NaN where a score was
__device__ __forceinline__ float row_lse(float m, float l) { return l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY; }
__device__ __forceinline__ float inverse(float l) { return l != 0.f ? 1.f / l : 0.f; }

using namespace tc5;                  // packed fp32 pairs

template <int KVH, int NQ, typename TO>
__global__ void __launch_bounds__(Cfg<NQ>::kThreads, Cfg<NQ>::kCtasPerSm)
stream_kernel(const Params P, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using C = Cfg<NQ>;
  constexpr int kStages = C::kStages, kThreads = C::kThreads;
  constexpr int kCap = NQ;                            // queries of an item
  constexpr int kSub = 4 / KVH;                       // 32-token parts of a stage
  constexpr int kUnit = 32 * kSub;                    // tokens of a stage
  constexpr int kChunks = kUnit / kChunk;             // 16-token chunks of a stage
  constexpr int kChunkBytes = KVH * kChunk * kD;      // one chunk of K or of V: [head][token][128 B]
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t ring = smem_u32(smem);
  StageInfo* info = reinterpret_cast<StageInfo*>(smem + C::kInfoOff);
  int* pre = reinterpret_cast<int*>(smem + C::kPreOff);
  int* tops = reinterpret_cast<int*>(smem + C::kLensOff);
  uint8_t* cnts = smem + C::kCntOff;
  const uint32_t bar_full = ring + C::kBarOff, bar_empty = bar_full + 8 * kStages, bar_meet = bar_empty + 8 * kStages;
  volatile int* misc = reinterpret_cast<volatile int*>(smem + C::kMiscOff);   // [0] abort, [1] longest, [2..] scan
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 kNotCut = make_int4(-1, 0, 0, 0);
  const int64_t width = (int64_t)P.max_blocks * P.block_size;

  // the folding kernel may be set up while this one runs (it waits for this one's end before it reads anything)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (threadIdx.x == 0) {
    prefetch_map(&map_k);
    prefetch_map(&map_v);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1 + 32);   // the stage's bytes, and each producer lane's exponents
      mbar_init(bar_empty + 8 * s, C::kWarps);
    }
    mbar_init(bar_meet, C::kWarps);
    misc[0] = 0;
    misc[1] = 0;
    pre[0] = 0;
    fence_mbar_init();
  }
  __syncthreads();
  // what came before on the stream is done from here on (this kernel may have been set up ahead of its end)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // ---- what every item costs, as an exclusive prefix: units of b occupy [pre[b], pre[b] + units), its charge follows ----
  {
    constexpr int kRun = (kMaxSeqs + kThreads - 1) / kThreads;
    const int run_len = (P.B + kThreads - 1) / kThreads;
    const int b_lo = threadIdx.x * run_len;
    int cnt[kRun], sum = 0, mx = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int b = b_lo + i;
      int c = 0;
      if (i < run_len && b < P.B) {
        int top, n = 1;
        if (P.seq_lens) {
          top = P.seq_lens[P.item0 + b];
        } else {
          const int v = P.item0 + b, s = v / P.per_seq, q0 = (v - s * P.per_seq) * kCap;
          n = P.query_start_loc[s + 1] - P.query_start_loc[s];
          n = (n < P.max_query_len ? n : P.max_query_len) - q0;
          n = n > kCap ? kCap : n;
          int ctx = P.context_lens[s];
          ctx = ctx < 0 ? 0 : (ctx > (1 << 30) ? (1 << 30) : ctx);
          top = n > 0 ? ctx + q0 + n : -1;   // -1: no such queries, nothing to write
        }
        // (tokens that the table has no entry for are not there)
        if (top > width && blockIdx.x == 0) raise_status(P.status, SBK_ST_BAD_BLOCK);
        tops[b] = top;
        cnts[b] = (uint8_t)(n > 0 ? n : 0);
        if (top < 0 && P.seq_lens) tops[b] = top = 0;
        if (top >= 0) {
          c = max(span_of<kUnit>(top, n, P.window_left, width).units, 1);   // an empty one keeps a unit: somebody writes its zeros
          mx = max(mx, c);
          c += C::kItemCost;
        } else if (blockIdx.x == 0 && P.cut_by_item) {
          P.cut[b] = kNotCut;
        }
      }
      cnt[i] = c;
      sum += c;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    if (lane == 0) atomicMax(const_cast<int*>(&misc[1]), mx);
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    if (lane == 31) misc[2 + warp] = incl;
    __syncthreads();
    int run = incl - sum;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w)
      if (w < warp) run += misc[2 + w];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int b = b_lo + i;
      if (i < run_len && b < P.B) {
        run += cnt[i];
        pre[b + 1] = run;
      }
    }
    __syncthreads();
  }
  const int total = pre[P.B], n_cta = (int)gridDim.x, me = (int)blockIdx.x;
  int per = (total + n_cta - 1) / n_cta;
  if (per < 1) per = 1;
  // A batch of near-equal items that fills the CTAs evenly streams fastest as whole items: no partials to write and fold. Against
  // cutting, us: 256 sequences of 8193, window 4096, 170 / 183; 592 equal ones 215 / 221, 10 % apart 211 / 215. Limits: rounds that are
  // filled to 10/11 (to 10/13: 309 against 283 on 1024 items), the longest item 9/8 of the mean (11/8: 78 against 74 on 148 items 30 %
  // apart, 166 against 158 on 592). A lone round leaves CTAs empty: it pays, whole against cut, on 200 equal items of four kv heads 96 / 102,
  // not on 160 (86 / 84); of two on 220 (102 / 104), not on 180 (94 / 90); of one not on 148 (84 / 64) nor 220 (88 / 85).
  const int rounds = (P.B + n_cta - 1) / n_cta;
  const bool whole = (KVH == 4 ? 8 * P.B >= 5 * n_cta : 4 * P.B >= 3 * n_cta) && ((P.B <= n_cta && !C::kShare) || 10 * rounds * n_cta <= 11 * P.B) &&
                     (int64_t)misc[1] * P.B <= ((int64_t)total - (int64_t)C::kItemCost * P.B) / 8 * 9;
  auto first_row = [&](int b) {
    if (P.seq_lens) return P.item0 + b;
    const int v = P.item0 + b, s = v / P.per_seq;
    return P.query_start_loc[s] + (v - s * P.per_seq) * kCap;
  };

  if (warp >= C::kWarps) {
    if constexpr (C::kShare) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kProducerRegs));   // (every warp of the warpgroup)
      if (warp > C::kWarps) return;
    }
    // ================================= producer =================================
    int it = 0;
    bool aborted = false;
    auto stream_item = [&](int b, int unit0, int n_units, int part) {
      const int top = tops[b], n_q = cnts[b];
      const int t0 = first_visible(top, n_q, P.window_left);
      const int seq = (P.item0 + b) / P.per_seq;
      const int row = first_row(b);
      const int32_t* table = P.block_tables + (int64_t)seq * P.max_blocks;
      // the consumers ask for the query rows when the first stage is there: by then they are in this SM's cache
      const uint8_t* q_rows = reinterpret_cast<const uint8_t*>(P.q + (int64_t)row * P.q_stride);
      for (int i = lane; i < n_q * P.H * kD / 64; i += 32) {
        const int qi = i / (P.H * kD / 64);
        prefetch_l1(q_rows + (int64_t)qi * P.q_stride * 2 + (i - qi * (P.H * kD / 64)) * 128);
      }
      int64_t pb_lane = -1;            // physical block of chunk (batch0 + lane): one table read per 32 chunks
      int batch0 = 0;
      const int n = n_units > 0 ? n_units : 1;
      for (int j = 0; j < n; ++j, ++it) {
        const int c0 = (unit0 + j) * kChunks;
        if (n_units > 0 && (j == 0 || c0 + kChunks > batch0 + 32)) {
          batch0 = c0;
          const int lb = (c0 + lane) * kChunk / P.block_size;
          pb_lane = (c0 + lane) * kChunk < top && lb < P.max_blocks ? (int64_t)table[lb] : -1;
        }
        const int s = it % kStages, use = it / kStages;
        if (use > 0 && !mbar_wait_bounded(bar_empty + 8 * s, (use - 1) & 1)) {
          if (lane == 0) { raise_status(P.status, SBK_ST_WAIT_TIMEOUT); misc[0] = 1; }
          aborted = true;
          return;
        }
        if (misc[0]) { aborted = true; return; }
        const int base = c0 * kChunk;
        const int lo = base > t0 ? base : t0;
        int hi = base + kUnit < top ? base + kUnit : top;
        if (hi > width) hi = (int)width;
        if (n_units == 0 || hi < lo) hi = lo;
        // chunks of this stage that hold visible tokens: [ca, cb)
        const int ca = (lo - base) / kChunk, cb = hi > lo ? (hi - 1 - base) / kChunk + 1 : ca;
        // lanes 0-15: exponents (chunk, head) of K and of V, 16 bytes each; lanes 16-31: the tiles
        const int x = lane & 15;
        const bool is_tile = lane >= 16;
        const int c = is_tile ? x % kChunks : x / KVH % kChunks;
        int src = c0 + c - batch0;
        src = src < 0 ? 0 : (src > 31 ? 31 : src);
        const int64_t pb = __shfl_sync(0xffffffffu, pb_lane, src);
        const bool in = c >= ca && c < cb;
        const bool bad = in && (pb < 0 || pb >= P.num_blocks);
        const uint32_t gone = __ballot_sync(0xffffffffu, bad) >> 16 & ((1u << kChunks) - 1u);   // (lanes 16 ...: chunks 0 ...)
        if (lane == 0) {
          StageInfo si;
          si.row = row; si.n_q = n_q; si.top = top; si.tok_base = base; si.lo = lo; si.hi = hi; si.part = part;
          si.flags = (j == 0 ? kFirst : 0) | (j == n - 1 ? kLast : 0) | (int)(gone << kGoneShift);
          info[s] = si;
          if (gone) raise_status(P.status, SBK_ST_BAD_BLOCK);
          mbar_arrive_expect_tx(bar_full + 8 * s, (uint32_t)(cb - ca - __popc(gone)) * 2u * kChunkBytes);
        }
        __syncwarp();
        if (in && !bad) {
          const int tin = (base + c * kChunk) % P.block_size;
          const uint32_t bar = bar_full + 8 * s;
          if (!is_tile) {
            if (x < kChunks * KVH) {
              const int h = x % KVH;
              const int64_t at = pb * P.scale_block_stride + (int64_t)h * P.block_size + tin;
              const uint32_t dst = ring + C::kScaleOff + s * kScaleBytes + (((c >> 1) * KVH + h) * 2 + (c & 1)) * 16;
              cp_async16(dst, P.k_scale + at);
              cp_async16(dst + 128, P.v_scale + at);
            }
          } else if (x < kChunks) {
            const uint32_t dst = ring + s * kStageBytes + c * kChunkBytes;
            if (P.tile_copy) {
              tma_load_4d(dst, &map_k, 0, tin, 0, (int)pb, bar);
              tma_load_4d(dst + kTileBytes, &map_v, 0, tin, 0, (int)pb, bar);
            } else {
              for (int h = 0; h < KVH; ++h) {
                tma_load_4d(dst + h * 2048, &map_k, 0, h, tin, (int)pb, bar);
                tma_load_4d(dst + kTileBytes + h * 2048, &map_v, 0, h, tin, (int)pb, bar);
              }
            }
          }
        }
        cp_async_arrive(bar_full + 8 * s);
      }
    };

    if (whole) {
      if (lane == 0) P.cut[me] = kNotCut;      // (entries per item, where they are that, are fewer than CTAs)
      for (int b = me; b < P.B && !aborted; b += n_cta) {
        if (tops[b] < 0) continue;
        const Span sp = span_of<kUnit>(tops[b], cnts[b], P.window_left, width);
        stream_item(b, sp.first, sp.units, -1);
      }
    } else {
      const int64_t g0 = (int64_t)me * per;
      const int64_t g1 = g0 + per < total ? g0 + per : total;
      int b0 = 0;
      int e = -1;
      int4 cut = kNotCut;
      if (g0 < total) {
        int hi_b = P.B;                 // largest b with pre[b] <= g0
        while (hi_b - b0 > 1) {
          const int mid = (b0 + hi_b) >> 1;
          if (pre[mid] <= g0) b0 = mid; else hi_b = mid;
        }
        // the item that holds the run's last slot: does it begin here and go on?
        int he = P.B;
        e = b0;
        while (he - e > 1) {
          const int mid = (e + he) >> 1;
          if (pre[mid] <= g1 - 1) e = mid; else he = mid;
        }
        const int cr = max(span_of<kUnit>(tops[e], cnts[e], P.window_left, width).units, 1);
        if (pre[e] >= g0 && pre[e] + cr > g1) cut = make_int4(first_row(e), me, (pre[e] + cr - 1) / per - me + 1, cnts[e]);
      }
      // (before anything is streamed: the folding kernel reads every entry, also of a launch that gave up on a wait)
      if (P.cut_by_item) {
        for (int b = b0 + lane; g0 < total && b < P.B && pre[b] < g1; b += 32)
          if (pre[b] >= g0 && tops[b] >= 0) P.cut[b] = b == e ? cut : kNotCut;
      } else if (lane == 0) {
        P.cut[me] = cut;
      }
      if (g0 < total) {
        for (int b = b0; b < P.B && pre[b] < g1 && !aborted; ++b) {
          if (tops[b] < 0) continue;
          const Span sp = span_of<kUnit>(tops[b], cnts[b], P.window_left, width);
          const int cr = sp.units > 0 ? sp.units : 1;
          const int va = (int)(g0 > pre[b] ? g0 - pre[b] : 0);
          if (va >= cr) continue;                               // only charged slots of b fall into this run
          int vb = (int)((g1 < pre[b + 1] ? g1 : pre[b + 1]) - pre[b]);
          if (vb > cr) vb = cr;
          const int part = va > 0 ? 0 : (vb < cr ? 1 : -1);
          stream_item(b, sp.first + va, sp.units > 0 ? vb - va : 0, part);
        }
      }
    }
    if (!aborted) {
      // the end marker travels through the ring like any stage
      const int s = it % kStages, use = it / kStages;
      if (use == 0 || mbar_wait_bounded(bar_empty + 8 * s, (use - 1) & 1)) {
        if (lane == 0) info[s].flags = kEnd;
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(bar_full + 8 * s, 0u);
        mbar_arrive(bar_full + 8 * s);
      } else if (lane == 0) {
        raise_status(P.status, SBK_ST_WAIT_TIMEOUT);
        misc[0] = 1;
      }
    } else {
      // copies in flight land before the CTA's shared memory goes back
      for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    }
    return;
  }

  // ================================== consumers ==================================
  if constexpr (C::kShare) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kConsumerRegs));
  const int hk = warp % KVH, sub = warp / KVH, G = P.H / KVH;
  const int g = lane >> 2, t = lane & 3;
  TO* const out = reinterpret_cast<TO*>(P.out);

  // A tile is [16 tokens][128 B], 16-byte column c of token r at r * 128 + ((c ^ (r & 7)) << 4).
  // K: lanes 0-7 and 8-15 name rows 0-7 and 8-15 at column c, lanes 16-31 the same rows at column c + 1
  const int rk = lane & 15, tokk = rk < 8 ? rk : 8 + ((rk - 8) ^ 4);
  // V: lane r (of each sixteen) names row r of the product, whose words run over rows 2t, 2t+1, 8+2t, 9+2t of the scores
  const int rv = 2 * (rk >> 2) + (rk & 1) + ((rk & 2) << 2), tokv = rv < 8 ? rv : 8 + ((rv - 8) ^ 4);
  const uint32_t tile0 = (uint32_t)(sub * 2 * kChunkBytes + hk * 2048);        // this warp's first sixteen tokens, its head
  const uint32_t k0 = tile0 + tokk * 128, v0 = kTileBytes + tile0 + tokv * 128;
  const int xk = (tokk & 7) ^ (lane >> 4), xv = (tokv & 7) ^ (lane >> 4);
  const int ta = g, tb8 = 8 + (g ^ 4);             // a thread's tokens in every sixteen

  constexpr int kR = C::kShare ? 1 : NQ;           // queries whose fragments and state are in registers all along
  uint32_t qf[kR][8][2];
  float acc[NQ][8][4];
  float m[kR][2], l[NQ][2], rs[kR][2], qs[kR][2];  // of heads 2t, 2t + 1 (rs = 2^-r)
  uint4* const q_sh = reinterpret_cast<uint4*>(smem + C::kQueryOff) + warp * NQ * 128 + lane;
  float4* const st_sh = reinterpret_cast<float4*>(smem + C::kStateOff) + warp * NQ * 4 + t;
  float* const fa_sh = reinterpret_cast<float*>(smem + C::kFactorOff) + warp * NQ * 8;
  uint32_t* const nan_sh = reinterpret_cast<uint32_t*>(smem + C::kNanOff) + warp * NQ * 4;
  auto load_state = [&](int n) {                   // of query n, to the registers of its slot
    if constexpr (C::kShare) {
      const float4 x = st_sh[4 * n];
      m[0][0] = x.x; m[0][1] = x.y; rs[0][0] = x.z; rs[0][1] = x.w;
    }
  };
  auto waited = [&](bool ok) {
    if (!ok && lane == 0) { raise_status(P.status, SBK_ST_WAIT_TIMEOUT); misc[0] = 1; }
    return ok;
  };
  // The consumer warps meet (bounded like every wait: a warp that gave up does not come), an even number of times in an item unless
  // it has one query and a warp to every kv head: so the phase is known where they meet. Who waited in vain goes on to the end of the
  // item (in bounds, with values that the status disowns), which costs no registers where leaving at once would.
  uint32_t met = 1;
  auto meet = [&](uint32_t phase) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_meet);
    met &= meet_wait(bar_meet, phase);
  };
  uint32_t odd_item = 0;
  for (int it = 0;; ++it) {
    const int s = it % kStages;
    if (!waited(mbar_wait_bounded(bar_full + 8 * s, (it / kStages) & 1))) return;
    const StageInfo si = info[s];
    if (si.flags & kEnd) return;
    const uint32_t stage = ring + s * kStageBytes;

    if (__builtin_expect(si.flags & kFirst, 0)) {
      if constexpr (NQ > 1) {
        __syncwarp();                              // (the item before is done with its state)
        if (lane < NQ * 4) nan_sh[lane] = 0u;
      }
#pragma unroll(kR)
      for (int n = 0; n < NQ; ++n) {
        const int r = C::kShare ? 0 : n;
        // q of head g: dims 16c + 4t ... + 3 (zeros for a head or a query that is not there)
        const bool head_ok = g < G && n < si.n_q;
        const __nv_bfloat16* qp =
            P.q + (int64_t)(si.row + (head_ok ? n : 0)) * P.q_stride + (int64_t)(hk * G + (head_ok ? g : 0)) * kD + 4 * t;
        uint32_t w[16];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          w[2 * c] = *reinterpret_cast<const uint32_t*>(qp + 16 * c);
          w[2 * c + 1] = *reinterpret_cast<const uint32_t*>(qp + 16 * c + 2);
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (!head_ok) w[i] = 0u;
          const float a = fabsf(__uint_as_float(w[i] << 16)), b = fabsf(__uint_as_float(w[i] & 0xffff0000u));
          top = fmaxf(top, fmaxf(q8::finite(a) ? a : 0.f, q8::finite(b) ? b : 0.f));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = q8::row_exponent(top);
        const float inv = q8::pow2i(6 - e), mine = P.scale_log2 * q8::pow2i(e - 6);   // 448 * 2^6 = 28672: inside fp16
#pragma unroll
        for (int i = 0; i < 16; ++i)         // (an infinity stays one: the head's scores are NaN or infinite)
          w[i] = pack_f16x2(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv);
        if constexpr (C::kShare) {
#pragma unroll
          for (int j = 0; j < 4; ++j) q_sh[(n * 4 + j) * 32] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
          if (t == 0) fa_sh[8 * n + g] = mine;
          if (g == 0) st_sh[4 * n] = make_float4(kNegBig, kNegBig, 1.f, 1.f);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) qf[r][i >> 1][i & 1] = w[i];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            qs[r][i] = __shfl_sync(0xffffffffu, mine, 4 * (2 * t + i));
            m[r][i] = kNegBig;
            rs[r][i] = 1.f;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) acc[n][mt][0] = acc[n][mt][1] = acc[n][mt][2] = acc[n][mt][3] = 0.f;
      }
      if constexpr (NQ > 1) __syncwarp();
    }

    const int tb = si.tok_base + 32 * sub;                      // my 32 tokens
    const int vlo = si.lo > tb ? si.lo : tb, vhi = si.hi < tb + 32 ? si.hi : tb + 32;
    if (vhi > vlo) {
      const uint32_t gone = (uint32_t)si.flags >> (kGoneShift + 2 * sub) & 3u;
      const bool edge = vlo > tb || vhi < tb + 32 || gone;
      if (__builtin_expect(edge, 0)) {
        // rows outside the visible range hold anything, or older data: a zero probability must not meet a NaN code
        for (int row = lane >> 3; row < 32; row += 4)
          if (tb + row < vlo || tb + row >= vhi || (gone >> (row >> 4) & 1u))
            *reinterpret_cast<uint4*>(smem + s * kStageBytes + kTileBytes + tile0 + (row >> 4) * kChunkBytes + (row & 15) * 128 +
                                      (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      bool cleared = edge;
      if constexpr (NQ > 1) {
        // Keys that only some of the item's queries see (in front of the last one's window, behind the first one's own key): their
        // weights are zero for the others, and a zero must not meet a NaN code. Such a code goes out of the tile, and the
        // queries that see it get its NaN at the end of the item.
        const int own = si.top - si.n_q;                       // the first query's own key
        const int common = P.window_left < 0 || si.top - 1 <= P.window_left ? 0 : si.top - 1 - P.window_left;
        if (__builtin_expect(vlo < common || vhi > own + 1, 0)) {
#pragma unroll 1
          for (int tok = vlo; tok < vhi; ++tok) {
            if (tok >= common && tok <= own) { tok = own; continue; }
            const int r = tok - tb;
            uint8_t* row = smem + s * kStageBytes + kTileBytes + tile0 + (r >> 4) * kChunkBytes + (r & 15) * 128;
            uint32_t* word = reinterpret_cast<uint32_t*>(row + (((lane >> 2) ^ (r & 7)) << 4)) + (lane & 3);
            const uint32_t nan = (((*word & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;    // 1 in every byte that is NaN
            if (__builtin_expect(!__any_sync(0xffffffffu, nan), 1)) continue;
            // (a lane's word is dims 4 lane ... 4 lane + 3: eight lanes to a word of the mask)
            uint32_t bits = ((nan & 1u) | (nan >> 7 & 2u) | (nan >> 14 & 4u) | (nan >> 21 & 8u)) << (4 * (lane & 7));
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, off);
            for (int n = 0; n < si.n_q; ++n)
              if ((lane & 7) == 0 && tok <= own + n && (P.window_left < 0 || tok >= own + n - P.window_left)) nan_sh[n * 4 + (lane >> 3)] |= bits;
            *word &= ~(nan * 255u);
            __syncwarp();
            cleared = true;
          }
        }
      }
      // ---- scores: [query][16-token half][token ta: heads 2t, 2t+1; token tb8: the same] ----
      float sc[NQ][2][4], ke[2][2], ve[2][2];
      const uint8_t* se = smem + C::kScaleOff + s * kScaleBytes + (sub * KVH + hk) * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ke[h][i] = __uint_as_float((uint32_t)se[16 * h + (i ? tb8 : ta)] << 23);
          ve[h][i] = __uint_as_float((uint32_t)se[128 + 16 * h + (i ? tb8 : ta)] << 23);
        }
      if constexpr (C::kShare) {
        // (one chain per query and half: there are enough of them)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[n][0][i] = sc[n][1][i] = 0.f;
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
          uint32_t w[2][4], a[2][4];
          uint4 q4[NQ];
#pragma unroll
          for (int n = 0; n < NQ; ++n) q4[n] = q_sh[(n * 4 + c / 2) * 32];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ldmatrix_x4(w[h], stage + h * kChunkBytes + k0 + ((c ^ xk) << 4));
            widen(a[h], w[h][0], w[h][1]);
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mma_f16(sc[n][0], a[0], q4[n].x, q4[n].y);
            mma_f16(sc[n][1], a[1], q4[n].x, q4[n].y);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) widen(a[h], w[h][2], w[h][3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mma_f16(sc[n][0], a[0], q4[n].z, q4[n].w);
            mma_f16(sc[n][1], a[1], q4[n].z, q4[n].w);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float cb[NQ][4];
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[n][h][i] = cb[n][i] = 0.f;
#pragma unroll
          for (int c = 0; c < 8; c += 2) {
            uint32_t w[4], a[4];
            ldmatrix_x4(w, stage + h * kChunkBytes + k0 + ((c ^ xk) << 4));
            widen(a, w[0], w[1]);
#pragma unroll
            for (int n = 0; n < NQ; ++n) mma_f16(sc[n][h], a, qf[n][c][0], qf[n][c][1]);
            widen(a, w[2], w[3]);
#pragma unroll
            for (int n = 0; n < NQ; ++n) mma_f16(cb[n], a, qf[n][c + 1][0], qf[n][c + 1][1]);
          }
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[n][h][i] += cb[n][i];
        }
      }
      if (__builtin_expect(edge, 0)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int a = tb + 16 * h + ta, b = tb + 16 * h + tb8;
          if (a < vlo || a >= vhi || (gone >> h & 1u)) ve[h][0] = 0.f;
          if (b < vlo || b >= vhi || (gone >> h & 1u)) ve[h][1] = 0.f;
        }
      }
      uint32_t pf[NQ][2][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int r = C::kShare ? 0 : n;
        load_state(n);
        if constexpr (C::kShare) {
          const float2 f = *reinterpret_cast<const float2*>(fa_sh + 8 * n + 2 * t);
          qs[0][0] = f.x; qs[0][1] = f.y;
        }
        const f32x2 q2 = pack2(qs[r][0], qs[r][1]);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; i += 2)
            unpack2(fmul2(pack2(sc[n][h][i], sc[n][h][i + 1]), fmul2(q2, pack2(ke[h][i >> 1], ke[h][i >> 1]))), sc[n][h][i], sc[n][h][i + 1]);
        // keys that this query sees; with several queries each has its own edge
        int nlo = vlo, nhi = vhi;
        if (NQ > 1) {
          const int last = si.top - si.n_q + n;            // the query's own position
          const int first = P.window_left < 0 || last <= P.window_left ? 0 : last - P.window_left;
          nlo = first > vlo ? first : vlo;
          nhi = last + 1 < vhi ? last + 1 : vhi;
        }
        if (__builtin_expect(nlo > tb || nhi < tb + 32 || gone, 0)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int a = tb + 16 * h + ta, b = tb + 16 * h + tb8;
            if (a < nlo || a >= nhi || (gone >> h & 1u)) sc[n][h][0] = sc[n][h][1] = -INFINITY;
            if (b < nlo || b >= nhi || (gone >> h & 1u)) sc[n][h][2] = sc[n][h][3] = -INFINITY;
          }
        }
        // ---- p = 2^(s - m), w = p * 2^(ev - r) with the offsets in use; they move only when a w leaves fp16 ----
        float w[2][4], ps[2], wtop;                 // (ps: sums of p)
        auto weigh = [&]() {
          const f32x2 nm = pack2(-m[r][0], -m[r][1]), r2 = pack2(rs[r][0], rs[r][1]);
          f32x2 sum = pack2(0.f, 0.f);
          wtop = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              float x, y;
              unpack2(fadd2(pack2(sc[n][h][i], sc[n][h][i + 1]), nm), x, y);
              const f32x2 p = pack2(fast_exp2(x), fast_exp2(y));
              sum = fadd2(sum, p);
              // (in this order: 2^-r is up to 2^70, 2^ev up to 2^63, and a weight of zero must not meet their product)
              unpack2(fmul2(fmul2(p, r2), pack2(ve[h][i >> 1], ve[h][i >> 1])), w[h][i], w[h][i + 1]);
              wtop = tc5::fmax3(wtop, w[h][i], w[h][i + 1]);
            }
          unpack2(sum, ps[0], ps[1]);
        };
        weigh();
        if (__builtin_expect(__any_sync(0xffffffffu, wtop > kMostW || fmaxf(ps[0], ps[1]) > kMostP), 0)) {
          // (rare: the first tokens of an item, and where a score or a V row outgrows all before it by 2^8)
          float mx[2], ne[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            mx[i] = fmaxf(fmaxf(sc[n][0][i], sc[n][0][2 + i]), fmaxf(sc[n][1][i], sc[n][1][2 + i]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
            mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float mn = fmaxf(m[r][i], mx[i]);
            ne[i] = fast_exp2(m[r][i] - mn);
            l[n][i] *= ne[i];
            m[r][i] = mn;
            mx[i] = 0.f;                        // from here on: the largest p * 2^ev
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              mx[i] = fmaxf(mx[i], fast_exp2(sc[n][h][i] - mn) * ve[h][0]);
              mx[i] = fmaxf(mx[i], fast_exp2(sc[n][h][2 + i] - mn) * ve[h][1]);
            }
          }
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
            mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // 2^-r: the power of two that takes the largest w so far to [2^6, 2^7) (those before had one of 2^6 at least)
            const float had = ne[i] * 64.f / rs[r][i];
            int e = (int)(__float_as_uint(fmaxf(mx[i], had)) >> 23) - 127;
            e = e < -64 ? -64 : (e > 63 ? 63 : e);
            const float rn = q8::pow2i(6 - e), al = ne[i] * (rn / rs[r][i]);
            rs[r][i] = rn;
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) { acc[n][mt][i] *= al; acc[n][mt][2 + i] *= al; }
          }
          weigh();
          if constexpr (C::kShare) {
            __syncwarp();
            if (g == 0) st_sh[4 * n] = make_float4(m[0][0], m[0][1], rs[0][0], rs[0][1]);
            __syncwarp();
          }
        }
        l[n][0] += ps[0];
        l[n][1] += ps[1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          pf[n][h][0] = movmatrix_trans(pack_f16x2(w[h][0], w[h][1]));
          pf[n][h][1] = movmatrix_trans(pack_f16x2(w[h][2], w[h][3]));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
          uint32_t v[4], a[4];
          ldmatrix_b8_trans(v, stage + h * kChunkBytes + v0 + ((c ^ xv) << 4));
          widen(a, v[0], v[1]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma_f16(acc[n][c], a, pf[n][h][0], pf[n][h][1]);
          widen(a, v[2], v[3]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma_f16(acc[n][c + 1], a, pf[n][h][0], pf[n][h][1]);
        }
      }
      if (cleared) fence_proxy_async_smem();   // what I wrote precedes the next copy into these rows
    }
    __syncwarp();
    // the last stage of an item becomes the scratch of its output before it goes back to the producer
    if (__builtin_expect(!(si.flags & kLast), 1)) {
      if (lane == 0) mbar_arrive(bar_empty + 8 * s);
      continue;
    }

    // ================= end of an item: its output rows, or its partials =================
    // [head][dim] floats of every warp in shared memory, four-float columns XOR-ed by the head (no bank is met twice);
    // warps that share a kv head (each took other tokens) are added up from there
    uint8_t* mbuf = smem + s * kStageBytes;
    float* wo = reinterpret_cast<float*>(mbuf + warp * kMergeWarpBytes);
    float* wml = reinterpret_cast<float*>(smem + C::kMlOff) + warp * C::kMlFloats;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = C::kShare ? 0 : n;
      load_state(n);
      // (where nothing was visible m is kNegBig, l and O are 0)
      float fix[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], off);
        fix[i] = 1.f / rs[r][i];
      }
      // every warp is done reading this stage, or the results of the query before
      meet(kSub > 1 ? 0u : (NQ > 1 ? (uint32_t)n & 1u : odd_item));
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int hrow = 2 * t + i, x = (hrow & 7) << 2;
          wo[hrow * kD + ((16 * mt + g) ^ x)] = acc[n][mt][i] * fix[i];
          wo[hrow * kD + ((16 * mt + g + 8) ^ x)] = acc[n][mt][2 + i] * fix[i];
        }
      if (g == 0) {
        wml[2 * t] = m[r][0]; wml[2 * t + 1] = m[r][1];
        wml[8 + 2 * t] = l[n][0]; wml[8 + 2 * t + 1] = l[n][1];
      }
      if constexpr (NQ > 1)
        if (lane < 4) wml[16 + lane] = __uint_as_float(nan_sh[n * 4 + lane]);
      if (kSub == 1) __syncwarp(); else meet(1u);
      if (n < si.n_q) {
        const int64_t orow = (int64_t)si.row + n;
        const int64_t prow = ((int64_t)(2 * me + (si.part > 0 ? 1 : 0)) * kCap + n) * P.H;
        // heads go round the warps (one warp to a kv head: its own heads), a lane takes four dims
        const int h_lo = kSub > 1 ? warp : hk * G, h_hi = kSub > 1 ? P.H : hk * G + G, h_step = kSub > 1 ? 4 : 1;
#pragma unroll 2
        for (int h = h_lo; h < h_hi; h += h_step) {
          const int kh = h / G, row = h - kh * G;
          float M = -INFINITY;
#pragma unroll
          for (int w2 = 0; w2 < kSub; ++w2)
            M = fmaxf(M, reinterpret_cast<const float*>(smem + C::kMlOff)[(kh + KVH * w2) * C::kMlFloats + row]);
          const float Ms = fmaxf(M, kNegBig);
          float L = 0.f;
          float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w2 = 0; w2 < kSub; ++w2) {
            const int src = kh + KVH * w2;
            const float* po = reinterpret_cast<const float*>(mbuf + src * kMergeWarpBytes);
            const float* ml = reinterpret_cast<const float*>(smem + C::kMlOff) + src * C::kMlFloats;
            const float wgt = kSub > 1 ? fast_exp2(ml[row] - Ms) : 1.f;
            const float4 o = *reinterpret_cast<const float4*>(po + row * kD + ((4 * lane) ^ ((row & 7) << 2)));
            L += ml[8 + row] * wgt;
            O.x += o.x * wgt; O.y += o.y * wgt; O.z += o.z * wgt; O.w += o.w * wgt;
            if constexpr (NQ > 1) {
              const uint32_t nan = __float_as_uint(ml[16 + (lane >> 3)]) >> (4 * (lane & 7));
              if (nan & 1u) O.x = __uint_as_float(0x7fffffffu);
              if (nan & 2u) O.y = __uint_as_float(0x7fffffffu);
              if (nan & 4u) O.z = __uint_as_float(0x7fffffffu);
              if (nan & 8u) O.w = __uint_as_float(0x7fffffffu);
            }
          }
          if (si.part < 0) {
            const float f = inverse(L);
            store4(out + orow * P.out_stride + (int64_t)h * kD + 4 * lane, make_float4(O.x * f, O.y * f, O.z * f, O.w * f));
            if (P.lse_out && lane == 0) P.lse_out[orow * P.H + h] = row_lse(M, L);
          } else {
            *reinterpret_cast<float4*>(P.ws_o + (prow + h) * kD + 4 * lane) = O;
            if (lane == 0) P.ws_ml[prow + h] = make_float2(M, L);
          }
        }
      }
    }
    fence_proxy_async_smem();               // these accesses precede the copies that refill the stage
    if (!waited(met)) return;
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_empty + 8 * s);
    odd_item ^= 1u;
  }
}

// Folds the partials of the items that were cut. Block (x, y): entry x of `cut`, heads HPC y ... of its cap * H (query, head) pairs;
// WPH warps share one, each taking every WPH-th piece with its loads issued eight at a time.
template <int WPH, int HPC, typename TO>
__global__ void __launch_bounds__(32 * WPH * HPC) fold_kernel(const Params P, int cap) {
  __shared__ float4 part_o[WPH * HPC][32];
  __shared__ float2 part_ml[WPH * HPC];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (the next launch waits for this one's end in the same way)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 cut = P.cut[blockIdx.x];                    // first query row, first CTA, pieces, queries
  if (cut.z <= 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hq = blockIdx.y * HPC + warp / WPH, w = warp % WPH;
  const bool on = hq < cut.w * P.H;
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kU = 8;
  for (int i0 = w; on && i0 < cut.z; i0 += WPH * kU) {
    float2 ml[kU];
    float4 o[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + WPH * u;
      ml[u] = make_float2(-INFINITY, 0.f);
      o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < cut.z) {
        const int64_t row = (int64_t)(2 * (cut.y + i) + (i == 0 ? 1 : 0)) * cap * P.H + hq;
        ml[u] = __ldcg(P.ws_ml + row);
        o[u] = __ldcg(reinterpret_cast<const float4*>(P.ws_o + row * kD) + lane);
      }
    }
    float Mn = M;
#pragma unroll
    for (int u = 0; u < kU; ++u) Mn = fmaxf(Mn, ml[u].x);
    const float Ms = fmaxf(Mn, kNegBig), resc = fast_exp2(M - Ms);
    L *= resc; O.x *= resc; O.y *= resc; O.z *= resc; O.w *= resc;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const float wgt = fast_exp2(ml[u].x - Ms);
      L += ml[u].y * wgt;
      O.x += o[u].x * wgt; O.y += o[u].y * wgt; O.z += o[u].z * wgt; O.w += o[u].w * wgt;
    }
    M = Mn;
  }
  part_o[warp][lane] = O;
  if (lane == 0) part_ml[warp] = make_float2(M, L);
  __syncthreads();
  if (w != 0 || !on) return;
  float Mt = -INFINITY;
#pragma unroll
  for (int q = 0; q < WPH; ++q) Mt = fmaxf(Mt, part_ml[warp + q].x);
  const float Ms = fmaxf(Mt, kNegBig);
  float Lt = 0.f;
  float4 Ot = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int q = 0; q < WPH; ++q) {
    const float2 ml = part_ml[warp + q];
    const float4 o = part_o[warp + q][lane];
    const float wgt = fast_exp2(ml.x - Ms);
    Lt += ml.y * wgt;
    Ot.x += o.x * wgt; Ot.y += o.y * wgt; Ot.z += o.z * wgt; Ot.w += o.w * wgt;
  }
  const float f = inverse(Lt);
  const int qi = hq / P.H, h = hq - qi * P.H;
  store4(reinterpret_cast<TO*>(P.out) + (int64_t)(cut.x + qi) * P.out_stride + (int64_t)h * kD + 4 * lane,
         make_float4(Ot.x * f, Ot.y * f, Ot.z * f, Ot.w * f));
  if (P.lse_out && lane == 0) P.lse_out[(int64_t)(cut.x + qi) * P.H + h] = row_lse(Mt, Lt);
}

constexpr int kMaxPartials = 2 * 2 * kMaxSms;          // two per CTA, two CTAs per SM
static size_t cut_bytes() { return (size_t)(2 * kMaxSms) * sizeof(int4); }

template <int KVH, int NQ, typename TO>
static int launch(const char* who, const Params& P0, int64_t items, int sms, const CUtensorMap& map_k, const CUtensorMap& map_v,
                  cudaStream_t st) {
  using C = Cfg<NQ>;
  constexpr int kCap = NQ, kUnit = 32 * 4 / KVH;
  auto kern = stream_kernel<KVH, NQ, TO>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) {
      set_error("%s: cannot opt in to %d bytes of shared memory: %s", who, C::kSmemBytes, cudaGetErrorString(e));
      return SBK_E_LAUNCH;
    }
    if (C::kShare) {      // (a split of the registers that the launch does not bring would wait forever)
      cudaFuncAttributes fa;
      const cudaError_t ea = cudaFuncGetAttributes(&fa, kern);
      if (ea != cudaSuccess ||
          fa.numRegs * C::kThreads < C::kConsumers * C::kConsumerRegs + (C::kThreads - C::kConsumers) * C::kProducerRegs) {
        set_error("%s: the kernel was built with %d registers per thread", who, ea == cudaSuccess ? fa.numRegs : -1);
        return SBK_E_LAUNCH;
      }
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int n_ctas = C::kCtasPerSm * (sms < kMaxSms ? sms : kMaxSms);
  const int64_t width = (int64_t)P0.max_blocks * P0.block_size, seen = (int64_t)P0.window_left + kCap;
  const int64_t vis = P0.window_left < 0 || width < seen ? width : seen;
  const int64_t per_item = vis / kUnit + 2 + C::kItemCost;     // units of an item, at the most
  int64_t step = 2147483647LL / per_item;                      // the units of a launch are counted in 32 bits
  step = step < 1 ? 1 : (step < kMaxSeqs ? step : kMaxSeqs);
  for (int64_t b0 = 0; b0 < items; b0 += step) {
    Params P = P0;
    P.item0 = (int)b0;
    P.B = (int)(items - b0 < step ? items - b0 : step);
    // no more CTAs than there can be units of work
    const int64_t most = (int64_t)P.B * per_item;
    int grid = (int)(most < n_ctas ? most : n_ctas);
    // A batch that nearly fills the CTAs, one item each: as many CTAs as items, so that every SM has work where near-equal items stay
    // whole. Measured against all CTAs, us, equal items: 256 items 111 / 115, 290 123 / 127; where lengths differ by up to half 90 / 92. With
    // fewer items it may only stay off: 148 equal ones 80 / 84, but 74 / 57 and 64 / 51 where lengths differ by a third and by half (7 + 1
    // heads). (Four queries to an item are bound by instructions, not by the copies that a lone CTA can keep up: there both CTAs of an SM
    // share.)
    if (!C::kShare && 4 * P.B >= 3 * n_ctas && P.B < n_ctas) grid = P.B;
    P.cut_by_item = P.B < grid;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t main_cfg = {};
    main_cfg.gridDim = dim3(grid);
    main_cfg.blockDim = dim3(C::kThreads);
    main_cfg.dynamicSmemBytes = C::kSmemBytes;
    main_cfg.stream = st;
    main_cfg.attrs = attr;
    main_cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&main_cfg, kern, P, map_k, map_v);
    if (e != cudaSuccess) {
      set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
      return SBK_E_LAUNCH;
    }
    // Few rows of output, each cut into two pieces a warp at least: sixteen warps to one, as long as the SMs hold them all at once.
    // Else four to a block of eight warps. (8 sequences x 1 token: 18.1 us against 19.3 the other way, 16 x 1: 25.6 against 28.7;
    // 8 x 4: 35 against 41; 8 x 16: 66 against 96)
    const bool few = (int64_t)P.B * P.H * kCap <= 4 * sms && grid >= 32 * P.B;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(P.cut_by_item ? P.B : grid, few ? P.H * kCap : (P.H * kCap + 3) / 4);
    cfg.blockDim = dim3(few ? 512 : 256);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = few ? cudaLaunchKernelEx(&cfg, fold_kernel<16, 1, TO>, P, kCap) : cudaLaunchKernelEx(&cfg, fold_kernel<2, 4, TO>, P, kCap);
    if (e != cudaSuccess) {
      set_error("%s: launch of the folding kernel failed: %s", who, cudaGetErrorString(e));
      return SBK_E_LAUNCH;
    }
  }
  return SBK_OK;
}

// rows of partials per head: runs have up to four queries to an item
static size_t partial_rows(bool runs) { return (size_t)kMaxPartials * (runs ? 4 : 1); }
size_t workspace_bytes(int H, bool runs) { return cut_bytes() + partial_rows(runs) * H * (kD + 2) * sizeof(float); }

int device_sms() {
  static int sm_count[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  int sms = dev >= 0 && dev < 64 ? sm_count[dev] : 0;
  if (sms == 0) {
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (sms <= 0) sms = 148;
    if (dev >= 0 && dev < 64) sm_count[dev] = sms;
  }
  return sms;
}

int stream_cache(const char* who, const Call& c, cudaStream_t st) {
  const bool runs = c.seq_lens == nullptr;
  Params P = {};
  P.q = (const __nv_bfloat16*)c.q; P.q_stride = c.q_stride;
  P.k_scale = (const uint8_t*)c.k_scale; P.v_scale = (const uint8_t*)c.v_scale; P.scale_block_stride = c.scale_block_stride;
  P.block_tables = c.block_tables; P.max_blocks = c.max_blocks; P.seq_lens = c.seq_lens;
  P.query_start_loc = c.query_start_loc; P.context_lens = c.context_lens; P.max_query_len = c.max_query_len;
  const bool two = c.max_query_len <= 2;                 // (what the registers hold)
  P.per_seq = !runs || two ? 1 : (c.max_query_len + 3) / 4;
  P.H = c.H; P.num_blocks = c.num_blocks; P.block_size = c.block_size; P.window_left = c.window_left;
  P.scale_log2 = c.scale * kLog2e; P.out = c.out; P.out_stride = c.out_stride; P.lse_out = c.lse_out; P.status = c.status;
  P.cut = (int4*)c.workspace;
  P.ws_o = (float*)((uint8_t*)c.workspace + cut_bytes());
  P.ws_ml = (float2*)(P.ws_o + partial_rows(runs) * c.H * kD);
  const int sms = device_sms();
  MapKey keys[2] = {MapKey{c.k_cache, c.kvh, c.num_blocks, c.block_size, c.cache_block_stride, c.kvh},
                    MapKey{c.v_cache, c.kvh, c.num_blocks, c.block_size, c.cache_block_stride, c.kvh}};
  for (MapKey& k : keys) { k.tok_stride = (int64_t)c.kvh * kD; k.rows = c.kvh; }
  CUtensorMap maps[2];
  if (!get_maps(maps, keys, 2, &P.tile_copy)) {
    set_error("%s: cuTensorMapEncodeTiled rejected the cache geometry (blocks=%lld block=%d kvh=%d)", who,
              (long long)c.num_blocks, c.block_size, c.kvh);
    return SBK_E_ARG;
  }
  const int64_t items = (int64_t)c.n_seqs * P.per_seq;
#define SBK_STREAM(NQ, TO)                                                                \
  switch (c.kvh) {                                                                        \
    case 1: return launch<1, NQ, TO>(who, P, items, sms, maps[0], maps[1], st);           \
    case 2: return launch<2, NQ, TO>(who, P, items, sms, maps[0], maps[1], st);           \
    default: return launch<4, NQ, TO>(who, P, items, sms, maps[0], maps[1], st);          \
  }
  if (runs && two) { SBK_STREAM(2, __nv_bfloat16) }
  if (runs) { SBK_STREAM(4, __nv_bfloat16) }
  if (c.out_dtype == SBK_BF16) { SBK_STREAM(1, __nv_bfloat16) } else { SBK_STREAM(1, float) }
#undef SBK_STREAM
}

}  // namespace decode_q8
}  // namespace sbk

extern "C" size_t sbk_swa_decode_q8_workspace_bytes(int B, int H, int D) {
  if (B <= 0 || H <= 0 || D <= 0) return 0;
  return sbk::decode_q8::workspace_bytes(H, false);
}

extern "C" int sbk_swa_decode_q8(const void* q, int64_t q_seq_stride, const void* k_cache, const void* v_cache,
                                 const void* k_scale, const void* v_scale, const int32_t* block_tables, int max_blocks,
                                 const int32_t* seq_lens, int B, int H, int kvh, int D, int64_t num_blocks,
                                 int block_size, int64_t cache_block_stride_bytes, int64_t scale_block_stride_bytes,
                                 int window_left, float scale, void* out, int out_dtype, int64_t out_seq_stride,
                                 float* lse_out, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace sbk;
  using namespace sbk::decode_q8;
  if (B < 0 || H <= 0 || kvh <= 0 || H % kvh != 0 || max_blocks <= 0 || num_blocks < 0) {
    set_error("sbk_swa_decode_q8: bad sizes B=%d H=%d kvh=%d max_blocks=%d", B, H, kvh, max_blocks);
    return SBK_E_ARG;
  }
  if (D != kD || H / kvh > kMaxG || !(kvh == 1 || kvh == 2 || kvh == 4)) {
    set_error("sbk_swa_decode_q8: unsupported shape D=%d H/kvh=%d kvh=%d (need D=128, group<=8, kvh in 1,2,4)", D, H / kvh, kvh);
    return SBK_E_ARG;
  }
  if (block_size <= 0 || block_size % 16 != 0) {
    set_error("sbk_swa_decode_q8: block_size=%d must be a positive multiple of 16", block_size);
    return SBK_E_ARG;
  }
  if ((int64_t)max_blocks * block_size > kMaxWidth) {
    set_error("sbk_swa_decode_q8: a table of %d blocks of %d tokens spans more than 2^30 tokens", max_blocks, block_size);
    return SBK_E_ARG;
  }
  if (out_dtype != SBK_BF16 && out_dtype != SBK_F32) {
    set_error("sbk_swa_decode_q8: out_dtype=%d unsupported", out_dtype);
    return SBK_E_ARG;
  }
  if (B == 0) return SBK_OK;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !block_tables || !seq_lens || !out) {
    set_error("sbk_swa_decode_q8: null pointer");
    return SBK_E_ARG;
  }
  if (!aligned16(k_cache) || !aligned16(v_cache) || !aligned16(k_scale) || !aligned16(v_scale) ||
      cache_block_stride_bytes % 16 || scale_block_stride_bytes % 16 || (reinterpret_cast<uintptr_t>(q) & 3u) ||
      (q_seq_stride & 1)) {
    set_error("sbk_swa_decode_q8: caches, scales and their block strides must be 16-byte multiples and q 4-byte aligned");
    return SBK_E_ALIGN;
  }
  if (cache_block_stride_bytes < (int64_t)kvh * D * block_size || scale_block_stride_bytes < (int64_t)kvh * block_size) {
    set_error("sbk_swa_decode_q8: a block stride is smaller than the block it spans");
    return SBK_E_ARG;
  }
  if (B > 1 && out_seq_stride < (int64_t)H * D) {
    set_error("sbk_swa_decode_q8: the rows of out overlap");
    return SBK_E_ARG;
  }
  const size_t need = sbk_swa_decode_q8_workspace_bytes(B, H, D);
  if (!workspace || workspace_bytes < need) {
    set_error("sbk_swa_decode_q8: workspace of %zu bytes given, %zu needed", workspace ? workspace_bytes : 0, need);
    return SBK_E_WORKSPACE;
  }
  if (!aligned16(workspace)) {
    set_error("sbk_swa_decode_q8: workspace must be 16-byte aligned");
    return SBK_E_ALIGN;
  }
  Call c = {};
  c.q = q; c.q_stride = q_seq_stride;
  c.k_cache = k_cache; c.v_cache = v_cache; c.k_scale = k_scale; c.v_scale = v_scale;
  c.cache_block_stride = cache_block_stride_bytes; c.scale_block_stride = scale_block_stride_bytes;
  c.block_tables = block_tables; c.max_blocks = max_blocks; c.seq_lens = seq_lens; c.max_query_len = 1;
  c.n_seqs = B; c.H = H; c.kvh = kvh; c.num_blocks = num_blocks; c.block_size = block_size; c.window_left = window_left;
  c.scale = scale; c.out = out; c.out_dtype = out_dtype; c.out_stride = out_seq_stride; c.lse_out = lse_out;
  c.workspace = workspace; c.status = status;
  return stream_cache("sbk_swa_decode_q8", c, (cudaStream_t)stream);
}
