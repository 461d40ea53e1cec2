// Sliding-window attention of one query token per sequence over the 8-bit paged K/V cache (format: kv_q8.cuh):
//     s_j = scale * 2^ek_j * sum_d q_d ck_jd      o = sum_j softmax(s)_j * 2^ev_j * cv_jd      lse = log sum_j exp(s_j)
// over the visible tokens j of a sequence, ck / cv being the e4m3 codes and ek / ev the exponents of a row.
//
// Bound by HBM: 2 kvh (D + 1) bytes per visible token, at 14 flops a byte.
//
// Products. The codes go into the tensor cores as they are stored (mma.sync m16n8k32, e4m3 x e4m3, exact products and
//   fp32 sums: measured, no product is cut). The other operand is made 8-bit without losing bits: a bf16 number is the sum of two
//   e4m3 numbers of four significant bits each, and a kv group has at most eight query heads, so the sixteen rows of the MMA are
//   the upper parts of eight heads and their remainders:
//       S[2 x 8, tokens] = [q_hi; q_lo] . K^T        O[2 x 8, dims] = [p_hi; 16 p_lo] . V
//   and one thread holds both rows of a head. q is scaled by the power of two that takes its largest value under 448; elements far
//   below it lose what lies under 2^-18 of that value. The padding of the group to eight heads is the only work beyond the formula.
//   Converting K and V to 16 bits instead would be two thirds of the kernel's instructions.
// Softmax. The V scale belongs to the probability's exponent: with m the running maximum of s, the normaliser sums 2^(s_j - m) and
//   the product takes w_j = 2^(s_j - m + ev_j - r + 8), r the running maximum of s_j - m + ev_j: w <= 256, and its two 4-bit parts
//   reach down to 2^-13. At the end O * 2^(r - 8) / l.
// Fragments. Column n of a score tile may be any token, as long as the rows of V come in the order of the probabilities' fragment:
//   thread t of a quad takes tokens 4t ... 4t+3 of every sixteen, which makes the probabilities the A operand of the second
//   product without any exchange, the scale bytes of a thread one 32-bit word, and all shared-memory reads conflict-free (eight
//   rows of a read lie in eight different 16-byte columns of the 128-byte swizzle).
// Data movement. One producer warp walks the block table and issues a TMA tensor copy per 16 tokens (kvh * 2 KiB of K, the same of V)
//   and sixteen 16-byte bulk copies of exponents per stage, into a ring of three 32.25 KiB stages; two CTAs per SM. A stage holds 32
//   tokens per consumer warp: warp w serves kv head w % kvh and the 32-token part w / kvh.
// Partition. The units (one stage of tokens each) of all sequences, laid end to end with a fixed charge per sequence, are cut
//   into one equal run per CTA. Only the first and the last sequence of a run can be cut, so a CTA writes at most two partial results
//   (m, l, O): the workspace is indexed by CTA, holds nothing between calls and needs no clearing. A second kernel, launched
//   ahead of the first one's end (programmatic dependent launch), folds the partials: no counters, no waits between CTAs.
#include "kv_q8.cuh"
#include "sbk_tma.cuh"

namespace sbk {
namespace decode_q8 {

constexpr int kD = 128, kChunk = 16, kMaxG = 8;
constexpr int kConsumerWarps = 4, kThreads = 32 * (kConsumerWarps + 1), kConsumers = 32 * kConsumerWarps;
constexpr int kMaxSeqs = 1024;        // sequences per launch (lengths and prefix in shared memory)
constexpr int kMaxCtas = 320;         // two per SM, as many as the workspace is laid out for
constexpr int kItemCost = 8;          // what starting and finishing a sequence is charged, in units
constexpr int kMinRun = 1;            // shortest run of a CTA, in units
constexpr int kStages = 3;
constexpr int kTileBytes = 16384;     // K, or V, of a stage
constexpr int kScaleBytes = 256;      // exponents of a stage: 128 of K, 128 of V
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kHeadStride = 132;      // floats per head row of the merge scratch (bank skew)
constexpr int kMergeWarpBytes = kMaxG * kHeadStride * 4 + 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kNegBig = -1.0e30f;
enum : int { kFirst = 1, kLast = 2, kBad = 4, kEnd = 8 };

struct StageInfo { int b, tok_base, lo, hi, flags, part; };   // part: partial slot of the item's result, or -1 (direct)

constexpr int kScaleOff = kStages * kStageBytes;
constexpr int kInfoOff = kScaleOff + kStages * kScaleBytes;
constexpr int kPreOff = kInfoOff + ((kStages * (int)sizeof(StageInfo) + 15) / 16) * 16;
constexpr int kLensOff = kPreOff + (kMaxSeqs + 4) * 4;
constexpr int kBarOff = kLensOff + kMaxSeqs * 4;
constexpr int kMiscOff = kBarOff + 2 * kStages * 8;
constexpr int kSmemBytes = kMiscOff + 48 + 1024;      // + slack to align the ring to 1 KiB
static_assert(kSmemBytes <= 115200, "two CTAs must fit one SM");
static_assert(kConsumerWarps * kMergeWarpBytes <= kStageBytes, "the merge scratch lives inside one stage");

struct Params {
  const __nv_bfloat16* q; int64_t q_stride;
  const uint8_t* k_scale; const uint8_t* v_scale; int64_t scale_block_stride;
  const int32_t* block_tables; int max_blocks; const int32_t* seq_lens;
  int B, H; int64_t num_blocks; int block_size, window_left; float scale_log2;
  void* out; int64_t out_stride; float* lse_out;
  int2* cut;            // [grid]: the sequence that begins in this CTA's run and goes on in the next ones, and its pieces (0: none)
  float* ws_o; float2* ws_ml;   // partials [2 * CTA + slot][H][D] and [..][H]: slot 0 a sequence that began before, 1 one that goes on
  int32_t* status; int tile_copy;
};

struct Span { int first, units; };    // units [first, first + units) of the token axis hold the visible tokens
template <int UNIT>
__device__ __forceinline__ Span span_of(int L, int window_left) {
  Span s;
  if (L <= 0) { s.first = 0; s.units = 0; return s; }
  s.first = first_visible(L, 1, window_left) / UNIT;
  s.units = (L - 1) / UNIT - s.first + 1;
  return s;
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two 16 x 16 byte matrices, transposed: lane 4g + t gets column g (r0) and g + 8 (r1) of the first, rows 4t ... 4t+3, and the
// same of the second (r2, r3); lanes 0-15 name the rows of the first matrix, 16-31 those of the second
__device__ __forceinline__ void ldmatrix_b8_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void consumer_bar() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory"); }

// four floats -> codes of their upper parts and of their remainders * up
__device__ __forceinline__ void split4(float a, float b, float c, float d, float up, uint32_t& hi, uint32_t& lo) {
  const uint32_t h0 = q8::pack_e4m3x2(a, b), h1 = q8::pack_e4m3x2(c, d);
  const float2 f0 = q8::e4m3x2_to_float2(h0), f1 = q8::e4m3x2_to_float2(h1);
  hi = h0 | (h1 << 16);
  lo = q8::pack_e4m3x2((a - f0.x) * up, (b - f0.y) * up) | (q8::pack_e4m3x2((c - f1.x) * up, (d - f1.y) * up) << 16);
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

template <int KVH, typename TO>
__global__ void __launch_bounds__(kThreads, 2)
decode_kernel(const Params P, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  constexpr int kSub = kConsumerWarps / KVH;          // 32-token parts of a stage
  constexpr int kUnit = 32 * kSub;                    // tokens of a stage
  constexpr int kChunks = kUnit / kChunk;             // 16-token chunks of a stage
  constexpr int kChunkBytes = KVH * kChunk * kD;      // one chunk of K or of V: [head][token][128 B]
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t ring = smem_u32(smem);
  StageInfo* info = reinterpret_cast<StageInfo*>(smem + kInfoOff);
  int* pre = reinterpret_cast<int*>(smem + kPreOff);
  int* lens = reinterpret_cast<int*>(smem + kLensOff);
  const uint32_t bar_full = ring + kBarOff, bar_empty = bar_full + 8 * kStages;
  volatile int* misc = reinterpret_cast<volatile int*>(smem + kMiscOff);   // [0] abort, [1] longest, [2..6] scan
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // the folding kernel may be set up while this one runs (it waits for this one's end before it reads anything)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, kConsumerWarps);
    }
    misc[0] = 0;
    misc[1] = 0;
    pre[0] = 0;
    fence_mbar_init();
  }
  __syncthreads();
  // ---- what every sequence costs, as an exclusive prefix: units of b occupy [pre[b], pre[b] + units), its charge follows ----
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
        int L = P.seq_lens[b];
        const int64_t width = (int64_t)P.max_blocks * P.block_size;
        if (L > width) {                   // tokens that the table has no entry for
          L = (int)width;
          if (blockIdx.x == 0) raise_status(P.status, SBK_ST_BAD_BLOCK);
        }
        lens[b] = L;
        c = L > 0 ? span_of<kUnit>(L, P.window_left).units : 1;   // an empty sequence keeps one: somebody writes its zeros
        mx = max(mx, c);
        c += kItemCost;
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
  if (per < kMinRun) per = kMinRun;
  // A batch of near-equal sequences that fills the CTAs evenly streams fastest as whole sequences: no partials to write and fold.
  const int rounds = (P.B + n_cta - 1) / n_cta;
  const bool whole = 2 * P.B >= n_cta && (P.B <= n_cta || 10 * rounds * n_cta <= 11 * P.B) &&
                     (int64_t)misc[1] * P.B <= ((int64_t)total - (int64_t)kItemCost * P.B) / 8 * 9;

  if (warp == kConsumerWarps) {
    // ================================= producer =================================
    int it = 0;
    bool aborted = false;
    auto stream_item = [&](int b, int unit0, int n_units, int part) {
      const int L = lens[b];
      const int t0 = first_visible(L, 1, P.window_left);
      const int32_t* table = P.block_tables + (int64_t)b * P.max_blocks;
      int64_t pb_lane = -1;            // physical block of chunk (batch0 + lane): one table read per 32 chunks
      int batch0 = 0;
      const int n = n_units > 0 ? n_units : 1;
      for (int j = 0; j < n; ++j, ++it) {
        const int c0 = (unit0 + j) * kChunks;
        if (n_units > 0 && (j == 0 || c0 + kChunks > batch0 + 32)) {
          batch0 = c0;
          const int lb = (c0 + lane) * kChunk / P.block_size;
          pb_lane = (c0 + lane) * kChunk < L && lb < P.max_blocks ? (int64_t)table[lb] : -1;
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
        int hi = base + kUnit < L ? base + kUnit : L;
        if (n_units == 0 || hi < lo) hi = lo;
        // chunks of this stage that hold visible tokens: [ca, cb)
        const int ca = (lo - base) / kChunk, cb = hi > lo ? (hi - 1 - base) / kChunk + 1 : ca;
        // lanes 0-15: exponents (chunk, head) of K and of V, 16 bytes each; lanes 16-31: the tiles
        const int x = lane & 15;
        const bool is_tile = lane >= 16;
        const int c = is_tile ? x % kChunks : x / KVH % kChunks;
        // every lane reads its chunk's block; what it issues is decided below
        int src = c0 + c - batch0;
        src = src < 0 ? 0 : (src > 31 ? 31 : src);
        const int64_t pb = __shfl_sync(0xffffffffu, pb_lane, src);
        const bool in = c >= ca && c < cb;
        const bool bad = __any_sync(0xffffffffu, in && (pb < 0 || pb >= P.num_blocks));
        if (lane == 0) {
          StageInfo si;
          si.b = b; si.tok_base = base; si.lo = lo; si.hi = hi; si.part = part;
          si.flags = (j == 0 ? kFirst : 0) | (j == n - 1 ? kLast : 0) | (bad ? kBad : 0);
          info[s] = si;
          if (bad) raise_status(P.status, SBK_ST_BAD_BLOCK);
          mbar_arrive_expect_tx(bar_full + 8 * s, bad ? 0u : (uint32_t)(cb - ca) * 2u * (kChunkBytes + KVH * kChunk));
        }
        __syncwarp();
        if (!bad && in) {
          const int tin = (base + c * kChunk) % P.block_size;
          const uint32_t bar = bar_full + 8 * s;
          if (!is_tile) {
            const int h = x % KVH;
            const int64_t at = pb * P.scale_block_stride + (int64_t)h * P.block_size + tin;
            const uint32_t dst = ring + kScaleOff + s * kScaleBytes + (((c >> 1) * KVH + h) * 2 + (c & 1)) * 16;
            if (x < kChunks * KVH) {
              bulk_g2s(dst, P.k_scale + at, 16, bar);
              bulk_g2s(dst + 128, P.v_scale + at, 16, bar);
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
      }
    };

    int2 cut = make_int2(-1, 0);
    if (whole) {
      if (lane == 0) P.cut[me] = cut;
      for (int b = me; b < P.B && !aborted; b += n_cta) {
        const Span sp = span_of<kUnit>(lens[b], P.window_left);
        stream_item(b, sp.first, sp.units, -1);
      }
    } else {
      const int64_t g0 = (int64_t)me * per;
      const int64_t g1 = g0 + per < total ? g0 + per : total;
      int b0 = 0;
      if (g0 < total) {
        int hi_b = P.B;                 // largest b with pre[b] <= g0
        while (hi_b - b0 > 1) {
          const int mid = (b0 + hi_b) >> 1;
          if (pre[mid] <= g0) b0 = mid; else hi_b = mid;
        }
        // the sequence that holds the run's last slot: does it begin here and go on?
        int e = b0, he = P.B;
        while (he - e > 1) {
          const int mid = (e + he) >> 1;
          if (pre[mid] <= g1 - 1) e = mid; else he = mid;
        }
        const int cr = lens[e] > 0 ? span_of<kUnit>(lens[e], P.window_left).units : 1;
        if (pre[e] >= g0 && pre[e] + cr > g1) cut = make_int2(e, (pre[e] + cr - 1) / per - me + 1);
      }
      if (lane == 0) P.cut[me] = cut;
      if (g0 < total) {
        for (int b = b0; b < P.B && pre[b] < g1 && !aborted; ++b) {
          const Span sp = span_of<kUnit>(lens[b], P.window_left);
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
        if (lane == 0) {
          info[s].flags = kEnd;
          mbar_arrive_expect_tx(bar_full + 8 * s, 0u);
        }
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
  const int hk = warp % KVH, sub = warp / KVH, G = P.H / KVH;
  const int g = lane >> 2, t = lane & 3;
  const bool head_ok = g < G;
  TO* const out = reinterpret_cast<TO*>(P.out);

  // Rows of a [16 tokens][128 B] tile, 16-byte column c of token r at r * 128 + ((c ^ (r & 7)) << 4).
  // K: lane 8i + n names token tau(tile, n) and column i (+ 4): tile 0 takes tokens 0 1 4 5 10 11 14 15, tile 1 the others
  const int n8 = lane & 7, i4 = lane >> 3;
  const int tok0 = 4 * (n8 >> 1) + ((n8 >> 1) & 2) + (n8 & 1), tok1 = tok0 ^ 2;
  // V: lane r names row kappa = r & 15 of the product, token 4 (kappa / 4) + ..., of the first or second sixteen
  const int kap = lane & 15;
  const int tokv = 4 * (kap >> 2) + ((((kap >> 1) & 1) ? 2 : 0) ^ ((kap >> 2) & 2)) + (kap & 1);
  const uint32_t tile0 = (uint32_t)(sub * 2 * kChunkBytes + hk * 2048);        // this warp's first sixteen tokens, its head
  const uint32_t k0 = tile0 + tok0 * 128, k1 = tile0 + tok1 * 128;
  const uint32_t v0 = kTileBytes + tile0 + (lane >> 4) * kChunkBytes + tokv * 128;
  const int pa = 4 * t + (t & 2), pb = pa ^ 2;     // a thread's tokens in score tile 0 (pa, pa + 1) and tile 1 (pb, pb + 1)
  const int sh = t & 2 ? 16 : 0;                   // bit position of tile 0's pair in the thread's word of exponents

  uint32_t qf[4][4];
  float acc[16][4];
  float m = -INFINITY, l = 0.f, r = -INFINITY, qs = 0.f;
  for (int it = 0;; ++it) {
    const int s = it % kStages;
    if (!mbar_wait_bounded(bar_full + 8 * s, (it / kStages) & 1)) {
      if (lane == 0) { raise_status(P.status, SBK_ST_WAIT_TIMEOUT); misc[0] = 1; }
      return;
    }
    const StageInfo si = info[s];
    if (si.flags & kEnd) return;
    const uint32_t stage = ring + s * kStageBytes;

    if (si.flags & kFirst) {
      // q of head g, dims 32 kk + 4t ... + 3 and 32 kk + 16 + 4t ... + 3
      const __nv_bfloat16* qp = P.q + (int64_t)si.b * P.q_stride + (int64_t)(hk * G + (head_ok ? g : 0)) * kD + 4 * t;
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[2 * i] = *reinterpret_cast<const uint32_t*>(qp + 16 * i);
        w[2 * i + 1] = *reinterpret_cast<const uint32_t*>(qp + 16 * i + 2);
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
      const float inv = q8::pow2i(-e);
      qs = P.scale_log2 * q8::pow2i(e);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x[4] = {__uint_as_float(w[2 * i] << 16), __uint_as_float(w[2 * i] & 0xffff0000u),
                      __uint_as_float(w[2 * i + 1] << 16), __uint_as_float(w[2 * i + 1] & 0xffff0000u)};
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = q8::finite(x[j]) ? x[j] * inv : __uint_as_float(0x7fffffffu);
        split4(x[0], x[1], x[2], x[3], 1.f, qf[i >> 1][2 * (i & 1)], qf[i >> 1][2 * (i & 1) + 1]);
      }
#pragma unroll
      for (int nt = 0; nt < 16; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
      m = r = -INFINITY;
      l = 0.f;
    }

    const int tb = si.tok_base + 32 * sub;                      // my 32 tokens
    const int vlo = si.lo > tb ? si.lo : tb, vhi = si.hi < tb + 32 ? si.hi : tb + 32;
    if (!(si.flags & kBad) && vhi > vlo) {
      const bool ragged = vlo > tb || vhi < tb + 32;
      if (ragged) {
        // rows outside the visible range hold anything, or older data: a zero probability must not meet a NaN code
        for (int r = lane >> 3; r < 32; r += 4)
          if (tb + r < vlo || tb + r >= vhi)
            *reinterpret_cast<uint4*>(smem + s * kStageBytes + kTileBytes + tile0 + (r >> 4) * kChunkBytes + (r & 15) * 128 +
                                      (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
        __syncwarp();
      }
      // ---- scores of 32 tokens: tiles 0, 1 of the first sixteen, 2, 3 of the second ----
      float sc[8];                                              // [16-token half][tile][pair]
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          uint32_t b[4];
          ldmatrix_x4(b, stage + h * kChunkBytes + k0 + (((4 * f + i4) ^ (tok0 & 7)) << 4));
          mma_e4m3(c0, qf[2 * f], b[0], b[1]);
          mma_e4m3(c0, qf[2 * f + 1], b[2], b[3]);
          ldmatrix_x4(b, stage + h * kChunkBytes + k1 + (((4 * f + i4) ^ (tok1 & 7)) << 4));
          mma_e4m3(c1, qf[2 * f], b[0], b[1]);
          mma_e4m3(c1, qf[2 * f + 1], b[2], b[3]);
        }
        sc[4 * h] = c0[0] + c0[2]; sc[4 * h + 1] = c0[1] + c0[3];
        sc[4 * h + 2] = c1[0] + c1[2]; sc[4 * h + 3] = c1[1] + c1[3];
      }
      float ev[8];
      {
        const uint8_t* se = smem + kScaleOff + s * kScaleBytes + (sub * KVH + hk) * 32 + 4 * t;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t kb = *reinterpret_cast<const uint32_t*>(se + 16 * h);
          const uint32_t vb = *reinterpret_cast<const uint32_t*>(se + 128 + 16 * h);
          const uint32_t kw[2] = {kb >> sh, kb >> (16 - sh)}, vw[2] = {vb >> sh, vb >> (16 - sh)};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sc[4 * h + 2 * i] *= qs * __uint_as_float((kw[i] & 255u) << 23);
            sc[4 * h + 2 * i + 1] *= qs * __uint_as_float((kw[i] & 0xff00u) << 15);
            // byte - 127, through the low bits of a float: 2^23 + byte
            ev[4 * h + 2 * i] = __uint_as_float(0x4b000000u | (vw[i] & 255u)) - 8388735.f;
            ev[4 * h + 2 * i + 1] = __uint_as_float(0x4b000000u | ((vw[i] >> 8) & 255u)) - 8388735.f;
          }
        }
      }
      if (ragged) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = tb + 16 * h + (i < 2 ? pa : pb) + (i & 1);
            if (tok < vlo || tok >= vhi) { sc[4 * h + i] = -INFINITY; ev[4 * h + i] = 0.f; }
          }
      }
      // ---- running maxima: m of s, and r of (s - m) + ev, which moves with m (s + ev itself would lose ev beside a large s) ----
      float mx = sc[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i]);
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      const float mn = fmaxf(m, mx), ms = fmaxf(mn, kNegBig);
      const float back = m - ms;
      const float al = fast_exp2(back);
      m = mn;
      float w[8], mx2 = -INFINITY, ls = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = sc[i] - ms;
        w[i] = d + ev[i];
        mx2 = fmaxf(mx2, w[i]);
        ls += fast_exp2(d);
      }
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) mx2 = fmaxf(mx2, __shfl_xor_sync(0xffffffffu, mx2, off));
      const float ro = r + back, rn = fmaxf(fmaxf(ro, mx2), kNegBig);
      const float al2 = fast_exp2(ro - rn);
      r = rn;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = fast_exp2(w[i] - (rn - 8.f));
      l = l * al + ls;
      if (__any_sync(0xffffffffu, al2 != 1.f)) {
#pragma unroll
        for (int nt = 0; nt < 16; ++nt) { acc[nt][0] *= al2; acc[nt][1] *= al2; acc[nt][2] *= al2; acc[nt][3] *= al2; }
      }
      uint32_t pf[4];
      split4(w[0], w[1], w[2], w[3], 16.f, pf[0], pf[1]);
      split4(w[4], w[5], w[6], w[7], 16.f, pf[2], pf[3]);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t b[4];
        ldmatrix_b8_trans(b, stage + v0 + ((c ^ (tokv & 7)) << 4));
        mma_e4m3(acc[2 * c], pf, b[0], b[2]);
        mma_e4m3(acc[2 * c + 1], pf, b[1], b[3]);
      }
      if (ragged) fence_proxy_async_smem();   // my zero fill precedes the next copy into these rows
    }
    __syncwarp();
    const bool keep_stage = kSub > 1 && (si.flags & kLast);     // becomes the merge scratch first
    if (lane == 0 && !keep_stage) mbar_arrive(bar_empty + 8 * s);
    if (!(si.flags & kLast)) continue;

    // ================= end of an item: its output row, or its partial =================
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    // O relative to m (0 where nothing was visible; a NaN score has made O and l NaN already)
    const float fix = r > kNegBig ? exp2f(r - 8.f) : 0.f;
    const int64_t prow = (int64_t)(2 * me + (si.part > 0 ? 1 : 0)) * P.H;
    if constexpr (kSub == 1) {
      if (head_ok) {
        const int h = hk * G + g;
        if (si.part < 0) {
          const float f = fix * inverse(l);
          TO* op = out + (int64_t)si.b * P.out_stride + (int64_t)h * kD + 2 * t;
#pragma unroll
          for (int nt = 0; nt < 16; ++nt)
            store2(op + 8 * nt, (acc[nt][0] + acc[nt][2] * 0.0625f) * f, (acc[nt][1] + acc[nt][3] * 0.0625f) * f);
          if (P.lse_out && t == 0) P.lse_out[(int64_t)si.b * P.H + h] = row_lse(m, l);
        } else {
          float* wp = P.ws_o + (prow + h) * kD + 2 * t;
#pragma unroll
          for (int nt = 0; nt < 16; ++nt)
            *reinterpret_cast<float2*>(wp + 8 * nt) =
                make_float2((acc[nt][0] + acc[nt][2] * 0.0625f) * fix, (acc[nt][1] + acc[nt][3] * 0.0625f) * fix);
          if (t == 0) P.ws_ml[prow + h] = make_float2(m, l);
        }
      }
    } else {
      // several warps share a kv head (each took other tokens): merge through the stage just consumed
      uint8_t* mbuf = smem + s * kStageBytes;
      float* wo = reinterpret_cast<float*>(mbuf + warp * kMergeWarpBytes);
      float* wml = wo + kMaxG * kHeadStride;
      consumer_bar();                       // every warp is done reading this stage
#pragma unroll
      for (int nt = 0; nt < 16; ++nt)
        *reinterpret_cast<float2*>(wo + g * kHeadStride + 8 * nt + 2 * t) =
            make_float2((acc[nt][0] + acc[nt][2] * 0.0625f) * fix, (acc[nt][1] + acc[nt][3] * 0.0625f) * fix);
      if (t == 0) { wml[g] = m; wml[8 + g] = l; }
      consumer_bar();
      for (int h = warp; h < P.H; h += kConsumerWarps) {
        const int kh = h / G, r = h - kh * G;
        float M = -INFINITY;
#pragma unroll
        for (int w2 = 0; w2 < kSub; ++w2)
          M = fmaxf(M, reinterpret_cast<const float*>(mbuf + (kh + KVH * w2) * kMergeWarpBytes)[kMaxG * kHeadStride + r]);
        const float Ms = fmaxf(M, kNegBig);
        float L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w2 = 0; w2 < kSub; ++w2) {
          const float* po = reinterpret_cast<const float*>(mbuf + (kh + KVH * w2) * kMergeWarpBytes);
          const float wgt = fast_exp2(po[kMaxG * kHeadStride + r] - Ms);
          const float4 o = *reinterpret_cast<const float4*>(po + r * kHeadStride + 4 * lane);
          L += po[kMaxG * kHeadStride + 8 + r] * wgt;
          O.x += o.x * wgt; O.y += o.y * wgt; O.z += o.z * wgt; O.w += o.w * wgt;
        }
        if (si.part < 0) {
          const float f = inverse(L);
          store4(out + (int64_t)si.b * P.out_stride + (int64_t)h * kD + 4 * lane,
                 make_float4(O.x * f, O.y * f, O.z * f, O.w * f));
          if (P.lse_out && lane == 0) P.lse_out[(int64_t)si.b * P.H + h] = row_lse(M, L);
        } else {
          *reinterpret_cast<float4*>(P.ws_o + (prow + h) * kD + 4 * lane) = O;
          if (lane == 0) P.ws_ml[prow + h] = make_float2(M, L);
        }
      }
      fence_proxy_async_smem();             // these writes precede the copies that refill the stage
      consumer_bar();
      if (lane == 0) mbar_arrive(bar_empty + 8 * s);
    }
  }
}

// Folds the partials of the sequence that begins in CTA c's run and goes on: one block per (c, four heads), four warps per
// head, each taking every fourth piece with its loads issued eight at a time.
constexpr int kFoldThreads = 512;
template <typename TO>
__global__ void __launch_bounds__(kFoldThreads) fold_kernel(const Params P) {
  __shared__ float part[16][32][6];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const int2 cut = P.cut[c];
  if (cut.y <= 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y * 4 + (warp >> 2), w = warp & 3;
  const bool on = h < P.H;
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kU = 8;
  for (int i0 = w; on && i0 < cut.y; i0 += 4 * kU) {
    float2 ml[kU];
    float4 o[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = i0 + 4 * u < cut.y ? i0 + 4 * u : i0;
      const int64_t row = (int64_t)(2 * (c + i) + (i == 0 ? 1 : 0)) * P.H + h;
      ml[u] = __ldcg(P.ws_ml + row);
      o[u] = __ldcg(reinterpret_cast<const float4*>(P.ws_o + row * kD) + lane);
      if (i0 + 4 * u >= cut.y) ml[u] = make_float2(-INFINITY, 0.f);
    }
    float Mn = M;
#pragma unroll
    for (int u = 0; u < kU; ++u) Mn = fmaxf(Mn, ml[u].x);
    const float Ms = fmaxf(Mn, kNegBig), resc = fast_exp2(M - Ms);
    L *= resc; O.x *= resc; O.y *= resc; O.z *= resc; O.w *= resc;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (i0 + 4 * u >= cut.y) break;
      const float wgt = fast_exp2(ml[u].x - Ms);
      L += ml[u].y * wgt;
      O.x += o[u].x * wgt; O.y += o[u].y * wgt; O.z += o[u].z * wgt; O.w += o[u].w * wgt;
    }
    M = Mn;
  }
  float* mine = part[warp][lane];
  mine[0] = M; mine[1] = L; mine[2] = O.x; mine[3] = O.y; mine[4] = O.z; mine[5] = O.w;
  __syncthreads();
  if (w != 0 || !on) return;
  float Mt = -INFINITY;
#pragma unroll
  for (int q = 0; q < 4; ++q) Mt = fmaxf(Mt, part[warp + q][lane][0]);
  const float Ms = fmaxf(Mt, kNegBig);
  float Lt = 0.f;
  float4 Ot = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float* p = part[warp + q][lane];
    const float wgt = fast_exp2(p[0] - Ms);
    Lt += p[1] * wgt;
    Ot.x += p[2] * wgt; Ot.y += p[3] * wgt; Ot.z += p[4] * wgt; Ot.w += p[5] * wgt;
  }
  const float f = inverse(Lt);
  store4(reinterpret_cast<TO*>(P.out) + (int64_t)cut.x * P.out_stride + (int64_t)h * kD + 4 * lane,
         make_float4(Ot.x * f, Ot.y * f, Ot.z * f, Ot.w * f));
  if (P.lse_out && lane == 0) P.lse_out[(int64_t)cut.x * P.H + h] = row_lse(Mt, Lt);
}

static size_t cut_bytes() { return (size_t)kMaxCtas * sizeof(int2); }

template <int KVH, typename TO>
static int launch(const Params& P0, int B_total, int sms, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t st) {
  auto kern = decode_kernel<KVH, TO>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) {
      set_error("sbk_swa_decode_q8: cannot opt in to %d bytes of shared memory: %s", kSmemBytes, cudaGetErrorString(e));
      return SBK_E_LAUNCH;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  constexpr int kUnit = 32 * kConsumerWarps / KVH;
  const int n_ctas = 2 * sms < kMaxCtas ? 2 * sms : kMaxCtas;
  for (int b0 = 0; b0 < B_total; b0 += kMaxSeqs) {
    Params P = P0;
    P.B = B_total - b0 < kMaxSeqs ? B_total - b0 : kMaxSeqs;
    P.q = P0.q + (int64_t)b0 * P0.q_stride;
    P.block_tables = P0.block_tables + (int64_t)b0 * P0.max_blocks;
    P.seq_lens = P0.seq_lens + b0;
    P.out = (uint8_t*)P0.out + (int64_t)b0 * P0.out_stride * sizeof(TO);
    if (P0.lse_out) P.lse_out = P0.lse_out + (int64_t)b0 * P0.H;
    // no more CTAs than there can be units of work
    const int64_t width = (int64_t)P.max_blocks * P.block_size;
    const int64_t vis = P.window_left < 0 || width < (int64_t)P.window_left + 1 ? width : (int64_t)P.window_left + 1;
    const int64_t most = (int64_t)P.B * (vis / kUnit + 2 + kItemCost);
    int grid = (int)(most < n_ctas ? most : n_ctas);
    // a batch between one and two sequences per SM: one CTA each, so that every SM has work either way of cutting
    if (2 * P.B >= n_ctas && P.B < n_ctas) grid = P.B;
    kern<<<grid, kThreads, kSmemBytes, st>>>(P, map_k, map_v);
    int rc = check_launch("sbk_swa_decode_q8");
    if (rc != SBK_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, (P.H + 3) / 4);
    cfg.blockDim = dim3(kFoldThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, fold_kernel<TO>, P);
    if (e != cudaSuccess) {
      set_error("sbk_swa_decode_q8: launch of the folding kernel failed: %s", cudaGetErrorString(e));
      return SBK_E_LAUNCH;
    }
  }
  return SBK_OK;
}

}  // namespace decode_q8
}  // namespace sbk

extern "C" size_t sbk_swa_decode_q8_workspace_bytes(int B, int H, int D) {
  using namespace sbk::decode_q8;
  if (B <= 0 || H <= 0 || D <= 0) return 0;
  return cut_bytes() + (size_t)kMaxCtas * 2 * H * ((size_t)D + 2) * sizeof(float);
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
  const size_t need = sbk_swa_decode_q8_workspace_bytes(B, H, D);
  if (!workspace || workspace_bytes < need) {
    set_error("sbk_swa_decode_q8: workspace of %zu bytes given, %zu needed", workspace ? workspace_bytes : 0, need);
    return SBK_E_WORKSPACE;
  }
  if (!aligned16(workspace)) {
    set_error("sbk_swa_decode_q8: workspace must be 16-byte aligned");
    return SBK_E_ALIGN;
  }
  Params P = {};
  P.q = (const __nv_bfloat16*)q; P.q_stride = q_seq_stride;
  P.k_scale = (const uint8_t*)k_scale; P.v_scale = (const uint8_t*)v_scale; P.scale_block_stride = scale_block_stride_bytes;
  P.block_tables = block_tables; P.max_blocks = max_blocks; P.seq_lens = seq_lens;
  P.H = H; P.num_blocks = num_blocks; P.block_size = block_size; P.window_left = window_left;
  P.scale_log2 = scale * kLog2e; P.out = out; P.out_stride = out_seq_stride; P.lse_out = lse_out; P.status = status;
  P.cut = (int2*)workspace;
  P.ws_o = (float*)((uint8_t*)workspace + cut_bytes());
  P.ws_ml = (float2*)(P.ws_o + (size_t)kMaxCtas * 2 * H * D);
  static int sm_count[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  int sms = dev >= 0 && dev < 64 ? sm_count[dev] : 0;
  if (sms == 0) {
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (sms <= 0) sms = 148;
    if (dev >= 0 && dev < 64) sm_count[dev] = sms;
  }
  MapKey keys[2] = {MapKey{k_cache, kvh, num_blocks, block_size, cache_block_stride_bytes, kvh},
                    MapKey{v_cache, kvh, num_blocks, block_size, cache_block_stride_bytes, kvh}};
  for (MapKey& k : keys) { k.tok_stride = (int64_t)kvh * kD; k.rows = kvh; }
  CUtensorMap maps[2];
  if (!get_maps(maps, keys, 2, &P.tile_copy)) {
    set_error("sbk_swa_decode_q8: cuTensorMapEncodeTiled rejected the cache geometry (blocks=%lld block=%d kvh=%d)",
              (long long)num_blocks, block_size, kvh);
    return SBK_E_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
#define SBK_DECODE_Q8(TO)                                                 \
  switch (kvh) {                                                          \
    case 1: return launch<1, TO>(P, B, sms, maps[0], maps[1], st);        \
    case 2: return launch<2, TO>(P, B, sms, maps[0], maps[1], st);        \
    default: return launch<4, TO>(P, B, sms, maps[0], maps[1], st);       \
  }
  if (out_dtype == SBK_BF16) { SBK_DECODE_Q8(__nv_bfloat16) } else { SBK_DECODE_Q8(float) }
#undef SBK_DECODE_Q8
}
