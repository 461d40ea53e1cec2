// Interface between the entry points of the attention over the 8-bit cache: the kernel that streams the cache once per
// sequence serves single query tokens (sbk_swa_decode_q8) and runs of a few (sbk_swa_prefill_q8).
#pragma once

#include "sbk_common.cuh"

namespace sbk {
namespace decode_q8 {

// tokens that a row of the block table may span: positions, and what is added to them, are 32-bit numbers
constexpr int64_t kMaxWidth = (int64_t)1 << 30;

struct Call {
  const void* q; int64_t q_stride;                       // elements between rows
  const void* k_cache; const void* v_cache; const void* k_scale; const void* v_scale;
  int64_t cache_block_stride, scale_block_stride;
  const int32_t* block_tables; int max_blocks;
  const int32_t* seq_lens;                               // single tokens: lengths [n_seqs]; NULL: runs, and
  const int32_t* query_start_loc; const int32_t* context_lens; int max_query_len;
  int n_seqs, H, kvh; int64_t num_blocks; int block_size, window_left; float scale;
  void* out; int out_dtype; int64_t out_stride; float* lse_out;
  void* workspace; int32_t* status;
};
size_t workspace_bytes(int H, bool runs);
int device_sms();                                        // multiprocessors of the current device
int stream_cache(const char* who, const Call& c, cudaStream_t st);

}  // namespace decode_q8
}  // namespace sbk
