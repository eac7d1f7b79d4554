// Launch parameters of the tensor-core chunk attention over 8-bit pages (chunk_q8_tc.cu).
#pragma once

#include "q8.cuh"

namespace bpkv {

struct ChunkQ8Params {
  const void* q;
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  const int32_t* bt;
  const int32_t* cu_q;  // null: request b has the one query row b
  const int32_t* lens;
  void* out;
  float* lse_out;
  float* part_o;    // [parts][total_q * Hq][D]
  float* part_lse;  // [parts][total_q * Hq]
  // How the row tiles are cut into pieces, a CTA per piece and KV head, longest row tile first (in a batch if
  // `ranked`: each CTA works the order out): `whole` row tiles whole, the others in `shares` shares of their tokens
  // each.  Or (pieces not null) planned on the device from the lengths: pieces[i] = (row tile or -1,
  // share | shares << 16), and n_shares of each row tile.
  int2* pieces;       // [n_pieces]
  int32_t* n_shares;  // [B * tiles]
  int whole, shares, n_pieces, ranked, max_shares, sms;
  int B, Hq, Hkv, n_rep, tiles, alt, causal, max_blocks, num_pages, total_q;
  int64_t q_st, q_sh, page_stride, scale_stride, bt_sb;
  float scale_log2;
  float empty;  // value of a row that sees no token
};

constexpr int kMaxRanked = 512;  // row tiles that can be put in order
constexpr int kMaxParts = 64;     // of a row; a multiple of 32
// head_dim 64 or 128, softmax scale > 0.
int chunk_q8_tc_launch(const ChunkQ8Params& p, int head_dim, int dtype, cudaStream_t st);

}  // namespace bpkv
