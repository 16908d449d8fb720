// The decode kernels over a list of work items made elsewhere (segment_attn.cu), and what a planner of such a list
// has to know about them.  Implemented in decode_attn.cu.
#pragma once
#include <cuda_runtime.h>

#include "decode_plan.hpp"

namespace pkv {

struct DecodeList {
  const void *q, *k_cache, *v_cache;
  const int *block_tables, *table_offset, *token_seq, *token_pos;   // token_pos: for the cluster form only
  void* out;
  int n_tokens, q_heads, kv_heads, head_dim, block_size;
  float scale;
  const PlanHeader* header;
  int stamp, cluster_stamp;    // what the header must show
  const WorkItem* items;
  int n_items;
  float *part_ml, *part_acc;
  unsigned long long pool_rows;
  unsigned int* host_err;
  bool behind_tiles;           // the launch before this one is the tile kernel of the same call (DecodeArgs::wait_last)
  int cluster, cluster_least;  // > 0: the cluster form, if the device takes it
};

// *merged: the cluster form ran; there are no partials to merge.
template <typename T> int decode_listed(const DecodeList& l, cudaStream_t stream, bool* merged);
// Whether the partials' maxima are in base-2 units.
template <typename T> bool decode_log2_domain(int q_heads, int kv_heads, int head_dim, int block_size, float scale);

int decode_sms();
int decode_max_extra(int kv_heads);
PlanLimits decode_plan_limits(int extra, int q_heads, int kv_heads, int head_dim);
// Blocks per cluster for a step whose every (token, kv head) gets a cluster (0: none), and the fewest that will do.
int decode_cluster_size(int n_tokens, int longest, int q_heads, int kv_heads, int head_dim, int* least);

}  // namespace pkv
