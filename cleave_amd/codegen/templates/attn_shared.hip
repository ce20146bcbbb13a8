// ---- decode attention of a batch whose requests begin with the same pages ----------------------------------
//
// A request's keys are the shared pages', then its own.  Softmax weights of any part of the keys add up with those of the others once
// each part carries its reference point and its sum, so a call is two kinds of work and a sum:
//   shared keys  read once for the whole batch: the queries of all requests are the rows of one matrix product per kv head
//                (pl_prefix_part, attn_prefill_lds.hip: 128 rows a workgroup, key tiles through LDS);
//   own keys     read by their request alone (att_own_part, attn_decode.hip: registers, nothing through LDS on the way in);
//   partials     of `prefix_ranges` ranges of the shared keys (request, range, query head[, d]) and, behind them, of items of
//                `own_chunk` entries of the requests' own table (item, query head[, d]), f32, merged by attn_combine.hip.
// Partials are f32; weights are rounded to the element type for either kind's value product, as the matrix cores take it, and summed before.
// Read by every request for itself, the shared keys would be `batch` times the traffic.
//
// One launch holds both kinds: the first part is bound by the matrix cores or L2, the second by HBM, and their workgroups run beside
// each other.
// 32 / 8 heads of 128, pages of 64, us with the sum of the partials (6 and 11 of them): f16, 64 requests of up to 1024 own keys behind
// 8192 43.5; bf16, 200 of 700 behind 32768 160, where the shared keys alone take 119 (0.98 PFLOP/s) and the own ones 50 (5.7
// TB/s).  A step of shared keys takes 0.62 us alone on a compute unit, 0.52 in pairs and 0.8 to 0.9 beside own keys; with all
// keys out of L2 the second call's launch takes 139.
//   run-time: batch, num_pages, n_shared (shared pages), n_idx (own table length), prefix_ranges, own_chunk, sm_scale
extern "C" __global__ void __launch_bounds__(256, 2)
CL_PARTIAL_NAME(CL_PARTIAL_PARAMS) {
  const int row_tiles = (batch * PL_GROUP + PL_ROWS - 1) / PL_ROWS;
  const int prefix_blocks = (CL_KV_HEADS * prefix_ranges + 7) / 8 * 8 * row_tiles;
  if ((int)blockIdx.x < prefix_blocks) pl_prefix_part(CL_PARTIAL_ARGS, blockIdx.x);
  else att_own_part(CL_PARTIAL_ARGS, blockIdx.x - prefix_blocks);
}
