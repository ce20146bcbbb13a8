// ---- causal prompts of a sliding window with sinks (GQA), key tiles shared through LDS -------------------
//
// Ragged queries; keys packed per request or through a token table.  The query at position p of a request sees its keys j with
// j <= p and (j > p - CL_WINDOW or j < CL_SINKS).  Tiles, images in LDS, operand reads, the skewed loop and the softmax (one pass,
// reference points raised only by weights that outgrow them) are those of attn_prefill_lds.hip: an item is 128 rows (PW_QT
// consecutive query tokens x the head group) of one request and kv head, four waves of 32 rows share every 32-key step of K and V.
//
// Scores, reference points, sums and outputs are f32.  Weights are rounded to the element type for the value product, as the matrix cores
// take it (half a step of a weight each, together at most about that of the result); their sum is taken before.
//
// Steps are numbered without the key tiles that no row of an item sees: step s is tile s of the request up to the sinks' last tile
// and tile s + skip behind it.  A step is masked in a wave where one of its rows sees a part of the tile: at the causal end
// (from n_full on) and where windows and sinks begin and end (before n_low).
//
// What bounds it: bf16, 32 / 8 heads, window 1024 + 4 sinks, six packed prompts of 31433 tokens 505 us, 0.95 PFLOP/s of what is seen: no
// one thing.  Without queries in and rows out 7 % less, without masks 7 %, without exponentials 10 %, without all of them 24 %;
// the matrix unit is busy 45 % of the time and the clock is at the power cap.  Workgroups that stay and ask for their next
// item's first tiles and queries ahead of their last one's stores were no faster (554 us against 551).
//
// `ranges` (a run-time argument) > 1, where a call has too few items for the chip: an item's steps in that many equal parts, each an
// item of its own that writes f32 partials (query token, range, query head[, d]) for attn_combine.hip.
//
// A masked key has weight 0, and 0 times a value that is not finite is not 0: a wave that meets such a value in a step that
// it masks takes its rows again at the end, key by key over what each sees.  Keys ahead of all the item's windows, whose cache rows
// may have been given away, are not read through a table.
//
//   CL_HEAD_DIM (64, 128, 256)  CL_KV_HEADS  CL_Q_HEADS (group divides 16)  CL_RAGGED  CL_WINDOW  CL_SINKS
//   run-time: batch, total_q, n_idx (table length / total_kv), num_pages (table form), ranges, sm_scale
#define PW_STEP 32
#define PW_GROUP (CL_Q_HEADS / CL_KV_HEADS)
#define PW_ROWS 128
#define PW_QT (PW_ROWS / PW_GROUP)            // query tokens per item
#define PW_PANELS (CL_HEAD_DIM / 64)
#define PW_PANEL (PW_STEP * 64)               // elements of one 64-feature panel
#define PW_IMG (PW_PANELS * PW_PANEL)         // elements of an image of K or V
#define PW_STAGES (CL_HEAD_DIM > 192 ? 4 : 3) // (the widest keys are read in two halves, the second out of an image still held)
#define PW_ALONE (PW_STAGES * 2 * PW_IMG * 4 > 163840)     // one workgroup of a compute unit: 512 registers a wave
#define PW_KJ (CL_HEAD_DIM / 32)
#define PW_FB (CL_HEAD_DIM / 16)
#define PW_UNITS (2 * PW_PANELS)              // 1 KiB loads per wave and step: its 8-key group of every panel of K and V
#define PW_SINK_STEPS ((CL_SINKS + PW_STEP - 1) / PW_STEP)
#define PW_PROW(it, m) ((((i64)(it).lo + (m) / PW_GROUP) * ranges + (it).split) * CL_Q_HEADS + (it).head * PW_GROUP + (m) % PW_GROUP)
static_assert(CL_Q_HEADS % CL_KV_HEADS == 0 && 16 % PW_GROUP == 0, "the head group divides the 16-row query tile");
static_assert(CL_HEAD_DIM % 64 == 0 && CL_HEAD_DIM <= 256 && CL_VDIM == CL_HEAD_DIM, "heads in whole 64-feature panels");

__shared__ __attribute__((aligned(1024))) elem_t pw_tiles[PW_STAGES * 2 * PW_IMG];
#if !CL_RAGGED
__shared__ __attribute__((aligned(256))) int pw_ids[2][4][64];   // table entries on their way in: [step parity][wave][lane]
#endif

struct PwItem {          // all of it the same in every lane
  int lo, n_rows;        // first query token, rows
  int head, split;
  int kv0, off;          // the request's first key; key position of query token 0 (off + token: that token's own key)
  int ext, skip;         // keys that the last row may see; tiles between the sinks' and the first window's
  int first_step, n_steps, first_key;     // this range's steps; the first window's first key
};
// The request of an item: a request has as many items as its query tokens fill, counted up over the requests, 64 of them at a time
// over the lanes of a wave.  (Items at the multiples of PW_QT packed tokens need no sum, but a request then has a part of one at either
// end: half an item more of each request; and its bits
// would depend on what is packed ahead of it.)
struct PwRequest { int q0, q1, kv0, kv1, first_item; };
CL_DEVICE int pw_running_sum(int x) {          // over the lanes of a wave, in order
#define PW_ADD_FROM(CTRL, ROWS) x += __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false)
  PW_ADD_FROM(0x111, 0xf);                     // of a row of 16 lanes, the lane 1, 2, 4 and 8 before
  PW_ADD_FROM(0x112, 0xf);
  PW_ADD_FROM(0x114, 0xf);
  PW_ADD_FROM(0x118, 0xf);
  PW_ADD_FROM(0x142, 0xa);                     // the last lane of rows 0 and 2 to the row behind each, of row 1 to rows 2 and 3
  PW_ADD_FROM(0x143, 0xc);
#undef PW_ADD_FROM
  return x;
}
CL_DEVICE PwRequest pw_find_request(const int* __restrict__ q_ptr, int batch, int total_q, const int* __restrict__ kv_ptr, int n_idx, int item, int lane) {
  PwRequest r = {0, 0, 0, 0, 0};               // (behind the last item: a request of nothing)
  int before = 0;
  for (int base = 0; base < batch; base += 64) {
    const int b = base + lane < batch ? base + lane : batch - 1;
    const int q0 = cl_clamp_ptr(q_ptr[b], total_q), q1 = cl_clamp_ptr(q_ptr[b + 1], total_q);
    const int kv0 = cl_clamp_ptr(kv_ptr[b], n_idx), kv1 = cl_clamp_ptr(kv_ptr[b + 1], n_idx);
    const int items = q1 > q0 && base + lane < batch ? (q1 - q0 + PW_QT - 1) / PW_QT : 0, sum = before + pw_running_sum(items);
    const unsigned long long reached = __builtin_amdgcn_ballot_w64(sum > item);
    if (reached) {
      const int l = __builtin_ctzll(reached);
      r.q0 = __builtin_amdgcn_readlane(q0, l);
      r.q1 = __builtin_amdgcn_readlane(q1, l);
      r.kv0 = __builtin_amdgcn_readlane(kv0, l);
      r.kv1 = __builtin_amdgcn_readlane(kv1, l);
      r.first_item = __builtin_amdgcn_readlane(sum - items, l);
      return r;
    }
    before = __builtin_amdgcn_readlane(sum, 63);
  }
  return r;
}
// the tile of step s
CL_DEVICE int pw_tile(const PwItem& it, int s) {
  s += it.first_step;
  return s >= PW_SINK_STEPS ? s + it.skip : s;
}
// output (and query) row of the item's row m, and the last key it may see
CL_DEVICE i64 pw_row(const PwItem& it, int m) { return (i64)(it.lo + m / PW_GROUP) * CL_Q_HEADS + it.head * PW_GROUP + m % PW_GROUP; }
CL_DEVICE int pw_limit(const PwItem& it, int m) { return it.off + it.lo + m / PW_GROUP; }

#if CL_EMIT_PARTIAL
extern "C" __global__ void __launch_bounds__(256, 2)
CL_PARTIAL_NAME(CL_PARTIAL_PARAMS) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  // the softmax scale as a positive factor of the raw scores (its sign goes into the Q rows, exactly)
  const float scale2 = fmaxf(fabsf(sm_scale) * 1.4426950408889634f, 1.0e-30f);
  const unsigned q_sign = sm_scale < 0.f ? 0x80008000u : 0u;
  const i64 row_bytes = (i64)CL_KV_HEADS * CL_HEAD_DIM * 2;            // K, V: (key row, kv head, feature)
  const unsigned tiles_byte = (unsigned)(size_t)(__attribute__((address_space(3))) elem_t*)pw_tiles;

  // ---- the item: requests one behind the other, each cut from its first query token on; (kv head, item) in one order, of which XCD x
  // walks the x-th eighth backwards: neighbouring items of a kv head, whose keys its L2 holds, later items of a request, which see
  // more keys, first.  In ranges, where a call has few items, neighbouring launches take the kv heads, then the ranges, of an item: the
  // numbers behind the last item come last and share no compute unit with real ones (spread between them, us, bf16, table, window
  // 4000: 1 x 8 tokens in 16 ranges 18.4 -> 14.2, 4 x 16 in 8 29.1 -> 24.6) ------------------------
  PwItem it;
  {
    // (XCD x is handed every eighth workgroup of a launch; the item axis is padded to a multiple of eight)
    const int gx = (int)gridDim.x, all_items = gx * CL_KV_HEADS * ranges;
    const int launch = (int)blockIdx.x + gx * ((int)blockIdx.y + CL_KV_HEADS * (int)blockIdx.z);
    int item;
    if (ranges > 1) {
      it.head = launch % CL_KV_HEADS;
      it.split = launch / CL_KV_HEADS % ranges;
      item = launch / CL_KV_HEADS / ranges;
    } else {
      const int lin = all_items - 1 - (launch % 8 * (all_items / 8) + launch / 8);
      item = lin % gx;
      it.head = lin / gx;
      it.split = 0;
    }
    const PwRequest found = pw_find_request(CL_ARG_QINDPTR, batch, total_q, CL_ARG_INDPTR, n_idx, item, lane);
    const int q1 = found.q1, kv0 = found.kv0, kv1 = found.kv1;
    it.lo = found.q0 + (item - found.first_item) * PW_QT;
    if (it.lo >= q1) return;                              // an index behind the last item
    const int hi = q1 < it.lo + PW_QT ? q1 : it.lo + PW_QT;
#if CL_RAGGED
    const int kv_len = kv1 > kv0 ? kv1 - kv0 : 0;
#else
    const int kv_len = kv1 > kv0 && num_pages > 0 ? kv1 - kv0 : 0;
#endif
    it.kv0 = kv0;
    it.off = kv_len - q1;
    it.n_rows = (hi - it.lo) * PW_GROUP;
    it.ext = it.off + hi;                                 // (the last row's own key, which is at most the request's last)
    it.ext = it.ext > 0 ? it.ext : 0;
    it.first_key = it.off + it.lo - CL_WINDOW + 1;        // the item's first row begins its window first
    it.skip = (it.first_key > 0 ? it.first_key : 0) / PW_STEP - PW_SINK_STEPS;
    it.skip = it.skip > 0 ? it.skip : 0;
    const int all = it.ext > 0 ? (it.ext + PW_STEP - 1) / PW_STEP - it.skip : 0, each = (all + ranges - 1) / ranges;
    it.first_step = it.split * each;
    it.n_steps = all - it.first_step < each ? all - it.first_step : each;
  }
  if (it.n_steps <= 0) {
    // rows without keys: zeros and -inf, or the partial of nothing
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const int m = 32 * wave + 16 * rt + c;
      if (m >= it.n_rows) continue;
      if (ranges > 1) {
        const i64 prow = PW_PROW(it, m);
#pragma unroll
        for (int fb = 0; fb < PW_FB; ++fb) *reinterpret_cast<f32x4*>(CL_ARG_PO + prow * CL_VDIM + 16 * fb + 4 * g) = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (g == 0) {
          CL_ARG_PM[prow] = CL_NEG_BIG;
          CL_ARG_PL[prow] = 0.f;
        }
      } else {
        elem_t* dst = CL_ARG_OUT + pw_row(it, m) * CL_VDIM + 16 * (g & 1) + 4 * (g & 2);
#pragma unroll
        for (int fp = 0; fp < PW_FB / 2; ++fp) *reinterpret_cast<u32x4*>(dst + 32 * fp) = (u32x4){0u, 0u, 0u, 0u};
#if CL_EMIT_LSE
        if (g == 0) CL_ARG_LSE[pw_row(it, m)] = CL_NEG_INF;
#endif
      }
    }
    return;
  }

  // ---- loads of one step, this wave's share: key rows 8 wave + lane / 8 of every 64-feature panel, the chunk for slot lane % 8.  A step
  // past the item's end repeats its last one into an image nobody reads, so that the load counter holds the same number of loads at
  // every wait; positions past the item's last key repeat it ------------------------------------------------------
  const int my_r = 8 * wave + (lane >> 3);
  const int chunk_byte = 16 * ((lane & 7) ^ pl_swz(my_r));
  const int last_step = it.n_steps - 1, tail_r = it.ext - 1 - PW_STEP * pw_tile(it, last_step);     // last row of the last step (31 and more: all)
  const int row_tail = my_r < tail_r ? my_r : tail_r;
  const char* kbase = reinterpret_cast<const char*>(CL_ARG_K) + (i64)it.head * CL_HEAD_DIM * 2;
  const char* vbase = reinterpret_cast<const char*>(CL_ARG_V) + (i64)it.head * CL_HEAD_DIM * 2;
#if CL_RAGGED
  // consecutive rows: a scalar base per step and one of two lane offsets (whole step / last step)
  const unsigned row_off = (unsigned)(my_r * (int)row_bytes + chunk_byte);
  const unsigned tail_off = (unsigned)(row_tail * (int)row_bytes + chunk_byte);
#endif
  auto issue = [&](const char* tensor, int s, unsigned image, auto lo_c, auto hi_c, int row) __attribute__((always_inline)) {
    s = s < last_step ? s : last_step;
    const unsigned dst = tiles_byte + image * (PW_IMG * 2) + (unsigned)(wave * 1024);
#if CL_RAGGED
    const char* base = tensor + (i64)(it.kv0 + pw_tile(it, s) * PW_STEP) * row_bytes;
    const unsigned off = s == last_step ? tail_off : row_off;
    pl_static_for<decltype(lo_c)::value, decltype(hi_c)::value>([&](auto p) __attribute__((always_inline)) {
      constexpr int P = decltype(p)::value;
      pl_dma16s<128 * P>(base, off, dst + (unsigned)(P * PW_PANEL * 2) - 128 * P);
    });
    (void)row;
#else
    const char* src = tensor + (i64)row * row_bytes + chunk_byte;
    pl_static_for<decltype(lo_c)::value, decltype(hi_c)::value>([&](auto p) __attribute__((always_inline)) {
      constexpr int P = decltype(p)::value;
      pl_dma16<128 * P>(src, dst + (unsigned)(P * PW_PANEL * 2) - 128 * P);
    });
#endif
  };
  auto issue_k = [&](int s, int slot, auto lo_c, auto hi_c, int row) __attribute__((always_inline)) { issue(kbase, s, slot, lo_c, hi_c, row); };
  auto issue_v = [&](int s, int slot, auto lo_c, auto hi_c, int row) __attribute__((always_inline)) { issue(vbase, s, PW_STAGES + slot, lo_c, hi_c, row); };
#if !CL_RAGGED
  auto key_pos = [&](int s) __attribute__((always_inline)) {
    const int pos = PW_STEP * pw_tile(it, s < last_step ? s : last_step) + (s < last_step ? my_r : row_tail);
    return pos < it.first_key && pos >= CL_SINKS ? it.first_key : pos;
  };
  auto row_of = [&](int s) __attribute__((always_inline)) { return pl_clamp(CL_ARG_INDICES[it.kv0 + key_pos(s)], 0, num_pages - 1); };
  // In the loop the lane's table entry travels like the tiles do, global -> LDS on the kernel's own load counter, a step ahead of
  // the loads that need it: entry of step s into pw_ids[s & 1][wave][lane].
  const unsigned ids_byte = (unsigned)(size_t)(__attribute__((address_space(3))) int*)&pw_ids[0][0][0];
  auto fetch_id = [&](int s) __attribute__((always_inline)) {
    pl_dma4(CL_ARG_INDICES + it.kv0 + key_pos(s), ids_byte + (unsigned)(((s & 1) * 4 + wave) * 256));
  };
  auto fetched_row = [&](int s) __attribute__((always_inline)) { return pl_clamp(pw_ids[s & 1][wave][lane], 0, num_pages - 1); };
#endif

  // ---- ahead of the loop: K 0, K 1, V 0, K 2, V 1 in the order the bodies wait for them, then the query rows as the B operand: lane
  // (c, g) holds Q[row][32 j + 8 g .. +8] of row c of each of the wave's row tiles; padded rows are 0 -------------------------
  using All = PlC<PW_PANELS>;
  int rows[2] = {0, 0};                        // table form: the lane's key rows of V of the next two bodies
#if CL_RAGGED
  constexpr int row0 = 0, row1 = 0, row3 = 0;
#else
  const int row0 = row_of(0), row1 = row_of(1), row3 = row_of(3);
  rows[0] = row_of(2);
  rows[1] = row3;
#endif
  issue_k(0, 0, PlC<0>{}, All{}, row0);
  issue_k(1, 1, PlC<0>{}, All{}, row1);
  issue_v(0, 0, PlC<0>{}, All{}, row0);
  issue_k(2, 2, PlC<0>{}, All{}, rows[0]);
#if !CL_RAGGED
  fetch_id(4);
#endif
  issue_v(1, 1, PlC<0>{}, All{}, row1);
  elem8 qf[2][PW_KJ];
  int lim_rel[2];                              // causal limit of the lane's rows relative to its first key slot
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const int m = 32 * wave + 16 * rt + c;
    const bool live = m < it.n_rows;
    lim_rel[rt] = (live ? pw_limit(it, m) : -1) - 4 * g;
    const elem_t* row = CL_ARG_Q + pw_row(it, live ? m : 0) * CL_HEAD_DIM + 8 * g;
#pragma unroll
    for (int j = 0; j < PW_KJ; ++j) {
      u32x4 raw = ld16(row + 32 * j);
      if (!live) raw = (u32x4){0u, 0u, 0u, 0u};
      qf[rt][j] = as_elem8(raw ^ q_sign);
    }
  }
  // Steps from n_low on and before n_full need no mask: every live row of this wave sees all their keys (the wave's first row has the
  // smallest limit, its last begins its window last; a wave without live rows masks nothing: its rows are not written).
  int n_full = it.n_steps, n_low = 0;
  if (32 * wave < it.n_rows) {
    const int first_limit = pw_limit(it, 32 * wave);
    n_full = first_limit < 0 ? 0 : (first_limit + 1) / PW_STEP - it.skip - it.first_step;
    n_full = n_full < it.n_steps ? n_full : it.n_steps;
    const int last_row = 32 * wave + 31 < it.n_rows ? 32 * wave + 31 : it.n_rows - 1;
    const int begun = pw_limit(it, last_row) - CL_WINDOW + 1;
    n_low = begun > 0 ? (begun + PW_STEP - 1) / PW_STEP - it.skip - it.first_step : 0;
  }
  n_full = __builtin_amdgcn_readfirstlane(n_full);
  n_low = __builtin_amdgcn_readfirstlane(n_low);

  // The values of masked steps times nothing: NaN from the first one on that is not finite.  (On the matrix cores, which have room:
  // us, six packed prompts of 31433 tokens, no check 533, this 545, dot products on the vector unit 548.)
  f32x4 taint = (f32x4){0.f, 0.f, 0.f, 0.f};
  u32x4 no_bits = (u32x4){0u, 0u, 0u, 0u};
  const elem8 none = as_elem8(no_bits);
  float m_run[2] = {CL_NEG_BIG, CL_NEG_BIG};   // reference point of a row's weights (log2 domain, the row's running max or up to 8 below it), uniform over g
  float l_run[2] = {0.f, 0.f};                 // this lane's share of the sum of the weights
  f32x4 acc[2][PW_FB];                         // acc[rt][fb][r] = O[row][16 fb + 4 g + r]
#pragma unroll
  for (int rt = 0; rt < 2; ++rt)
#pragma unroll
    for (int fb = 0; fb < PW_FB; ++fb) acc[rt][fb] = (f32x4){0.f, 0.f, 0.f, 0.f};

  // This lane's operand addresses in the first K and the first V image (LDS bytes), one per XOR pattern of a block: what is left of
  // every read is its immediate.  Hidden from the optimiser once a body, or it keeps a register for each sum and spills them.
  unsigned ka[2], va[4];
  {
    const int a_lo = c * 64 + ((g ^ pl_swz(c)) << 3);
    const int vtok = 4 * g + (c >> 2);
    const int v_lo = vtok * 64 + (((((c & 3) >> 1)) ^ pl_swz(vtok)) << 3) + 4 * (c & 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) ka[i] = tiles_byte + 2 * (a_lo ^ (32 * i));
#pragma unroll
    for (int i = 0; i < 4; ++i) va[i] = tiles_byte + 2 * (PW_STAGES * PW_IMG + (v_lo ^ (16 * i)));
  }
  auto keep_addresses = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) asm volatile("" : "+v"(ka[i]));
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(va[i]));
  };
  // key fragment of 16-key half h and 32-feature block j out of the K image in stage SLOT
  auto k_frag = [&](auto slot_c, int j, int h) __attribute__((always_inline)) {
    constexpr int SLOT = decltype(slot_c)::value;
    return *(const pl_lds_elem8*)(ka[j & 1] + (unsigned)((SLOT * PW_IMG + (j >> 1) * PW_PANEL + 16 * h * 64) * 2));
  };
  // value operand for feature block fb out of the V image in stage SLOT: rows = features
  // 16 fb + (0..15), slots = keys 4 g + (0..3), 16 + 4 g + (0..3)
  auto v_frag = [&](auto slot_c, int fb) __attribute__((always_inline)) {
    constexpr int SLOT = decltype(slot_c)::value;
    const unsigned p = va[fb & 3] + (unsigned)((SLOT * PW_IMG + (fb >> 2) * PW_PANEL) * 2);
    const pl_s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pl_lds_s16x4*)(p));
    const pl_s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pl_lds_s16x4*)(p + 16 * 64 * 2));
    return __builtin_bit_cast(elem8, (pl_s16x8)__builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x4 st[2][2];                              // raw scores^T of the step the next body weighs
  // (256-wide keys: fragments are held half a step at a time, or query fragments are spilled)
  constexpr int KH = PW_KJ > 6 ? PW_KJ / 2 : PW_KJ;
  static_assert(KH == PW_KJ || PW_STAGES == 4, "K of the step in hand keeps its image where it is read in two halves");
  elem8 kf[KH][2];                             // key fragments of the step the next body scores
  auto read_keys = [&](auto slot_c, int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < KH; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) kf[j][h] = k_frag(slot_c, j0 + j, h);
  };
  // scores of the fragments in hand: feature blocks j0 ..
  auto score = [&](f32x4 (&sc)[2][2], int j0) __attribute__((always_inline)) {
    if (j0 == 0) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) sc[rt][0] = sc[rt][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int j = 0; j < KH; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) sc[rt][h] = mfma16(kf[j][h], qf[rt][j0 + j], sc[rt][h]);
  };
  // slot i of the lane is key 32 tile + 16 (i / 4) + 4 g + i % 4; a masked slot scores -inf, which a finite reference turns
  // into a weight of exactly 0.  The causal end and the beginning of windows each by itself: few steps have both.
  auto mask = [&](f32x4 (&sc)[2][2], int step) __attribute__((always_inline)) {
    const int t0 = pw_tile(it, step) * PW_STEP;
    if (step >= n_full) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[rt][i >> 2][i & 3] = 16 * (i >> 2) + (i & 3) <= lim_rel[rt] - t0 ? sc[rt][i >> 2][i & 3] : CL_NEG_INF;
    }
    if (step < n_low) {
      const int sink_room = CL_SINKS - 4 * g - t0;
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = 16 * (i >> 2) + (i & 3);
          sc[rt][i >> 2][i & 3] = key > lim_rel[rt] - t0 - CL_WINDOW || (CL_SINKS > 0 && key < sink_room) ? sc[rt][i >> 2][i & 3] : CL_NEG_INF;
        }
    }
  };
  auto step_max = [&](const f32x4 (&sc)[2]) __attribute__((always_inline)) {
    float v = sc[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) v = fmaxf(v, sc[i >> 2][i & 3]);
    return v;
  };

  // Body of step `step`, step % PW_STAGES == S: turns the scores of the step (made in the body before) into weights, adds their value
  // product and makes the scores of step + 1 from key fragments that are in registers when it begins; the value fragments are read
  // beside the score products and the key fragments of step + 2 beside the value products.
  auto do_step = [&](auto s_c, const int step) __attribute__((always_inline)) {
    constexpr int S = decltype(s_c)::value;
    keep_addresses();
#if CL_RAGGED
    constexpr int row_v = 0, row_k = 0;
#else
    // (V of step + 2, whose row was looked up two bodies ago; K of step + 4, whose entry was asked for in the last body
    // ahead of the loads that the wait before this one left out)
    const int row_v = rows[0], row_k = fetched_row(step + 4);
    rows[0] = rows[1];
    rows[1] = row_k;
    fetch_id(step + 5);
#endif
    // the loads of this body, in four shares between its matrix work: V of step + 2, K of step + 4
    auto ask = [&](auto place_c) __attribute__((always_inline)) {
      constexpr int LO = decltype(place_c)::value * PW_UNITS / 4, HI = (decltype(place_c)::value + 1) * PW_UNITS / 4;
      constexpr int VL = LO < PW_PANELS ? LO : PW_PANELS, VH = HI < PW_PANELS ? HI : PW_PANELS;
      issue_v(step + 2, (S + 2) % PW_STAGES, PlC<VL>{}, PlC<VH>{}, row_v);
      issue_k(step + 4, (S + 4) % PW_STAGES, PlC<LO - VL>{}, PlC<HI - VH>{}, row_k);
    };
    __builtin_amdgcn_sched_barrier(0);
    if (step >= n_full || step < n_low) mask(st, step);
    __builtin_amdgcn_sched_barrier(0);

    elem8 pf[2];
    float psum[2] = {0.f, 0.f};
    auto weigh = [&](int rt) __attribute__((always_inline)) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = fast_exp2(__builtin_fmaf(st[rt][i >> 2][i & 3], scale2, -m_run[rt]));
        sum += p;
        pf[rt][i] = to_elem(p);
      }
      psum[rt] = sum;
    };
    // Where a lane's eight weights sum to more than 2^8 the row's reference is raised to the step's maximum and the weights are
    // taken again.  Only that row's: a row's bits do not depend on the rows beside it in the wave.
    auto settle = [&](int rt) __attribute__((always_inline)) {
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(psum[rt] > 256.0f) != 0, 0)) {
        const float mx = pl_max_over_groups(step_max(st[rt])) * scale2;
        const bool over = pl_max_over_groups(psum[rt]) > 256.0f;
        const float m_new = over ? fmaxf(mx, m_run[rt]) : m_run[rt];
        const float alpha = fast_exp2(m_run[rt] - m_new);
        m_run[rt] = m_new;
        l_run[rt] *= alpha;
#if PW_ALONE
        // (512 registers: the accumulators live in the half that only matrix ops reach, and their way to these multiplications
        // begins here, not in every step)
#pragma unroll
        for (int fb = 0; fb < PW_FB; ++fb) asm volatile("" : "+a"(acc[rt][fb]));
#endif
#pragma unroll
        for (int fb = 0; fb < PW_FB; ++fb) acc[rt][fb] *= alpha;
        weigh(rt);
      }
      l_run[rt] += psum[rt];
    };

    // ---- score products of step + 1 and value fragments of this step beside the weights of the first row tile --------
    f32x4 sn[2][2];
    ask(PlC<0>{});
    if constexpr (KH < PW_KJ) {
      score(sn, 0);
      __builtin_amdgcn_sched_barrier(0);
      read_keys(PlC<(S + 1) % PW_STAGES>{}, KH);
      score(sn, KH);
    } else {
      score(sn, 0);
    }
    elem8 vf[PW_FB];
#pragma unroll
    for (int fb = 0; fb < PW_FB; ++fb) vf[fb] = v_frag(PlC<S>{}, fb);
    weigh(0);
    if constexpr (KH == PW_KJ) {
#pragma unroll
      for (int i = 0; i < 4 * PW_KJ; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, (2 * PW_FB + 4 * PW_KJ - 1) / (4 * PW_KJ), 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    settle(0);
    __builtin_amdgcn_sched_barrier(0);
    ask(PlC<1>{});

    // ---- value product of the first row tile and key fragments of step + 2 beside the weights of the second ----------
#pragma unroll
    for (int fb = 0; fb < PW_FB; ++fb) acc[0][fb] = mfma16(vf[fb], pf[0], acc[0][fb]);
    read_keys(PlC<(S + 2) % PW_STAGES>{}, 0);
    weigh(1);
#pragma unroll
    for (int i = 0; i < PW_FB; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, (2 * KH + PW_FB - 1) / PW_FB, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    settle(1);
    __builtin_amdgcn_sched_barrier(0);
    ask(PlC<2>{});

    // ---- value product of the second row tile ------------------------------------------------
#pragma unroll
    for (int fb = 0; fb < PW_FB; ++fb) acc[1][fb] = mfma16(vf[fb], pf[1], acc[1][fb]);
    ask(PlC<3>{});
    // (here: a branch between the products above, whose operands it reads, keeps them from running beside each other, 5 % of a call)
    if (step >= n_full || step < n_low) {
#pragma unroll
      for (int fb = 0; fb < PW_FB; ++fb) taint = mfma16(vf[fb], none, taint);
    }
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int h = 0; h < 2; ++h) st[rt][h] = sn[rt][h];
  };
  // Between two bodies: the loads of all bodies but the last have landed, everybody's (V of the next step and the keys that
  // it reads ahead), and the images that the last body read last are free for what the next one asks for.
  auto turn = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    PL_WAITCNT(PW_UNITS);
    pl_barrier();
  };

  PL_WAITCNT(3 * PW_PANELS + !CL_RAGGED);
  pl_barrier();
#pragma unroll
  for (int j0 = 0; j0 < PW_KJ; j0 += KH) {
    read_keys(PlC<0>{}, j0);
    score(st, j0);
  }
  read_keys(PlC<1>{}, 0);
#if CL_HEAD_DIM <= 192
  // (the first reference points, so that the first weights need not be taken twice; the widest heads have no registers for it)
  if (n_full <= 0 || n_low > 0) mask(st, 0);
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const float mx = pl_max_over_groups(step_max(st[rt])) * scale2;
    m_run[rt] = mx > CL_NEG_BIG ? mx : CL_NEG_BIG;
  }
#endif
  // the images of body 0 (V 0, K 2) have landed; K 0 has been read by everybody
  PL_WAITCNT(PW_PANELS);
  pl_barrier();
  issue_k(3, 3 % PW_STAGES, PlC<0>{}, All{}, row3);
  for (int step = 0;;) {
    do_step(PlC<0>{}, step);
    if (++step >= it.n_steps) break;
    turn();
    do_step(PlC<1>{}, step);
    if (++step >= it.n_steps) break;
    turn();
    do_step(PlC<2>{}, step);
    if (++step >= it.n_steps) break;
    turn();
    if constexpr (PW_STAGES > 3) {
      do_step(PlC<3>{}, step);
      if (++step >= it.n_steps) break;
      turn();
    }
  }
  // no load may still be on its way into LDS when the workgroup ends
  PL_WAITCNT(0);

  // ---- an item's results ---------------------------------------------------------------------------------
  // (row coordinates are worked out again from the lane number, behind a barrier for the optimiser: kept across the loop they
  // would cost registers the loop needs)
  int lane_e = lane;
  asm volatile("" : "+v"(lane_e));
  const int c_e = lane_e & 15, g_e = lane_e >> 4;
  const float tainted = (taint[0] + taint[1]) + (taint[2] + taint[3]);
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(tainted != tainted) != 0, 0)) {
    // the wave's rows key by key, 64 features at a time: the largest score of what a row sees, then its weights
    for (int mw = 0; mw < 32; ++mw) {
      const int m = 32 * wave + mw;
      if (m >= it.n_rows) break;
      const int last = pw_limit(it, m);
      const i64 row = pw_row(it, m);
      float q[PW_PANELS], o[PW_PANELS], top = CL_NEG_BIG, sum = 0.f;
#pragma unroll
      for (int i = 0; i < PW_PANELS; ++i) {
        q[i] = to_f32(CL_ARG_Q[row * CL_HEAD_DIM + 64 * i + lane_e]);
        o[i] = 0.f;
      }
      for (int pass = 0; pass < 2; ++pass)
        for (int s = 0; s < it.n_steps; ++s)
          for (int r = 0; r < PW_STEP; ++r) {
            const int pos = PW_STEP * pw_tile(it, s) + r;
            if (pos > last || (pos <= last - CL_WINDOW && pos >= CL_SINKS)) continue;
#if CL_RAGGED
            const i64 key = it.kv0 + pos;
#else
            const i64 key = pl_clamp(CL_ARG_INDICES[it.kv0 + pos], 0, num_pages - 1);
#endif
            const elem_t* kr = reinterpret_cast<const elem_t*>(kbase + key * row_bytes);
            const elem_t* vr = reinterpret_cast<const elem_t*>(vbase + key * row_bytes);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < PW_PANELS; ++i) dot += q[i] * to_f32(kr[64 * i + lane_e]);
#pragma unroll
            for (int b = 1; b < 64; b *= 2) dot += lane_xor(dot, lane_e, b);
            const float value = (q_sign ? -dot : dot) * scale2;
            if (pass == 0) {
              top = fmaxf(top, value);
            } else {
              const float w = fast_exp2(value - top);
              sum += w;
#pragma unroll
              for (int i = 0; i < PW_PANELS; ++i) o[i] += w * to_f32(vr[64 * i + lane_e]);
            }
          }
      if (ranges > 1) {
        const i64 prow = PW_PROW(it, m);
#pragma unroll
        for (int i = 0; i < PW_PANELS; ++i) CL_ARG_PO[prow * CL_VDIM + 64 * i + lane_e] = o[i];
        if (lane_e == 0) {
          CL_ARG_PM[prow] = top;
          CL_ARG_PL[prow] = sum;
        }
      } else {
        const float inv = 1.0f / fmaxf(sum, 1.0e-30f);
#pragma unroll
        for (int i = 0; i < PW_PANELS; ++i) CL_ARG_OUT[row * CL_VDIM + 64 * i + lane_e] = to_elem(o[i] * inv);
#if CL_EMIT_LSE
        if (lane_e == 0) CL_ARG_LSE[row] = cl_lse(top, sum);
#endif
      }
    }
    return;
  }
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    float l = l_run[rt];
    l += lane_xor(l, lane_e, 16);
    l += lane_xor(l, lane_e, 32);
    const int m = 32 * wave + 16 * rt + c_e;
    if (m >= it.n_rows) continue;
    if (ranges > 1) {
      // unnormalised f32 values (16 bytes per lane and block), m and l by the g == 0 lanes
      const i64 prow = PW_PROW(it, m);
      float* dstp = CL_ARG_PO + prow * CL_VDIM + 4 * g_e;
#pragma unroll
      for (int fb = 0; fb < PW_FB; ++fb) *reinterpret_cast<f32x4*>(dstp + 16 * fb) = acc[rt][fb];
      if (g_e == 0) {
        CL_ARG_PM[prow] = m_run[rt];
        CL_ARG_PL[prow] = l;
      }
    } else {
      const i64 row = pw_row(it, m);
      pl_store_row<PW_FB, false>(CL_ARG_OUT + row * CL_VDIM, acc[rt], 1.0f / fmaxf(l, 1.0e-30f), g_e);
#if CL_EMIT_LSE
      if (g_e == 0) CL_ARG_LSE[row] = cl_lse(m_run[rt], l);
#endif
    }
  }
}
#endif  // CL_EMIT_PARTIAL
