// GQA decode, verify and tree steps: the host side of the one-launch kernel of gqa_stream_kernel.cuh, and its launches for the bf16 cache.
#include "gqa_stream_kernel.cuh"

namespace relux {

bool gqa_stream_eligible(const Pool* p, const relux_attn_args& a) {
  const relux_pool_params& prm = p->prm;
  const int g = a.num_heads / std::max(1, prm.gqa_num_kv_heads);
  return p->has_tmap && prm.page_tokens == kGqaPageTok && prm.gqa_head_dim == kGqaD && g >= 1 && g <= 32 && a.q_tokens >= 1 &&
         a.q_tokens <= 32 / g;
}

// A step's new rows can ride in the attention launch: the pages it loads must cover them (rows past the visible tokens of
// a sequence would be nobody's), and the bookkeeping of reference-compat pools stays with the plain append.
bool gqa_append_fusable(const Pool* p, const relux_attn_args& a, int max_new_rows, bool advance) {
  return !p->compat && a.mode == RELUX_ATTN_FAST && gqa_stream_eligible(p, a) && (advance || max_new_rows <= a.extra_tokens);
}

// q: device [n][S][H][128] token-major (f32 or bf16).  out: device, same shape, f32 or bf16.  With `app` (advance = 1) the
// host lengths already count the new rows.  `tree` (with `app`, advance = 0): the new rows are its nodes.
int32_t launch_gqa_stream(Pool* p, const SeqBatch& sb, const relux_attn_args& a, const void* d_q, void* d_out, bool out_bf16,
                          const GqaAppend* app, const GqaTree* tree) {
  const relux_pool_params& prm = p->prm;
  const int n = sb.n_seqs, Hkv = prm.gqa_num_kv_heads, g = a.num_heads / Hkv, R = g * a.q_tokens;
  GqaStreamCommon c{};
  GqaSeq inl[kInlineLarge + 1];
  GqaSeq* seqs = inl;
  int slot_index = 0;
  if (n > kInlineLarge) {
    if (tree && stream_captured(p->dev)) {
      set_error("tree_verify: a call of more than %d sequences cannot be captured", kInlineLarge);
      return RELUX_ERR_UNSUPPORTED;
    }
    int32_t* slot = nullptr;
    if (int32_t rc = stage_acquire(p, &slot, &slot_index)) return rc;
    seqs = (GqaSeq*)slot;
  }
  int64_t units64 = 0;
  int rows = 0;
  for (int i = 0; i < n; i++) {
    const int s = sb.seq[i], len = p->h_len[(size_t)a.layer * prm.max_seqs + s], n_new = app ? app->rows[i] : 0;
    seqs[i] = GqaSeq{s, app && app->advance ? len - n_new : len, (int32_t)units64, rows};
    // one page at least: a tree without nodes on an empty sequence sees nothing of it
    units64 += std::max(1, (len + (tree ? n_new : a.extra_tokens) + kGqaPageTok - 1) / kGqaPageTok) + kStreamUnits;
    rows += n_new;
  }
  seqs[n] = GqaSeq{0, 0, (int32_t)units64, rows};
  units64 *= Hkv;
  if (units64 >= ((int64_t)1 << 31)) { set_error("more cached pages than one attention launch addresses"); return RELUX_ERR_UNSUPPORTED; }
  const int units = (int)units64;
  // One range per SM; ranges of fewer than two units do not pay for their share of the merge.  Where streams are a page or two,
  // some ranges hold no page and their CTAs leave at once; that costs nothing: one sequence of 60 to 120 tokens, 8 kv heads, takes
  // 4.1 us on 20 or 24 CTAs, and 6.1 with one unit a stream, whose ranges split the two pages.
  int workers = std::max(1, std::min(p->dev->sm_count, units / 2));
  if (const int ov = p->tune.get(RELUX_TUNE_CHUNK_PAGES)) workers = std::max(1, std::min(units, (units + ov - 1) / ov));   // tuning knob
  const size_t part_rows = (size_t)2 * workers * R;
  int32_t rc = grow(p->dev, p->part_o, part_rows * (kGqaD + 2) * sizeof(float));
  if (rc) return rc;
  const size_t ctr_bytes = (size_t)n * Hkv * kFinishers * sizeof(uint32_t);
  const size_t ctr_cap = p->stream_done.cap;
  if ((rc = grow(p->dev, p->stream_done, ctr_bytes))) return rc;
  if (p->stream_done.cap != ctr_cap) RELUX_CUDA_TRY(cudaMemsetAsync(p->stream_done.p, 0, p->stream_done.cap, p->dev->stream));
  if (seqs != inl) {
    size_t bytes = sizeof(GqaSeq) * ((size_t)n + 1);
    if (tree) {   // behind the sequences
      const size_t tree_bytes = (size_t)kTreeNodes * (tree->one ? 1 : n);
      memcpy((char*)seqs + bytes, tree->parents, tree_bytes);
      bytes += tree_bytes;
    }
    if ((rc = grow(p->dev, p->seq_list, bytes))) return rc;
    RELUX_CUDA_TRY(cudaMemcpyAsync(p->seq_list.p, seqs, bytes, cudaMemcpyHostToDevice, p->dev->stream));
    if ((rc = stage_release(p, slot_index))) return rc;
    c.seqs = (const GqaSeq*)p->seq_list.p;
    if (tree) c.parents = (const int8_t*)(c.seqs + n + 1);
  }
  c.table = p->d_table;
  c.table_stride = prm.max_pages_per_seq;
  c.num_pages = prm.num_pages;
  c.n_seqs = n;
  c.range = units / workers;
  c.range_more = units % workers;
  c.Hkv = Hkv;
  c.H = a.num_heads;
  c.g = g;
  c.S = a.q_tokens;
  c.R = R;
  c.one_tree = tree && tree->one;
  c.extra = a.extra_tokens;
  c.causal = a.causal;
  const int64_t rows_per_block = (int64_t)prm.num_pages * Hkv * kGqaPageTok;
  c.krow0 = (int32_t)((int64_t)a.layer * 2 * rows_per_block);
  c.vrow0 = (int32_t)((int64_t)a.layer * 2 * rows_per_block + rows_per_block);
  c.streams = (units64 - (int64_t)kStreamUnits * n * Hkv) * (p->int8 ? kInt8StageBytes + kInt8ScaleBytes : kGqaStageBytes) > kResidentBytes;
  c.scale_log2 = a.scale * 1.4426950408889634f;
  c.q = d_q;
  c.q_bf16 = a.q_dtype == RELUX_DTYPE_BF16;
  c.out_bf16 = out_bf16;
  c.out = d_out;
  c.part_o = (float*)p->part_o.p;
  c.part_ml = c.part_o + part_rows * kGqaD;
  c.done = (uint32_t*)p->stream_done.p;
  if (app && rows > 0) {
    c.k_new = app->k;
    c.v_new = app->v;
    c.new_f32 = app->dtype == RELUX_DTYPE_F32;
    c.head_major = app->layout == RELUX_LAYOUT_HEAD_MAJOR;
    c.advance = app->advance;
  }
  c.k_base = (uint16_t*)p->rows_at(a.layer, 0);
  c.v_base = (uint16_t*)p->rows_at(a.layer, 1);
  if (p->int8) c.scales = p->scales_at(a.layer);
  c.len = p->d_len + (size_t)a.layer * prm.max_seqs;
  c.status = p->d_status;
  c.time = time_stamp_next(p, p->attn_times);
  const int8_t* parents = tree ? tree->parents : nullptr;
  if (tree) return p->int8 ? launch_gqa_stream_tree_int8(p, c, seqs, parents, workers) : launch_gqa_stream_tree(p, c, seqs, parents, workers);
  return p->int8 ? launch_gqa_stream_int8(p, c, seqs, workers) : launch_variant<0>(p, c, seqs, nullptr, workers);
}

}  // namespace relux
