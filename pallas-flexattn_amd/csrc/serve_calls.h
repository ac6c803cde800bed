// Argument checks and kernel arguments of the C ABI calls for prompts over a paged cache, caches of
// latent vectors, and pages (included by capi.hip inside its anonymous namespace, behind cache_calls.h).

// What the calls on a paged cache have in common.
int paged_ok(int B, int page_size, int max_pages, int num_pages, const int32_t* table) {
  if (B < 1 || page_size < FA_KV_RUN || page_size % FA_KV_RUN || num_pages < 1 || max_pages < 1) return FA_ERR_SHAPE;
  return !table && (max_pages != 1 || num_pages < B) ? FA_ERR_SHAPE : FA_OK;
}
bool normal_or_zero(float x) { return x == 0.f || (x >= FLT_MIN && x <= FLT_MAX); }

// (*workspace: its bytes)
int prefill_args(const fa_prefill_call* c, int cus, fa::PrefillArgs* a, size_t* workspace) {
  if (!c) return FA_ERR_NULL;
  if (c->abi_version != FA_ABI_VERSION) return FA_ERR_VERSION;
  if (c->cache_dtype != FA_DTYPE_BF16 && c->cache_dtype != FA_DTYPE_FP8_E4M3) return FA_ERR_DTYPE;
  if (c->D != 32 && c->D != 64 && c->D != 128) return FA_ERR_UNSUPPORTED;
  const int Hq = c->query.heads;
  if (const int rc = paged_ok(c->B, c->page_size, c->max_pages, c->num_pages, c->page_table)) return rc;
  if (c->T < 1 || c->Hkv < 1 || Hq < 1 || Hq % c->Hkv || c->out.heads != Hq) return FA_ERR_SHAPE;
  if (c->kv_len < 1 || c->kv_len > 0x7fffffff - 2 * fa::kPrefillKeys || (long long)c->max_pages * c->page_size < c->kv_len)
    return FA_ERR_SHAPE;
  if (!normal_or_zero(c->softcap) || !normal_or_zero(c->scale)) return FA_ERR_SHAPE;
  if (c->q_lens && c->q_starts) return FA_ERR_UNSUPPORTED;
  const bool fp8 = c->cache_dtype == FA_DTYPE_FP8_E4M3;
  if (!c->query.data || !c->out.data || !c->lse || !c->k_cache || !c->v_cache) return FA_ERR_NULL;
  if (fp8 && (!c->k_scale || !c->v_scale)) return FA_ERR_NULL;
  if (!rows16(c->query, 2) || !rows16(c->out, 2) || !aligned16({c->k_cache, c->v_cache})) return FA_ERR_SHAPE;
  // (run indices are 32 bits, and so are the rows of a batch row and the tiles of a call)
  if ((long long)c->num_pages * c->Hkv * (c->page_size / FA_KV_RUN) > 0x7fffffffll) return FA_ERR_SHAPE;
  const bool packed = c->q_starts != nullptr;
  const int g = Hq / c->Hkv;
  if ((long long)c->T * Hq > 0x7fffffffll - fa::kPrefillRows) return FA_ERR_SHAPE;
  const long long tiles = fa::prefill_tiles(packed, c->B, c->T, g), items = tiles * c->Hkv;
  if (items > 0x7fffffll) return FA_ERR_SHAPE;
  *a = fa::PrefillArgs{};
  a->q = c->query.data;
  a->qsb = c->query.stride_b, a->qsh = c->query.stride_h, a->qst = c->query.stride_t;
  a->o = const_cast<void*>(c->out.data);
  a->osb = c->out.stride_b, a->osh = c->out.stride_h, a->ost = c->out.stride_t;
  a->lse = c->lse;
  a->k = static_cast<const char*>(c->k_cache);
  a->v = static_cast<const char*>(c->v_cache);
  a->ks = c->k_scale;
  a->vs = c->v_scale;
  a->page_table = c->page_table;
  a->kv_lens = c->kv_lens;
  a->q_lens = c->q_lens;
  a->starts = c->q_starts;
  a->B = c->B;
  a->Hq = Hq;
  a->Hkv = c->Hkv;
  a->Sq = c->T;
  a->g = g;
  a->page_runs = c->page_size / FA_KV_RUN;
  a->max_pages = c->max_pages;
  a->num_pages = c->num_pages;
  a->cap = c->kv_len;
  a->win_left = c->window_left < 0 || c->window_left >= c->kv_len ? -1 : c->window_left;
  a->win_right = c->window_right < 0 ? -1 : c->window_right;
  a->scale = c->scale == 0.f ? 1.0f / sqrtf((float)c->D) : c->scale;
  a->scale_log2 = a->scale * fa::kLog2e;
  a->softcap = c->softcap;
  a->alibi = c->alibi_slopes;
  a->tiles = (int)tiles;
  long long walk = (c->kv_len + (long long)fa::kPrefillKeys - 1) / fa::kPrefillKeys;  // the longest that an item can have
  if (a->win_left >= 0)
    walk = std::min(walk, ((long long)a->win_left + fa::kPrefillRows / g + fa::kPrefillKeys) / fa::kPrefillKeys + 2);
  // Workgroups for all that run at a time, two per compute unit at D = 128, else three (300 items of D = 64, 8192 keys: 129 us in
  // two ranges each, 164 whole).  Packed rows: as many tiles as full ones, or as rows (31 of one token, 4200 keys: 63 us; in 32
  // ranges, as for the tokens in one tile: 129); with lengths: about half the rows are there, which is not
  // known (16 ragged rows, 512 items: 110 us in two ranges, 130 whole; where most of them are: 258, 242).
  const long long full = packed ? std::max<long long>((long long)c->T * g / fa::kPrefillRows, std::min(c->B, c->T)) * c->Hkv
                                : c->q_lens ? (items + 1) / 2 : items;
  const fa::PrefillCut cut = fa::prefill_cut(full, (int)walk, (c->D == 128 ? 2 : 3) * cus, !c->q_lens);
  const bool fits = items * cut.n <= 0x7fffffll;
  a->n_splits = fits ? cut.n : 1;
  a->few = fits ? cut.few : 0;
  const size_t rows = (size_t)(packed ? 1 : c->B) * Hq * c->T;
  if (rows > 0x7fffffffull) return FA_ERR_SHAPE;
  *workspace = a->n_splits > 1 ? rows * a->n_splits * (c->D + 2) * sizeof(float) : 0;
  return FA_OK;
}

// (tokens of one head each: the strides of rows and tokens)
int latent_append_args(const fa_latent_append_call* c, fa::LatentAppendArgs* a) {
  if (!c) return FA_ERR_NULL;
  if (c->abi_version != FA_ABI_VERSION) return FA_ERR_VERSION;
  if ((c->latent_dim != 128 && c->latent_dim != 256 && c->latent_dim != 512) || (c->rope_dim != 32 && c->rope_dim != 64))
    return FA_ERR_UNSUPPORTED;
  if (const int rc = paged_ok(c->B, c->page_size, c->max_pages, c->num_pages, c->page_table)) return rc;
  if (c->T < 1 || c->latent.heads != 1 || c->rope.heads != 1 || c->query.heads < 0) return FA_ERR_SHAPE;
  if (!c->latent.data || !c->rope.data || !c->cache || !c->kv_lens) return FA_ERR_NULL;
  if (!rows16(c->latent, 2) || !rows16(c->rope, 2) || !aligned16({c->cache})) return FA_ERR_SHAPE;
  const bool turn = c->rotary.pairs != 0;
  if (turn) {
    if (!c->rotary.inv_freq) return FA_ERR_NULL;
    if (c->rotary.pairs < 0 || 2 * (long long)c->rotary.pairs > c->rope_dim || !aligned(c->rotary.inv_freq, 8)) return FA_ERR_SHAPE;
    if (c->rotary.pairs % 8) return FA_ERR_UNSUPPORTED;
  }
  *a = fa::LatentAppendArgs{};
  a->latent = c->latent.data;
  a->rope = c->rope.data;
  a->lsb = c->latent.stride_b, a->lst = c->latent.stride_t;
  a->rsb = c->rope.stride_b, a->rst = c->rope.stride_t;
  a->cache = static_cast<uint16_t*>(c->cache);
  a->page_table = c->page_table;
  a->kv_lens = c->kv_lens;
  a->new_lens = c->new_lens;
  a->page_size = c->page_size;
  a->max_pages = c->max_pages;
  a->num_pages = c->num_pages;
  a->B = c->B;
  a->T = c->T;
  a->L = c->latent_dim;
  a->R = c->rope_dim;
  if (turn) {
    a->freq = c->rotary.inv_freq;
    a->n = c->rotary.pairs;
    a->interleaved = c->rotary.interleaved != 0;
    a->scale = c->rotary.scale;
  }
  a->units = (c->latent_dim + c->rope_dim) / 16;
  if ((long long)c->B * c->T > 0x7fffff00ll / a->units) return FA_ERR_SHAPE;
  a->kv_blocks = (int)(((long long)c->B * c->T * a->units + 255) / 256);
  if (c->query.heads > 0) {
    if (!turn) return FA_ERR_SHAPE;  // nothing to do for the queries
    if (!c->query.data || !c->query_out) return FA_ERR_NULL;
    if (!rows16(c->query, 2) || !aligned(c->query_out, 16)) return FA_ERR_SHAPE;
    fa::RotaryArgs& q = a->q;
    q.t[0] = {c->query.data, c->query_out, c->query.stride_b, c->query.stride_h, c->query.stride_t, c->query.heads};
    q.B = c->B;
    q.T = c->T;
    q.D = c->rope_dim;
    q.freq = a->freq;
    q.n = a->n;
    q.interleaved = a->interleaved;
    q.scale = a->scale;
    q.kv_lens = c->kv_lens;
    const long long threads = rotary_units(&q, true);
    return rotary_groups(&q, threads, heads_per_thread(threads * c->query.heads));
  }
  return FA_OK;
}

struct LatentLayout {
  int nb;
  size_t part, ml, bytes;
};
int latent_args(const fa_latent_call* c, int cus, fa::LatentArgs* a, LatentLayout* L) {
  if (!c) return FA_ERR_NULL;
  if (c->abi_version != FA_ABI_VERSION) return FA_ERR_VERSION;
  if ((c->latent_dim != 128 && c->latent_dim != 256 && c->latent_dim != 512) || (c->rope_dim != 32 && c->rope_dim != 64))
    return FA_ERR_UNSUPPORTED;
  if (const int rc = paged_ok(c->B, c->page_size, c->max_pages, c->num_pages, c->page_table)) return rc;
  const int H = c->query.heads;
  if (c->T < 1 || H < 1 || c->query_rope.heads != H) return FA_ERR_SHAPE;
  if (c->kv_len < 1 || c->kv_len > 0x7fffffff - 2 * fa::kLatentKeys || (long long)c->max_pages * c->page_size < c->kv_len)
    return FA_ERR_SHAPE;
  if (!(c->scale >= FLT_MIN && c->scale <= FLT_MAX)) return FA_ERR_SHAPE;
  if (!c->query.data || !c->query_rope.data || !c->o || !c->lse || !c->cache) return FA_ERR_NULL;
  if (!rows16(c->query, 2) || !rows16(c->query_rope, 2) || !aligned16({c->cache, c->o})) return FA_ERR_SHAPE;
  if ((long long)c->num_pages * (c->page_size / FA_KV_RUN) > 0x7fffffffll) return FA_ERR_SHAPE;  // (run indices)
  const long long rows = (long long)H * c->T;
  if (rows > 0x7ffffffll || c->B > 0x7ffffffll / rows) return FA_ERR_SHAPE;
  *a = fa::LatentArgs{};
  fa::DecodeArgs& d = a->d;
  const int left = c->window_left < 0 || c->window_left >= c->kv_len ? -1 : c->window_left;
  long long tiles = (c->kv_len + (long long)fa::kTileKeys - 1) / fa::kTileKeys;
  if (left >= 0) tiles = std::min(tiles, ((long long)left + c->T + fa::kTileKeys - 2) / fa::kTileKeys + 1);
  // rows of an item: up to 64, so that a key is read for as many at once, and of one size (16 batch rows of 96 rows: 45.5 us
  // in two blocks of 48, 49.4 in 64 and 32)
  const long long rt = (rows + 63) / 64, items = c->B * rt;
  L->nb = (int)(((rows + 15) / 16 + rt - 1) / rt);
  if (items * tiles > 0x7fffffffll - (1 << 20)) return FA_ERR_SHAPE;  // tile numbers of a call are 32 bits
  d.page_table = c->page_table;
  d.kv_lens = c->kv_lens;
  d.q_lens = c->q_lens;
  d.o = c->o;
  d.lse = c->lse;
  d.B = c->B;
  d.Hkv = 1;
  d.Sq = c->T;
  d.g = H;
  d.page_runs = c->page_size / FA_KV_RUN;
  d.max_pages = c->max_pages;
  d.num_pages = c->num_pages;
  d.cap = c->kv_len;
  d.win_left = left;
  d.win_right = c->window_right < 0 || c->window_right >= c->T - 1 ? -1 : c->window_right;
  d.scale = c->scale;
  d.scale_log2 = c->scale * fa::kLog2e;
  d.rt = 1;
  a->rt = (int)rt;
  a->cache = static_cast<const uint16_t*>(c->cache);
  a->q = c->query.data;
  a->qsb = c->query.stride_b, a->qsh = c->query.stride_h, a->qst = c->query.stride_t;
  a->qr = c->query_rope.data;
  a->rsb = c->query_rope.stride_b, a->rsh = c->query_rope.stride_h, a->rst = c->query_rope.stride_t;
  d.by_item = tiles <= 8 || (items >= cus && tiles <= 128) || c->B > 64 * fa::kMostLaneRows || c->B * rows > (1 << 22);
  d.pieces = d.pieces_even = (int)std::max(1ll, cus / rt);
  d.least = 2;
  const long long units = d.by_item ? c->B : fa::decode_grid(c->B, (int)tiles, d.pieces, d.least);
  a->near = fa::latent_near(units, (int)rt);
  const long long grid = fa::latent_grid(units, (int)rt, a->near);
  if (grid > 0x7fffffll) return FA_ERR_SHAPE;
  d.grid = (int)grid;
  const size_t slots = d.by_item ? 0 : (size_t)fa::decode_slots(units, d.pieces) * rt * 16 * L->nb;
  L->part = ((2 * (size_t)c->B + 2) * sizeof(int) + 255) & ~(size_t)255;
  L->ml = L->part + slots * c->latent_dim * sizeof(float);
  L->bytes = d.by_item ? 0 : L->ml + slots * 2 * sizeof(float);
  return FA_OK;
}

// Tensors in launches of at most kCopyTensors.
int copy_tensors(const fa_paged_tensor* t, int count, int num_pages, const int* src, const int* dst, const int* live, int pairs,
                 hipStream_t s) {
  for (int i0 = 0; i0 < count; i0 += fa::kCopyTensors) {
    fa::CopyArgs a{};
    a.count = std::min(count - i0, fa::kCopyTensors);
    a.num_pages = num_pages;
    a.pairs = pairs;
    a.src = src;
    a.dst = dst;
    a.live = live;
    for (int i = 0; i < a.count; ++i) {
      a.data[i] = t[i0 + i].data;
      a.page_bytes[i] = t[i0 + i].page_bytes;
      a.first[i + 1] = a.first[i] + (int)((a.page_bytes[i] + fa::kCopyPiece - 1) / fa::kCopyPiece);
    }
    if (const int rc = fa::launch_copy_pages(a, s)) return rc;
  }
  return FA_OK;
}
int tensors_ok(const fa_paged_tensor* t, int count) {
  if (count < 0) return FA_ERR_SHAPE;
  if (count && !t) return FA_ERR_NULL;
  for (int i = 0; i < count; ++i) {
    if (!t[i].data) return FA_ERR_NULL;
    // (pieces of 64 tensors' pages are 32 bits together)
    if (t[i].page_bytes < 4 || t[i].page_bytes % 4 || t[i].page_bytes > (1ll << 36) || !aligned(t[i].data, 4)) return FA_ERR_SHAPE;
  }
  return FA_OK;
}

struct PlanLayout {
  size_t marks, first, list, src, dst, moved, bytes;
  int pairs;
};
bool small_plan(const fa_page_plan_call* c) {
  return c->num_pages <= fa::kPlanPages && c->N <= fa::kPlanRows && (long long)c->N * c->max_pages <= fa::kPlanEntries;
}
int plan_args(const fa_page_plan_call* c, bool fork, fa::PagePlan* a, PlanLayout* L) {
  if (!c) return FA_ERR_NULL;
  if (c->abi_version != FA_ABI_VERSION) return FA_ERR_VERSION;
  if (c->B < 1 || c->N < 1 || c->max_pages < 1 || c->page_size < 1 || c->num_pages < 1 || c->room_all < 0) return FA_ERR_SHAPE;
  if (!c->parents && c->N != c->B) return FA_ERR_SHAPE;
  if (!fork && (c->parents || c->room)) return FA_ERR_UNSUPPORTED;
  // (ranks of pages are 32 bits)
  if ((long long)c->N * c->max_pages > 0x7fffffffll || c->num_pages > 0x7fffffff - 4 * 1024) return FA_ERR_SHAPE;
  if (!c->page_table || !c->kv_lens || !c->out_table || !c->out_count || (fork && !c->out_lens)) return FA_ERR_NULL;
  if (const int rc = tensors_ok(c->tensors, c->tensor_count)) return rc;
  *a = fa::PagePlan{};
  a->table = c->page_table;
  a->kv_lens = c->kv_lens;
  a->parents = c->parents;
  a->room = c->room;
  a->keep = c->keep;
  a->room_all = c->room_all;
  a->B = c->B;
  a->N = c->N;
  a->max_pages = c->max_pages;
  a->page_size = c->page_size;
  a->num_pages = c->num_pages;
  a->out_table = c->out_table;
  a->out_lens = c->out_lens;
  a->out_count = c->out_count;
  // a fork copies a page per row at most, a compaction half of them
  L->pairs = fork ? c->N : c->num_pages / 2 + 1;
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t first = at;
    at += (n * sizeof(int) + 15) & ~(size_t)15;
    return first;
  };
  L->marks = take(small_plan(c) ? 0 : c->num_pages);
  L->first = take(fork ? c->N : 0);
  L->list = take(c->num_pages);
  L->src = take(L->pairs);
  L->dst = take(L->pairs);
  L->moved = take(1);
  L->bytes = at;
  return FA_OK;
}
int run_plan(const fa_page_plan_call* c, bool fork, void* workspace, size_t workspace_bytes, void* stream) {
  fa::PagePlan a;
  PlanLayout L;
  if (const int rc = plan_args(c, fork, &a, &L)) return rc;
  if (!workspace || workspace_bytes < L.bytes || !aligned16({workspace})) return FA_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  auto ints = [&](size_t off) { return reinterpret_cast<int*>(ws + off); };
  a.marks = small_plan(c) ? nullptr : ints(L.marks);
  a.first = ints(L.first);
  a.list = ints(L.list);
  a.pair_src = ints(L.src);
  a.pair_dst = ints(L.dst);
  a.moved = ints(L.moved);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int rc = fa::launch_page_plan(a, fork, s)) return rc;
  return copy_tensors(c->tensors, c->tensor_count, c->num_pages, a.pair_src, a.pair_dst, fork ? nullptr : a.moved, L.pairs, s);
}
