// Argument checks and kernel arguments of the C ABI calls around a KV cache
// (included by capi.hip inside its anonymous namespace).

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Rows of a strided tensor start at multiples of 16 bytes.
bool rows16(const fa_strided& t, int es) {
  const long long m = 16 / es - 1;
  return aligned(t.data, 16) && !(t.stride_b & m) && !(t.stride_h & m) && !(t.stride_t & m);
}

// Heads that one thread takes its angles through (`work`: threads of the call with
// one head each): the angles of eight pairs cost about as much as four heads'
// arithmetic, and past four there is nothing to gain; fewer where that would
// leave under three workgroups of 256 threads per unit.  GPU time in us with 1 / 2 / 4 /
// 8 heads: B4 Hq32 Hkv32 T8192 314 / 227 / 197 / 203, B1 Hq32 Hkv8 T3000 18.8 / 15.3 / 14.1 /
// 14.0, T300 5.0 / 5.2 / 6.1 / 8.0, B32 T1 4.4 / 4.8 / 5.7 / 7.6 (D = 128).
int heads_per_thread(long long work) {
  const long long per = work / (3ll * 256 * device_cus());
  return per < 1 ? 1 : per < 4 ? (int)per : 4;
}

// Threads of a rotary call per head (B T < 2^31).
long long rotary_units(fa::RotaryArgs* a, bool vec) {
  const int pairs = (a->n + 7) / 8;
  a->units = vec ? a->D / 16 : pairs + (a->D - 2 * a->n + 15) / 16;
  return (long long)a->B * a->T * a->units;
}
int rotary_groups(fa::RotaryArgs* a, long long threads, int per) {
  const int heads = a->t[0].heads + a->t[1].heads;
  a->per = std::min(per, heads);
  a->groups = cdiv(heads, a->per);
  // (one thread index; the last workgroup's included)
  return threads * a->groups > 0x7fffff00ll ? FA_ERR_SHAPE : FA_OK;
}

int rotary_args(const fa_rotary_call* c, fa::RotaryArgs* a, bool* vec) {
  if (!c) return FA_ERR_NULL;
  if (c->abi_version != FA_ABI_VERSION) return FA_ERR_VERSION;
  if (c->dtype != FA_DTYPE_BF16 && c->dtype != FA_DTYPE_F32) return FA_ERR_DTYPE;
  if (c->B < 1 || c->T < 1 || c->D < 1 || c->D > 1024 || c->count < 1 || c->count > 2) return FA_ERR_SHAPE;
  if ((long long)c->B * c->T > 0x7fffffffll) return FA_ERR_SHAPE;
  if (c->rotary.pairs < 1 || 2 * (long long)c->rotary.pairs > c->D) return FA_ERR_SHAPE;
  if (!c->rotary.inv_freq) return FA_ERR_NULL;
  if (!aligned(c->rotary.inv_freq, 8) || !aligned(c->positions, c->positions_64 ? 8 : 4)) return FA_ERR_SHAPE;
  *a = fa::RotaryArgs{};
  const int es = c->dtype == FA_DTYPE_F32 ? 4 : 2;
  *vec = c->rotary.pairs % 8 == 0 && c->D % 16 == 0;
  for (int i = 0; i < c->count; ++i) {
    const fa_strided& t = c->in[i];
    if (!t.data || !c->out[i]) return FA_ERR_NULL;
    if (t.heads < 1 || !aligned(t.data, es) || !aligned(c->out[i], es)) return FA_ERR_SHAPE;
    *vec = *vec && rows16(t, es) && aligned(c->out[i], 16);
    a->t[i] = {t.data, c->out[i], t.stride_b, t.stride_h, t.stride_t, t.heads};
  }
  if (c->count == 2 && (long long)c->in[0].heads + c->in[1].heads > 0x7fffffffll) return FA_ERR_SHAPE;
  a->B = c->B;
  a->T = c->T;
  a->D = c->D;
  a->freq = c->rotary.inv_freq;
  a->n = c->rotary.pairs;
  a->interleaved = c->rotary.interleaved != 0;
  a->inverse = c->inverse != 0;
  a->scale = c->rotary.scale;
  a->positions = c->positions;
  a->pos64 = c->positions_64 != 0;
  a->pos_stride = c->positions_stride;
  a->offset = c->offset;
  const long long threads = rotary_units(a, *vec);
  if (threads > 0x7fffff00ll) return FA_ERR_SHAPE;
  return rotary_groups(a, threads, heads_per_thread(threads * (a->t[0].heads + a->t[1].heads)));
}

int append_args(const fa_kv_append_call* c, fa::AppendArgs* a) {
  if (!c) return FA_ERR_NULL;
  if (c->abi_version != FA_ABI_VERSION) return FA_ERR_VERSION;
  if (c->cache_dtype != FA_DTYPE_BF16 && c->cache_dtype != FA_DTYPE_FP8_E4M3) return FA_ERR_DTYPE;
  const bool fp8 = c->cache_dtype == FA_DTYPE_FP8_E4M3;
  if (c->D != 32 && c->D != 64 && c->D != 128) return FA_ERR_UNSUPPORTED;
  const int Hkv = c->key.heads;
  if (c->B < 1 || c->T < 1 || Hkv < 1 || c->value.heads != Hkv || c->query.heads < 0) return FA_ERR_SHAPE;
  if (c->page_size < FA_KV_RUN || c->page_size % FA_KV_RUN || c->num_pages < 1 || c->max_pages < 1) return FA_ERR_SHAPE;
  if (!c->page_table && (c->max_pages != 1 || c->num_pages < c->B)) return FA_ERR_SHAPE;
  if (!c->key.data || !c->value.data || !c->k_cache || !c->v_cache || !c->kv_lens) return FA_ERR_NULL;
  if (fp8 && (!c->k_scale || !c->v_scale)) return FA_ERR_NULL;
  if (!rows16(c->key, 2) || !rows16(c->value, 2) || !aligned16({c->k_cache, c->v_cache})) return FA_ERR_SHAPE;
  const bool turn = c->rotary.pairs != 0;
  if (turn) {
    if (!c->rotary.inv_freq) return FA_ERR_NULL;
    if (c->rotary.pairs < 0 || 2 * (long long)c->rotary.pairs > c->D || !aligned(c->rotary.inv_freq, 8)) return FA_ERR_SHAPE;
    if (c->rotary.pairs % 8) return FA_ERR_UNSUPPORTED;
  }
  *a = fa::AppendArgs{};
  a->k = c->key.data;
  a->v = c->value.data;
  a->ksb = c->key.stride_b, a->ksh = c->key.stride_h, a->kst = c->key.stride_t;
  a->vsb = c->value.stride_b, a->vsh = c->value.stride_h, a->vst = c->value.stride_t;
  a->kc = c->k_cache;
  a->vc = c->v_cache;
  a->ks = c->k_scale;
  a->vs = c->v_scale;
  a->page_table = c->page_table;
  a->page_size = c->page_size;
  a->max_pages = c->max_pages;
  a->num_pages = c->num_pages;
  a->kv_lens = c->kv_lens;
  a->new_lens = c->new_lens;
  a->B = c->B;
  a->Hkv = Hkv;
  a->T = c->T;
  if (turn) {
    a->freq = c->rotary.inv_freq;
    a->n = c->rotary.pairs;
    a->interleaved = c->rotary.interleaved != 0;
    a->scale = c->rotary.scale;
  }
  const long long runs = ((long long)c->T + FA_KV_RUN - 2) / FA_KV_RUN + 1;
  if (runs * c->B > 0x7fffffll) return FA_ERR_SHAPE;
  const long long token_threads = runs * FA_KV_RUN * c->B * (c->D / 16);
  a->runs = (int)runs;
  auto heads = [&](long long work) {  // `work`: as heads_per_thread, keys and queries together
    a->per = std::min(heads_per_thread(work), Hkv);
    a->groups = cdiv(Hkv, a->per);
    const long long blocks = runs * c->B * a->groups;
    a->kv_blocks = (int)std::min(blocks, 0x7fffffll);
    return blocks > 0x7fffffll ? FA_ERR_SHAPE : FA_OK;
  };
  if (c->query.heads > 0) {
    if (!turn) return FA_ERR_SHAPE;  // nothing to do for the queries
    if (!c->query.data || !c->query_out) return FA_ERR_NULL;
    if (!rows16(c->query, 2) || !aligned(c->query_out, 16)) return FA_ERR_SHAPE;
    fa::RotaryArgs& q = a->q;
    q.t[0] = {c->query.data, c->query_out, c->query.stride_b, c->query.stride_h, c->query.stride_t, c->query.heads};
    q.B = c->B;
    q.T = c->T;
    q.D = c->D;
    q.freq = a->freq;
    q.n = a->n;
    q.interleaved = a->interleaved;
    q.scale = a->scale;
    q.kv_lens = c->kv_lens;
    const long long threads = rotary_units(&q, true), work = token_threads * Hkv + threads * c->query.heads;
    const int rc = heads(work);
    return rc ? rc : rotary_groups(&q, threads, heads_per_thread(work));
  }
  return heads(token_threads * Hkv);
}

struct DecodeLayout {
  int nq;               // 16-row query blocks per work item
  bool general;         // score modifiers, or a block's rows see different keys
  bool stream;          // cache reads past the caches
  size_t part, ml, bytes;
};

int decode_args(const fa_params* p, const fa_fp8_cache* kv, int cus, fa::DecodeArgs* a, DecodeLayout* L) {
  if (!p || !kv) return FA_ERR_NULL;
  if (p->abi_version != FA_ABI_VERSION) return FA_ERR_VERSION;
  if (p->dtype != FA_DTYPE_FP8_E4M3) return FA_ERR_DTYPE;
  if (p->D != 32 && p->D != 64 && p->D != 128) return FA_ERR_UNSUPPORTED;
  if (p->B < 1 || p->Hq < 1 || p->Hkv < 1 || p->Hq % p->Hkv || p->Sq < 1 || p->Skv < 1 ||
      p->Skv > 0x7fffffff - 2 * fa::kTileKeys)
    return FA_ERR_SHAPE;
  auto number = [](float x) { return x == 0.f || (x >= FLT_MIN && x <= FLT_MAX); };
  if (!number(p->softcap) || !number(p->scale)) return FA_ERR_SHAPE;
  if (p->q_doc_ids || p->kv_doc_ids || p->doc_start || p->doc_end || p->kv_num_blocks || p->kv_indices ||
      p->full_kv_num_blocks || p->full_kv_indices)
    return FA_ERR_UNSUPPORTED;
  if (kv->page_size < FA_KV_RUN || kv->page_size % FA_KV_RUN || kv->num_pages < 1 || kv->max_pages < 1) return FA_ERR_SHAPE;
  if (!kv->page_table && (kv->max_pages != 1 || kv->num_pages < p->B)) return FA_ERR_SHAPE;
  if ((long long)kv->max_pages * kv->page_size < p->Skv) return FA_ERR_SHAPE;
  const long long runs = (long long)kv->num_pages * p->Hkv * (kv->page_size / FA_KV_RUN);
  if (runs > 0x7fffffffll) return FA_ERR_SHAPE;  // run indices are 32 bits (2^36 token rows)
  if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale) return FA_ERR_NULL;
  if (!aligned16({kv->k, kv->v})) return FA_ERR_SHAPE;
  *a = fa::DecodeArgs{};
  const int g = p->Hq / p->Hkv;
  const long long rows = (long long)g * p->Sq;
  if (rows > 0x7ffffffll || (long long)p->B * p->Hkv > 0x7ffffffll / rows) return FA_ERR_SHAPE;
  // tiles that a row walks at most: all of its keys', or the window's
  // (a window of at least all keys is none)
  const int left = p->window_left < 0 || p->window_left >= p->Skv ? -1 : p->window_left;
  long long tiles = (p->Skv + fa::kTileKeys - 1) / fa::kTileKeys;
  if (left >= 0) tiles = std::min(tiles, ((long long)left + p->Sq + fa::kTileKeys - 2) / fa::kTileKeys + 1);
  L->nq = fa::decode_blocks(rows, p->B * (long long)p->Hkv, tiles);
  const long long rt = (rows + 16 * L->nq - 1) / (16 * L->nq);
  const long long items = p->B * (long long)p->Hkv * rt;
  if (items * tiles > 0x7fffffffll - (1 << 20)) return FA_ERR_SHAPE;  // tile numbers of a call are 32 bits
  a->k = static_cast<const uint8_t*>(kv->k);
  a->v = static_cast<const uint8_t*>(kv->v);
  a->ks = kv->k_scale;
  a->vs = kv->v_scale;
  a->page_table = kv->page_table;
  a->kv_lens = kv->kv_lens;
  a->q_lens = kv->q_lens;
  a->B = p->B;
  a->Hkv = p->Hkv;
  a->Sq = p->Sq;
  a->g = g;
  a->page_runs = kv->page_size / FA_KV_RUN;
  a->max_pages = kv->max_pages;
  a->num_pages = kv->num_pages;
  a->cap = p->Skv;
  a->win_left = left;
  // (the first of Sq queries stands Sq - 1 before the last key at most)
  a->win_right = p->window_right < 0 || p->window_right >= p->Sq - 1 ? -1 : p->window_right;
  // A row of an item sees the item's keys or, padded, none, unless there are several queries
  // and a window: then NaN values must be kept from the rows that do not see their key, which
  // costs registers that the plain walk has no room for (D = 128: with it alone 138 for 126, three waves per
  // SIMD for four; 256 mixed lengths to 257 tiles 58.3 us for 54.5. These kernels, with the
  // modifiers too, take 146).
  L->general = p->alibi_slopes || p->softcap > 0.f || (p->Sq > 1 && (left >= 0 || a->win_right >= 0));
  a->scale = p->scale == 0.f ? 1.0f / sqrtf((float)p->D) : p->scale;
  a->scale_log2 = a->scale * fa::kLog2e;
  a->softcap = p->softcap;
  a->alibi = p->alibi_slopes;
  a->rt = (int)rt;
  // How the walk is cut (csrc/decode_index.h), from the longest walk that the
  // sizes allow; GPU time per call in us in replayed graphs, D = 128 unless named, by item in
  // eight waves / in pieces of four.  One workgroup per item, without a second launch, where
  // walks are short (8 items of 16 tiles 7.2 / 10.7, 128 of 34 11.4 / 14.8, of up to 61 16.8 / 16.6)
  // or where the kv heads fill the units and no walk is very long (256 of 121 45.2 / 49.8, of up to
  // 118 30.3 / 30.8, most of them short 25.5 / 20.1; 512 of 68 37.5 / 38.8, of up to 127 59.4 / 56.1,
  // D = 64 512 of 65 19.9 / 22.3).  Pieces beyond: 8 of 126 25.6 / 13.0, 128 of up to 122 27.8 / 23.2,
  // of 125 29.8 / 28.7, 64 of 127 26.7 / 19.9, 32 of 127 with two blocks of rows 27.4 / 21.2, 256 of
  // mixed lengths to 257 61 / 55; they lose on many equal long rows (D = 64 256 of 513 88 / 96) and
  // many items (1024 rows to 156 with four heads 262 / 298), and keep one long row among many from
  // being the call's time (300 rows with one head to 981 317 / 96, one of 3125 among 299 of 16
  // 540 / 37; 1024 to 254 131 / 126). Past 1024 rows each workgroup's search for its piece costs
  // more than that, and the join's launch of a wave per query row has no room for more than 2^26 - 4
  // of those (2^32 threads).
  a->by_item = tiles <= 48 || ((long long)p->B * p->Hkv >= cus && tiles <= 128) || p->B > 64 * fa::kMostLaneRows ||
               p->B * (long long)p->Hkv * rows > (1 << 26) - 4;
  // At most four pieces per unit (two where the rows are equally long: decode_unit).
  a->pieces = 4 * cus;
  // At least 16 tiles a piece, four per wave, so that the merge stays short (8 of 500
  // 16.5 us, with 8 tiles 18.8); 8 where that makes at most 16 pieces (8 of 126 12.4, 11.8).
  a->least = tiles <= 128 ? 8 : 16;
  // A call that reads more than fits the 256 MB last-level cache beside other data
  // reads past it (through / past the caches: 64 items of 1024 tiles 107 / 97 us, 256 mixed
  // 61 / 56, 128 of 127, 133 MB, 36 / 29.5); smaller ones may find theirs there (100 MB 24.4 / 27.5,
  // 33 MB 14.8 / 15.7, D = 64 51 MB 14.3 / 15.2).
  L->stream = 2ll * p->B * p->Hkv * tiles * fa::kTileKeys * p->D > 112ll << 20;
  const long long grid = a->by_item ? items : fa::decode_grid(items, (int)tiles, a->pieces, a->least);
  if (grid > 0x7fffffll) return FA_ERR_SHAPE;
  a->grid = (int)grid;
  const size_t slots = a->by_item ? 0 : (size_t)fa::decode_slots(grid, a->pieces) * 16 * L->nq;
  L->part = ((2 * (size_t)p->B + 2) * sizeof(int) + 255) & ~(size_t)255;
  L->ml = L->part + slots * p->D * sizeof(float);
  L->bytes = a->by_item ? 0 : L->ml + slots * 2 * sizeof(float);
  return FA_OK;
}
