// extern "C" entry points of the paged 4-bit serving operators (declared in include/dsv2.h).
// Same rules as api.cu (which this file follows in the translation unit): arguments are
// checked here, nothing allocates device memory or synchronises.

namespace {

// up to here a shared projection with one partial shares a launch with the second product (n 3648, k 2048,
// shared / separate: 1 token 7.3 / 9.2 us, 9 of rank 16 8.1 / 15.4, 16 of rank 32 11.5 / 17.8, 16 of rank
// 64 18.8 / 27.8; 32 of rank 32 15.8 / 16.2, of rank 128 36 / 23)
constexpr int kLoraGemvTokens = 16;
// The projection and its adapters are one GEMM above 256 tokens where the adapters' steps are few beside the
// projection's: it pays a pass that orders the tokens and a step for every two pieces of 16 ranks in a tile, and
// saves the fp32 partials.  The limit is 16 + k / 128 pieces up to 512 tokens and half as many again above, where the
// partials weigh more.  One GEMM / separate launches, us, (pieces):
//   k 2048, n 3648: 257 tokens of rank 32 with 10 adapters 29.2 / 29.3 (20), with 16 30.9 / 29.6 (32), with 42 54 / 32 (84);
//     400 of rank 64 with 10 33 / 35 (28), with 25 45 / 37 (68); 768 of rank 64 with 32 46 / 54 (44), with 64 62 / 59 (88);
//     1024 of rank 32 with 64 37 / 39 (34), with 128 52 / 45 (66); 4001 with 6 71 / 133 (2)
//   k 256, n 3648: 300 of rank 16 with 18 19.6 / 19.9 (16), with 30 24.6 / 21.0 (26); 1024 with 102 31 / 34 (26), with 170
//     40.0 / 38.6 (43)
//   k 10944, n 2048, rank 128: 300 with 12 102 / 152 (88), with 37 191 / 187 (256)
// Up to 256 tokens the projection reads its weights once either way.
constexpr int kLoraGemmTokens = 256;
bool lora_one_gemm(long long tokens, long long adapters, long long rank, long long k) {
  // adapters of a tile, if the tokens are spread over them evenly, and their pieces
  const long long in_tile = std::min(adapters, adapters * kLgM / tokens + 1), pieces = in_tile * ((rank + kLgPiece - 1) / kLgPiece);
  return tokens > kLoraGemmTokens && k % 64 == 0 && 2 * pieces < (tokens > 2 * kLoraGemmTokens ? 3 : 2) * (16 + k / 128);
}
// fewest units of a CTA (64 positions): one row of 512 with 1 / 4 / 16: 13.9 / 13.6 / 14.8 us, of 64:
// 11.7 / 10.3 / 10.3
constexpr int kQ4MinUnits = 4;

// rows of a latent4 call: [n, 576] bf16 with 16-byte aligned rows
int latent4_args(const char* what, const void* rows, int64_t row_stride, const int64_t* slots, int64_t n,
                 const void* cache, int64_t n_blocks) {
  if (n < 0) return fail(DSV2_ERR_INVALID, "%s: n %lld", what, (long long)n);
  if (n > 0 && (!rows || !slots || !cache)) return fail(DSV2_ERR_INVALID, "%s: null pointer", what);
  if (n > 0x7fffffffLL) return fail(DSV2_ERR_UNSUPPORTED, "%s: n %lld exceeds one launch", what, (long long)n);
  if (n_blocks <= 0) return fail(DSV2_ERR_INVALID, "%s: n_blocks %lld", what, (long long)n_blocks);
  if (!aligned16(rows) || !aligned16(cache) || row_stride % 8 || row_stride < 576)
    return fail(DSV2_ERR_INVALID, "%s: rows of 576 elements and the cache must be 16-byte aligned", what);
  return DSV2_OK;
}

}  // namespace

extern "C" {

int dsv2_page_plan(const dsv2_page_plan_args* a, void* stream) {
  if (!a || !a->free_ring || !a->ring_in || !a->ring_out || !a->cu_new || !a->counts || !a->sync)
    return fail(DSV2_ERR_INVALID, "page_plan: null pointer");
  if (a->requests < 0 || a->width <= 0 || a->ring_size <= 0 || a->token_capacity < 0 || a->table_stride < a->width)
    return fail(DSV2_ERR_INVALID, "page_plan: requests %d width %d ring %lld capacity %d", a->requests, a->width,
                (long long)a->ring_size, a->token_capacity);
  if (a->requests > 0 && (!a->cached || !a->fresh || !a->lens || !a->block_table))
    return fail(DSV2_ERR_INVALID, "page_plan: null pointer");
  if (a->token_capacity > 0 && (!a->token_row || !a->positions || !a->slots))
    return fail(DSV2_ERR_INVALID, "page_plan: null pointer");
  if (a->page_size <= 0 || a->page_size % DSV2_L4_BLOCK_TOKENS)
    return fail(DSV2_ERR_INVALID, "page_plan: page_size %d (a positive multiple of %d)", a->page_size,
                DSV2_L4_BLOCK_TOKENS);
  if (static_cast<int64_t>(a->width) * a->page_size > 0x7fffffffLL)
    return fail(DSV2_ERR_UNSUPPORTED, "page_plan: a table row of %d pages of %d tokens exceeds 2^31 tokens", a->width,
                a->page_size);
  const char* c = static_cast<const char*>(a->cached);
  const char* l = reinterpret_cast<const char*>(a->lens);
  const int64_t c_bytes = static_cast<int64_t>(a->requests) * (a->cached_is64 ? 8 : 4), l_bytes = static_cast<int64_t>(a->requests) * 4;
  if (a->requests > 0 && c < l + l_bytes && l < c + c_bytes)
    return fail(DSV2_ERR_INVALID, "page_plan: lens must not overlap cached");
  int sms = 0;
  if (int rc = ensure_init(&sms)) return rc;
  PagePlanParams p = {};
  p.cached = a->cached;
  p.cached64 = a->cached_is64 != 0;
  p.fresh = a->fresh;
  p.requests = a->requests;
  p.page = a->page_size;
  p.table = a->block_table;
  p.table_stride = a->table_stride;
  p.width = a->width;
  p.ring = a->free_ring;
  p.ring_size = a->ring_size;
  p.ring_in = reinterpret_cast<const long long*>(a->ring_in);
  p.ring_out = reinterpret_cast<long long*>(a->ring_out);
  p.capacity = a->token_capacity;
  p.token_row = a->token_row;
  p.positions = reinterpret_cast<long long*>(a->positions);
  p.slots = reinterpret_cast<long long*>(a->slots);
  p.cu_new = a->cu_new;
  p.lens = a->lens;
  p.counts = a->counts;
  p.sync = a->sync;
  return check_launch(launch_page_plan(p, sms, static_cast<cudaStream_t>(stream)), "page_plan");
}

int dsv2_latent4_write(const void* rows, int64_t row_stride, const int64_t* slots, int64_t n, void* cache,
                       int64_t n_blocks, void* stream) {
  if (int rc = latent4_args("latent4_write", rows, row_stride, slots, n, cache, n_blocks)) return rc;
  if (n == 0) return DSV2_OK;
  Latent4Params p = {};
  p.rows = static_cast<const bf16*>(rows);
  p.row_stride = row_stride;
  p.slots = reinterpret_cast<const long long*>(slots);
  p.n = n;
  p.cache = static_cast<unsigned char*>(cache);
  p.n_blocks = n_blocks;
  return check_launch(launch_latent4_write(p, static_cast<cudaStream_t>(stream)), "latent4_write");
}

int dsv2_latent4_read(const void* cache, int64_t n_blocks, const int64_t* slots, int64_t n, void* out,
                      int64_t out_row_stride, void* stream) {
  if (int rc = latent4_args("latent4_read", out, out_row_stride, slots, n, cache, n_blocks)) return rc;
  if (n == 0) return DSV2_OK;
  Latent4Params p = {};
  p.out = static_cast<bf16*>(out);
  p.row_stride = out_row_stride;
  p.slots = reinterpret_cast<const long long*>(slots);
  p.n = n;
  p.cache = static_cast<unsigned char*>(const_cast<void*>(cache));
  p.n_blocks = n_blocks;
  return check_launch(launch_latent4_read(p, static_cast<cudaStream_t>(stream)), "latent4_read");
}

int dsv2_mla_decode_q4(const dsv2_mla_decode_q4_args* a, void* stream) {
  if (!a) return fail(DSV2_ERR_INVALID, "mla_decode_q4: null pointer");
  if (a->rows < 0 || a->seqs <= 0 || a->width <= 0 || a->n_blocks <= 0 || a->table_stride < a->width)
    return fail(DSV2_ERR_INVALID, "mla_decode_q4: rows %d seqs %d width %d blocks %lld", a->rows, a->seqs, a->width,
                (long long)a->n_blocks);
  if (a->rows == 0) return DSV2_OK;
  if (!a->q_abs || !a->q_pe || !a->cache || !a->block_table || !a->positions || !a->o_lat || !a->o_part ||
      !a->ml_part || !a->cuts)
    return fail(DSV2_ERR_INVALID, "mla_decode_q4: null pointer");
  if (a->part_slots < 2) return fail(DSV2_ERR_INVALID, "mla_decode_q4: %d partial slots (at least 2)", a->part_slots);
  if (a->page_size <= 0 || a->page_size % DSV2_L4_BLOCK_TOKENS)
    return fail(DSV2_ERR_INVALID, "mla_decode_q4: page_size %d (a positive multiple of %d)", a->page_size,
                DSV2_L4_BLOCK_TOKENS);
  if (static_cast<int64_t>(a->width) * a->page_size > 0x7fffffffLL)
    return fail(DSV2_ERR_UNSUPPORTED, "mla_decode_q4: a table row of %d pages of %d tokens exceeds 2^31 tokens",
                a->width, a->page_size);
  if (!aligned16(a->q_abs) || !aligned16(a->q_pe) || !aligned16(a->cache) || !aligned16(a->o_lat) ||
      !aligned16(a->o_part) || !aligned16(a->ml_part) || !aligned16(a->cuts))
    return fail(DSV2_ERR_INVALID, "mla_decode_q4: operands must be 16-byte aligned");
  int sms = 0;
  if (int rc = ensure_init(&sms)) return rc;
  MlaQ4Params p = {};
  p.q_abs = static_cast<const bf16*>(a->q_abs);
  p.q_pe = static_cast<const bf16*>(a->q_pe);
  p.cache = static_cast<const unsigned char*>(a->cache);
  p.n_blocks = a->n_blocks;
  p.table = a->block_table;
  p.table_stride = a->table_stride;
  p.width = a->width;
  p.seqs = a->seqs;
  p.page_blocks = a->page_size / DSV2_L4_BLOCK_TOKENS;
  p.positions = reinterpret_cast<const long long*>(a->positions);
  p.seq_rows = a->seq_rows;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.o_lat = static_cast<bf16*>(a->o_lat);
  p.rows = a->rows;
  p.min_units = kQ4MinUnits;
  p.o_part = a->o_part;
  p.ml_part = a->ml_part;
  p.part_slots = a->part_slots;
  p.cuts = reinterpret_cast<int4*>(a->cuts);
  if (!a->seq_rows && a->seqs < a->rows)
    return fail(DSV2_ERR_INVALID, "mla_decode_q4: %d query rows, %d table rows (pass seq_rows)", a->rows, a->seqs);
  return check_launch(launch_mla_q4(p, sms, static_cast<cudaStream_t>(stream)), "mla_decode_q4");
}

int dsv2_lora(const dsv2_lora_args* a, void* stream) {
  if (!a) return fail(DSV2_ERR_INVALID, "lora: null pointer");
  if (a->tokens < 0 || a->adapters < 0 || a->n_base < 0 || a->ids_len < 0)
    return fail(DSV2_ERR_INVALID, "lora: tokens %d adapters %d partials %d", a->tokens, a->adapters, a->n_base);
  if (a->tokens == 0) return DSV2_OK;
  // a long run of tokens: one GEMM over the tokens in adapter order, no partials
  const bool fused = a->w && a->xs && a->lists && a->y_dtype == DSV2_BF16 && lora_one_gemm(a->tokens, a->adapters, a->rank, a->k);
  if (a->w && !fused && (!a->base || a->n_base < 1)) return fail(DSV2_ERR_INVALID, "lora: w needs base and n_base for its partials");
  if (!a->x || !a->ids || !a->y || !a->low || (a->adapters > 0 && (!a->a || !a->b || !a->ranks || !a->scales)) ||
      (a->n_base > 0 && !a->base))
    return fail(DSV2_ERR_INVALID, "lora: null pointer");
  if (a->low_parts < 1 || a->low_parts > 64 || (a->tokens > kLoraTile && !a->order))
    return fail(DSV2_ERR_INVALID, "lora: low_parts %d (1 .. 64), order is required above %d tokens", a->low_parts, kLoraTile);
  if (!a->token_row && a->ids_len < a->tokens)
    return fail(DSV2_ERR_INVALID, "lora: %d ids for %d tokens (pass token_row)", a->ids_len, a->tokens);
  if (a->k <= 0 || a->n <= 0 || a->rank <= 0 || a->k % 8 || a->n % 8 || a->rank % 8 || a->rank > 128)
    return fail(DSV2_ERR_UNSUPPORTED, "lora: k %d, n %d, rank %d (multiples of 8, rank at most 128)", a->k, a->n, a->rank);
  if (a->y_dtype != DSV2_BF16 && a->y_dtype != DSV2_F32) return fail(DSV2_ERR_UNSUPPORTED, "lora: y dtype %d", a->y_dtype);
  if (!aligned16(a->x) || !aligned16(a->a) || !aligned16(a->b) || !aligned16(a->base) || !aligned16(a->low) ||
      !aligned16(a->order) || !aligned16(a->y) || a->x_row_stride % 8 || a->base_part_stride % 4 || a->base_row_stride % 4 ||
      a->y_row_stride % (a->y_dtype == DSV2_F32 ? 4 : 8))
    return fail(DSV2_ERR_INVALID, "lora: operands must be 16-byte aligned rows");
  if (!aligned16(a->xs) || !aligned16(a->lists)) return fail(DSV2_ERR_INVALID, "lora: xs and lists must be 16-byte aligned");
  const bool few = a->w && a->tokens <= kLoraGemvTokens && a->n_base == 1;
  if (a->w && !few && a->k % 64)   // dsv2_linear's condition, told before anything is launched
    return fail(DSV2_ERR_UNSUPPORTED, "lora: k %d: with w and more than %d tokens or pieces of k, a multiple of 64", a->k,
                kLoraGemvTokens);
  int sms = 0;
  if (int rc = ensure_init(&sms)) return rc;
  if ((few || fused) && (!aligned16(a->w) || a->w_row_stride % 8 || a->w_row_stride < a->k))
    return fail(DSV2_ERR_INVALID, "lora: w must be 16-byte aligned rows");
  if (a->w && !fused && !few) {
    dsv2_linear_args l = {};
    l.w = a->w;
    l.w_row_stride = a->w_row_stride;
    l.n_rows = a->n;
    l.k = a->k;
    l.x = a->x;
    l.x_row_stride = a->x_row_stride;
    l.y = const_cast<float*>(a->base);
    l.y_row_stride = a->base_row_stride;
    l.epilogue = DSV2_EPI_STORE_F32;
    l.n_groups = 1;
    l.n_tokens = a->tokens;
    l.w_group_rows = a->n;
    l.x_group_rows = a->tokens;
    l.k_splits = a->n_base;
    l.y_split_stride = a->base_part_stride;
    if (int rc = dsv2_linear(&l, DSV2_FAMILY_BATCH, stream)) return rc;
  }
  LoraParams p = {};
  p.x = static_cast<const bf16*>(a->x);
  p.x_row_stride = a->x_row_stride;
  p.a = static_cast<const bf16*>(a->a);
  p.b = static_cast<const bf16*>(a->b);
  p.ids = a->ids;
  p.token_row = a->token_row;
  p.ranks = a->ranks;
  p.scales = a->scales;
  p.adapters = a->adapters;
  p.rank = a->rank;
  p.tokens = a->tokens;
  p.k = a->k;
  p.n = a->n;
  p.ids_len = a->ids_len;
  p.low = a->low;
  p.low_parts = a->low_parts;
  p.order = a->tokens > kLoraTile ? a->order : nullptr;
  p.base = a->base;
  p.base_parts = a->n_base;
  p.base_part_stride = a->base_part_stride;
  p.base_row_stride = a->base_row_stride;
  p.y = a->y;
  p.y_f32 = a->y_dtype == DSV2_F32;
  p.y_row_stride = a->y_row_stride;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few) {
    p.w = static_cast<const bf16*>(a->w);
    p.w_row_stride = a->w_row_stride;
    p.base_parts = 0;
  }
  if (!fused) return check_launch(launch_lora(p, sms, st), "lora");
  p.xs = static_cast<bf16*>(a->xs);
  p.lists = a->lists;
  p.base_parts = 0;
  const int n_tile = lora_gemm_tile(a->tokens, a->n, sms);
  const uint64_t T = static_cast<uint64_t>(a->tokens), N = static_cast<uint64_t>(a->n), K = static_cast<uint64_t>(a->k);
  const uint64_t ws = static_cast<uint64_t>(a->w_row_stride) * 2;
  CUtensorMap tm_x, tm_w;
  if (int rc = tensor_map_3d(a->xs, K, T, 1, K * 2, T * K * 2, kLgRows, &tm_x)) return rc;
  if (int rc = tensor_map_3d(a->w, K, N, 1, ws, N * ws, static_cast<uint32_t>(n_tile / 2), &tm_w)) return rc;
  if (int rc = check_launch(launch_lora_rows(p, sms, st), "lora: rows")) return rc;
  return check_launch(launch_lora_gemm(p, tm_x, tm_w, n_tile, sms, st), "lora: gemm");
}

}  // extern "C"
