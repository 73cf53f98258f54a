// extern "C" boundary of the paged key/value cache: argument checks and launches.  As in capi.cu nothing here allocates device
// memory, synchronises the device or throws.
#include "capi_common.cuh"

#include <algorithm>
#include <mutex>

#include "attn_cache.cuh"
#include "attn_cache_tile.cuh"

namespace {

using chitu::cuda_fail;
using chitu::fail;

constexpr int64_t kHeaderBytes = CHITU_SPLITKV_HEADER_BYTES;
constexpr int kMaxDevices = 64;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int page_shift_of(int page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// Element strides of a [tokens, heads, D] tensor: multiples of 16 bytes, positive where the extent is above one.
bool strides_fit(const int64_t* st, int64_t extent0, int64_t extent1, int bytes) {
  return (extent0 <= 1 || (st[0] > 0 && (st[0] * bytes) % 16 == 0)) && (extent1 <= 1 || (st[1] > 0 && (st[1] * bytes) % 16 == 0));
}

int check_cache(const chitu_b200_kv_cache* c, const char* what) {
  if (!c) return fail(CHITU_E_INVALID, "%s: null cache descriptor", what);
  if (!c->k || !c->v || !c->block_table || !c->lens || !c->cu_seqlens) return fail(CHITU_E_INVALID, "%s: null pointer in the cache descriptor", what);
  if (c->format != CHITU_CACHE_16BIT && c->format != CHITU_CACHE_E4M3) return fail(CHITU_E_UNSUPPORTED, "%s: pages must be 16-bit or e4m3", what);
  if (c->format == CHITU_CACHE_E4M3 && (!c->k_scale || !c->v_scale)) return fail(CHITU_E_INVALID, "%s: 8-bit pages need k_scale and v_scale", what);
  if (page_shift_of(c->page_size) < 0) return fail(CHITU_E_UNSUPPORTED, "%s: page_size must be 16, 32, 64, 128 or 256 (got %d)", what, c->page_size);
  if (c->batch < 0 || c->table_width < 1 || c->n_pages < 1 || c->heads < 1 || c->table_stride < 0)
    return fail(CHITU_E_INVALID, "%s: bad batch, table or page count", what);
  if (static_cast<int64_t>(c->table_width) * c->page_size > (1 << 30))
    return fail(CHITU_E_UNSUPPORTED, "%s: a table may name at most 2^30 tokens per sequence", what);
  const int es = c->format == CHITU_CACHE_E4M3 ? 1 : 2;
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(CHITU_E_INVALID, "%s: pages must be 16-byte aligned", what);
  for (const int64_t* st : {c->k_strides, c->v_strides}) {
    const int64_t extents[3] = {c->n_pages, c->page_size, c->heads};
    for (int i = 0; i < 3; ++i)
      if (extents[i] > 1 && (st[i] <= 0 || (st[i] * es) % 16 != 0))
        return fail(CHITU_E_INVALID, "%s: cache stride[%d] = %lld must be positive and a multiple of 16 bytes", what, i, static_cast<long long>(st[i]));
  }
  return CHITU_OK;
}

int check_table(const float* table, int64_t rows, int rot, const char* what) {
  if (!aligned16(table)) return fail(CHITU_E_INVALID, "%s: the rotary table must be 16-byte aligned", what);
  if (rot < 16 || (rot & 15) || rows < 0) return fail(CHITU_E_UNSUPPORTED, "%s: rotated channels must be a positive multiple of 16 (got %d)", what, rot);
  return CHITU_OK;
}

// More than 48 KB of shared memory is granted once per device and kernel.
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, bool (&done)[kMaxDevices]) {
  static std::mutex mu;
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  std::lock_guard<std::mutex> lock(mu);
  if (!done[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done[dev] = true;
  }
  return e;
}

constexpr int kSms = 148;

// Appended tokens per sequence up to which eight threads take all of them (kv_append_few_kernel), about a microsecond each.  That
// against the form for many, whose time hardly depends on their number up to a page: 1 sequence, 5 tokens 6.4 : 3.1 us, 8 sequences, 4 and
// 5 tokens 5.6 : 4.9 and 6.6 : 5.0; 64 sequences, 4 and 12 tokens 5.7 : 13.0 and 13.5 : 13.9; 256 sequences, 4 and 16 tokens 8.3 : 38
// and 34 : 44 (8-bit pages of 64, 48 heads).
constexpr int kAppendFew = 4;

// Tensor map over a pool: channels, heads, tokens of a page, pages; a box is 128 bytes of the channels by
// box_tokens of a page, its rows swizzled (the layout of the matrix operands) or as they are.
int make_cache_map(CUtensorMap* map, const chitu_b200_kv_cache* c, const void* base, const int64_t* st, int box_tokens, bool swizzled,
                   const char* name) {
  auto encode = chitu::get_encode_fn();
  if (!encode) return fail(CHITU_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const bool eight = c->format == CHITU_CACHE_E4M3;
  const int es = eight ? 1 : 2;
  // (a dimension of extent 1 never advances; give it any legal stride)
  auto bytes = [&](int i, int64_t extent) { return extent == 1 ? cuuint64_t{256} : static_cast<cuuint64_t>(st[i]) * es; };
  cuuint64_t dims[4] = {128, static_cast<cuuint64_t>(c->heads), static_cast<cuuint64_t>(c->page_size), static_cast<cuuint64_t>(c->n_pages)};
  cuuint64_t strides[3] = {bytes(2, c->heads), bytes(1, c->page_size), bytes(0, c->n_pages)};
  cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / es), 1, static_cast<cuuint32_t>(box_tokens), 1};
  cuuint32_t elem[4] = {1, 1, 1, 1};
  CUresult r = encode(map, eight ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box,
                      elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(CHITU_E_CUDA, "%s: cuTensorMapEncodeTiled failed with CUresult %d", name, static_cast<int>(r));
  return CHITU_OK;
}

// Grid of the rows kernel: all CTAs resident at once, or as many as there can be runs of a tile.
constexpr int kRowsGrid = kSms * 3;
int64_t rows_workspace_bytes() { return kHeaderBytes + static_cast<int64_t>(kRowsGrid) * 2 * chitu::kRowsPieceFloats * 4; }

template <bool kFp16, bool kEightBit>
cudaError_t launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const chitu::CacheAttnParams& p, int max_q, int max_kv, cudaStream_t st) {
  static bool done[kMaxDevices] = {};
  constexpr int smem = chitu::RowsShape<kEightBit>::smem;
  cudaError_t e = allow_smem(chitu::attn_cache_rows_kernel<kFp16, kEightBit>, smem, done);
  if (e != cudaSuccess) return e;
  const int64_t items = static_cast<int64_t>(p.batch) * p.heads_kv * ((static_cast<int64_t>(max_q) * p.group + 15) / 16);
  const int64_t runs = items * ((max_kv + chitu::RowsShape<kEightBit>::tile - 1) / chitu::RowsShape<kEightBit>::tile);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kSms * chitu::RowsShape<kEightBit>::ctas_per_sm, runs)));
  chitu::attn_cache_rows_kernel<kFp16, kEightBit><<<grid, chitu::kRowsThreads, smem, st>>>(tk, tv, p);
  return cudaGetLastError();
}

// Which kernel a call takes.  16 query rows of a key head (tokens x heads that share it) are one tile of the rows kernel, which
// reads the cache once per 16 rows (from the L2 cache where two tiles of rows are in step).  Rows against tile kernel, 8-bit
// pages, 8 key heads: 32 rows, 64 sequences of 500 keys 40 : 65 us, of 16000 keys 655 : 778, 8 of 4000 36 : 40, one of 16000 35 : 33;
// 48 rows, 64 of 500 69 : 79 but of 16000 970 : 816; 64 rows, 8 of 4000 56 : 40, 64 of 16000 1291 : 823.
bool takes_tile_kernel(int max_q, int group) { return static_cast<int64_t>(max_q) * group > 32 && group <= 128; }
// Shortest run of a CTA, in tiles of 128 keys (a block's fixed cost is four): 1, 2, 4 and 8 of them take, 8-bit pages of 64, 40 queries over 4000
// keys, 2 key heads of 4 query heads: 30.2, 24.7, 24.0, 28.6 us; 64 over 1000, 8 key heads: 20.0, 19.9, 22.0, 27.7; 4 x 64 over
// 500, 4 key heads: 18.2, 19.9, 22.1, 19.8; 300 over 900, twice, 2 key heads of 2: 20.3, 19.9, 22.4, 28.1.
constexpr int kTileMinTiles = 2;
int64_t tile_workspace_bytes() { return kHeaderBytes + static_cast<int64_t>(kSms) * (2 * chitu::kTilePieceFloats * 4 + sizeof(chitu::TileJoin)); }

template <bool kFp16, bool kEightBit>
cudaError_t launch_tile(const CUtensorMap& tk, const CUtensorMap& tv, const chitu::CacheAttnParams& p, cudaStream_t st) {
  static bool done[kMaxDevices] = {};
  constexpr int smem = chitu::TileShape<kEightBit>::smem;
  cudaError_t e = allow_smem(chitu::attn_cache_tile_kernel<kFp16, kEightBit>, smem, done);
  if (e != cudaSuccess) return e;
  chitu::attn_cache_tile_kernel<kFp16, kEightBit><<<kSms, chitu::kTileThreads, smem, st>>>(tk, tv, p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kSms - 1, chitu::kTileRows / 32);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, chitu::attn_cache_join_kernel<kFp16>, p, kSms);
}

template <bool kFp16, bool kEightBit, int kThreads>
cudaError_t launch_append_of(const chitu::AppendParams& p, dim3 grid, cudaStream_t st) {
  static bool done[kMaxDevices] = {};
  constexpr int smem = chitu::AppendShape<kThreads>::smem;
  cudaError_t e = allow_smem(chitu::kv_append_kernel<kFp16, kEightBit, kThreads>, smem, done);
  if (e != cudaSuccess) return e;
  chitu::kv_append_kernel<kFp16, kEightBit, kThreads><<<grid, kThreads, smem, st>>>(p);
  return cudaGetLastError();
}
template <bool kFp16, bool kEightBit>
cudaError_t launch_append(const chitu::AppendParams& p, int threads, dim3 grid, cudaStream_t st) {
  if constexpr (kEightBit) {
    if (threads == 512) return launch_append_of<kFp16, kEightBit, 512>(p, grid, st);
    if (threads == 1024) return launch_append_of<kFp16, kEightBit, 1024>(p, grid, st);
  }
  return launch_append_of<kFp16, kEightBit, 256>(p, grid, st);
}

}  // namespace

extern "C" {

int chitu_b200_rotary(const void* const* x, void* const* out, const int64_t* x_strides, const int64_t* out_strides,
                      const int* heads, int n, int64_t tokens, int head_dim, int rot, int dtype, const void* positions,
                      int positions_are_int64, const float* table, int64_t table_rows, int interleaved, void* stream) {
  if (!x || !out || !x_strides || !out_strides || !heads || !positions || !table) return fail(CHITU_E_INVALID, "rotary: null pointer");
  if (n < 1 || n > 3) return fail(CHITU_E_UNSUPPORTED, "rotary: one to three tensors (got %d)", n);
  if (dtype < 0 || dtype > 2) return fail(CHITU_E_UNSUPPORTED, "rotary: dtype must be bf16, fp16 or fp32");
  if (head_dim < 16 || head_dim > 512 || (head_dim & 15)) return fail(CHITU_E_UNSUPPORTED, "rotary: head_dim must be a multiple of 16 up to 512 (got %d)", head_dim);
  if (rot > head_dim) return fail(CHITU_E_INVALID, "rotary: %d rotated channels of %d", rot, head_dim);
  if (int rc = check_table(table, table_rows, rot, "rotary")) return rc;
  if (tokens < 0 || tokens > 0x7fffffff) return fail(CHITU_E_INVALID, "rotary: bad token count");
  const int es = dtype == CHITU_DTYPE_FP32 ? 4 : 2;
  chitu::RotaryParams p;
  int64_t heads_total = 0;
  for (int i = 0; i < n; ++i) {
    if (!x[i] || !out[i] || !aligned16(x[i]) || !aligned16(out[i])) return fail(CHITU_E_INVALID, "rotary: tensor %d null or not 16-byte aligned", i);
    if (heads[i] < 1 || heads[i] > 65535) return fail(CHITU_E_INVALID, "rotary: tensor %d has no heads, or too many", i);
    if (!strides_fit(x_strides + 2 * i, tokens, heads[i], es) || !strides_fit(out_strides + 2 * i, tokens, heads[i], es))
      return fail(CHITU_E_INVALID, "rotary: strides of tensor %d must be positive multiples of 16 bytes", i);
    p.job[i] = {x[i], out[i], x_strides[2 * i], x_strides[2 * i + 1], out_strides[2 * i], out_strides[2 * i + 1], heads[i]};
    heads_total += heads[i];
  }
  if (tokens == 0) return CHITU_OK;
  p.positions = positions;
  p.wide_positions = positions_are_int64;
  p.table = reinterpret_cast<const float2*>(table);
  p.table_rows = table_rows;
  p.tokens = static_cast<int>(tokens);
  p.head_dim = head_dim;
  p.rot = rot;
  const int per_block = chitu::kRotaryThreads / (head_dim / 16);
  const int64_t blocks = (tokens + per_block - 1) / per_block;
  // heads of one thread: one where that fits the machine at once (three blocks per SM), else as many as then do
  const int64_t chunks = std::min<int64_t>(heads_total, std::max<int64_t>(1, kSms * 3 / blocks));
  p.heads_each = static_cast<int>((heads_total + chunks - 1) / chunks);
  int rows = 0;
  for (int i = 0; i < 3; ++i) {
    if (i < n) rows += (heads[i] + p.heads_each - 1) / p.heads_each;
    p.chunk_end[i] = rows;
  }
  if (rows > 65535) return fail(CHITU_E_UNSUPPORTED, "rotary: too many heads for one call");
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(rows));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define CHITU_ROTARY(DT) \
  (interleaved ? chitu::rotary_kernel<DT, true><<<grid, chitu::kRotaryThreads, 0, st>>>(p) \
               : chitu::rotary_kernel<DT, false><<<grid, chitu::kRotaryThreads, 0, st>>>(p))
  if (dtype == CHITU_DTYPE_BF16)
    CHITU_ROTARY(chitu::kBF16);
  else if (dtype == CHITU_DTYPE_FP16)
    CHITU_ROTARY(chitu::kFP16);
  else
    CHITU_ROTARY(chitu::kFP32);
#undef CHITU_ROTARY
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CHITU_OK : cuda_fail(e, "rotary: launch");
}

int chitu_b200_kv_append(const chitu_b200_kv_cache* cache, const void* k, const void* v, const void* q,
                         const int64_t* k_strides, const int64_t* v_strides, const int64_t* q_strides, void* q_out,
                         int q_heads, int64_t tokens, int dtype, int max_new, const void* positions, int positions_are_int64,
                         const float* table, int64_t table_rows, int rot, int interleaved, void* stream) {
  if (int rc = check_cache(cache, "kv_append")) return rc;
  if (!k || !v || !k_strides || !v_strides) return fail(CHITU_E_INVALID, "kv_append: null pointer");
  if (dtype != CHITU_DTYPE_BF16 && dtype != CHITU_DTYPE_FP16) return fail(CHITU_E_UNSUPPORTED, "kv_append: inputs must be bf16 or fp16");
  if (tokens < 0 || tokens > 0x7fffffff) return fail(CHITU_E_INVALID, "kv_append: bad token count");
  if (!aligned16(k) || !aligned16(v) || !strides_fit(k_strides, tokens, cache->heads, 2) || !strides_fit(v_strides, tokens, cache->heads, 2))
    return fail(CHITU_E_INVALID, "kv_append: k and v must be 16-byte aligned, strides positive multiples of 8 elements");
  if (q != nullptr) {
    if (!q_strides || !q_out || q_heads < 1) return fail(CHITU_E_INVALID, "kv_append: q needs strides, heads and q_out");
    if (!aligned16(q) || !aligned16(q_out) || !strides_fit(q_strides, tokens, q_heads, 2))
      return fail(CHITU_E_INVALID, "kv_append: q must be 16-byte aligned, strides positive multiples of 8 elements");
  }
  if (table != nullptr) {
    if (int rc = check_table(table, table_rows, rot, "kv_append")) return rc;
    if (rot > 128) return fail(CHITU_E_INVALID, "kv_append: %d rotated channels of 128", rot);
  }
  if (tokens == 0 || cache->batch == 0) return CHITU_OK;
  chitu::AppendParams p = {};
  const void* src[3] = {k, v, q};
  const int64_t* st3[3] = {k_strides, v_strides, q != nullptr ? q_strides : k_strides};
  for (int i = 0; i < 3; ++i) {
    p.src[i] = src[i];
    p.src_token[i] = st3[i][0];
    p.src_head[i] = st3[i][1];
  }
  const int es = cache->format == CHITU_CACHE_E4M3 ? 1 : 2;
  p.cache[0] = cache->k;
  p.cache[1] = cache->v;
  p.scale[0] = cache->k_scale;
  p.scale[1] = cache->v_scale;
  for (int i = 0; i < 2; ++i) {
    const int64_t* cs = i == 0 ? cache->k_strides : cache->v_strides;
    const int64_t* ss = i == 0 ? cache->k_scale_strides : cache->v_scale_strides;
    p.c_page[i] = cs[0] * es;
    p.c_token[i] = cs[1] * es;
    p.c_head[i] = cs[2] * es;
    p.s_page[i] = ss[0];
    p.s_head[i] = ss[1];
  }
  p.q_out = q_out;
  p.block_table = cache->block_table;
  p.table_stride = cache->table_stride;
  p.lens = cache->lens;
  p.cu = cache->cu_seqlens;
  p.positions = positions;
  p.wide_positions = positions_are_int64;
  p.rope = reinterpret_cast<const float2*>(table);
  p.rope_rows = table_rows;
  p.rot = table != nullptr ? rot : 0;
  p.interleaved = interleaved;
  p.batch = cache->batch;
  p.tokens = static_cast<int>(tokens);
  p.width = cache->table_width;
  p.n_pages = cache->n_pages;
  p.heads_kv = cache->heads;
  p.heads_q = q != nullptr ? q_heads : 0;
  p.page = cache->page_size;
  p.page_shift = page_shift_of(cache->page_size);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool fp16 = dtype == CHITU_DTYPE_FP16, eight = es == 1;
  const int expected = std::max<int>(1, static_cast<int>(std::min<int64_t>(max_new, tokens)));
  const int planes = 2 * p.heads_kv + p.heads_q;
  if (expected <= kAppendFew) {
    const dim3 grid(static_cast<unsigned>(p.batch), static_cast<unsigned>((planes + 31) / 32));
    if (grid.y > 65535) return fail(CHITU_E_UNSUPPORTED, "kv_append: too many heads for one call");
    if (fp16 && eight)
      chitu::kv_append_few_kernel<true, true><<<grid, 256, 0, st>>>(p);
    else if (fp16)
      chitu::kv_append_few_kernel<true, false><<<grid, 256, 0, st>>>(p);
    else if (eight)
      chitu::kv_append_few_kernel<false, true><<<grid, 256, 0, st>>>(p);
    else
      chitu::kv_append_few_kernel<false, false><<<grid, 256, 0, st>>>(p);
  } else {
    // rows of a run, threads, heads of a block at a time (see kv_append_kernel)
    const int q_rows = std::min(p.page, 64), kv_rows = eight ? p.page : q_rows;
    const int threads = std::max(256, 4 * kv_rows);
    const int kv_each = threads / (4 * kv_rows), q_each = threads / (4 * q_rows);
    p.slots = (expected + q_rows - 2) / q_rows + 1;
    const int64_t blocks = static_cast<int64_t>(p.batch) * p.slots;
    const int kv_groups = (p.heads_kv + kv_each - 1) / kv_each, q_groups = (p.heads_q + q_each - 1) / q_each;
    // groups of a block: as many as leave every SM six blocks
    p.turns = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(16, blocks * (2 * kv_groups + q_groups) / (kSms * 6))));
    p.kv_blocks = (kv_groups + p.turns - 1) / p.turns;
    const int64_t rows = 2 * p.kv_blocks + (q_groups + p.turns - 1) / p.turns;
    if (blocks > 0x7fffffff || rows > 65535) return fail(CHITU_E_UNSUPPORTED, "kv_append: too many pages or heads for one call");
    auto launch = [&](int n_threads, int64_t y) {
      const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(y));
      if (fp16) return eight ? launch_append<true, true>(p, n_threads, grid, st) : launch_append<true, false>(p, n_threads, grid, st);
      return eight ? launch_append<false, true>(p, n_threads, grid, st) : launch_append<false, false>(p, n_threads, grid, st);
    };
    cudaError_t e;
    if (threads > 512 && q != nullptr) {
      // Pages of 256 tokens want blocks without room for the factors, queries do not: 12 prompts 127 us in one launch, 108 in two
      // (pages of 128: 80 and 84).
      e = launch(threads, 2 * p.kv_blocks);
      const int each = 256 / (4 * q_rows);
      const int groups = (p.heads_q + each - 1) / each;
      p.turns = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(16, blocks * groups / (kSms * 6))));
      p.kv_blocks = 0;
      if (e == cudaSuccess) e = launch(256, (groups + p.turns - 1) / p.turns);
    } else {
      e = launch(threads, rows);
    }
    if (e != cudaSuccess) return cuda_fail(e, "kv_append: launch");
  }
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? CHITU_OK : cuda_fail(e, "kv_append: launch");
}

int64_t chitu_b200_attn_cache_workspace_bytes(int heads, int q_heads, int max_q) {
  if (heads < 1 || q_heads < heads) return 0;
  return takes_tile_kernel(max_q, q_heads / heads) ? tile_workspace_bytes() : rows_workspace_bytes();
}

int chitu_b200_attn_fwd_cache(const chitu_b200_kv_cache* cache, const void* q, const int64_t* q_strides, void* out, float* lse,
                              int q_heads, int64_t tokens, float softmax_scale, int causal, int dtype, int max_q, int max_kv,
                              void* workspace, int64_t workspace_bytes, int* status, void* stream) {
  if (int rc = check_cache(cache, "attn_fwd_cache")) return rc;
  if (!q || !q_strides || !out) return fail(CHITU_E_INVALID, "attn_fwd_cache: null pointer");
  if (dtype != CHITU_DTYPE_BF16 && dtype != CHITU_DTYPE_FP16) return fail(CHITU_E_UNSUPPORTED, "attn_fwd_cache: q must be bf16 or fp16");
  if (q_heads < 1 || q_heads % cache->heads != 0)
    return fail(CHITU_E_INVALID, "attn_fwd_cache: %d query heads over %d key heads", q_heads, cache->heads);
  if (tokens < 0 || tokens > 0x7fffffff / q_heads) return fail(CHITU_E_INVALID, "attn_fwd_cache: bad token count");
  if (!(softmax_scale > 0.f) || softmax_scale > 1e30f) return fail(CHITU_E_INVALID, "attn_fwd_cache: softmax_scale must be positive and finite");
  if (!aligned16(q) || !aligned16(out) || !strides_fit(q_strides, tokens, q_heads, 2))
    return fail(CHITU_E_INVALID, "attn_fwd_cache: q and out must be 16-byte aligned, strides positive multiples of 8 elements");
  if (tokens == 0 || cache->batch == 0) return CHITU_OK;
  max_q = std::max(max_q, 1);
  max_kv = std::max(max_kv, 1);
  const int64_t need = chitu_b200_attn_cache_workspace_bytes(cache->heads, q_heads, max_q);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(CHITU_E_INVALID, "attn_fwd_cache: workspace must be 16-byte aligned and hold %lld bytes", static_cast<long long>(need));
  chitu::CacheAttnParams p = {};
  const int es = cache->format == CHITU_CACHE_E4M3 ? 1 : 2;
  p.q = q;
  p.q_token = q_strides[0];
  p.q_head = q_strides[1];
  p.out = out;
  p.lse = lse;
  p.scale[0] = cache->k_scale;
  p.scale[1] = cache->v_scale;
  for (int i = 0; i < 2; ++i) {
    const int64_t* ss = i == 0 ? cache->k_scale_strides : cache->v_scale_strides;
    p.s_page[i] = ss[0];
    p.s_head[i] = ss[1];
  }
  p.block_table = cache->block_table;
  p.table_stride = cache->table_stride;
  p.lens = cache->lens;
  p.cu = cache->cu_seqlens;
  p.status = status;
  p.batch = cache->batch;
  p.tokens = static_cast<int>(tokens);
  p.width = cache->table_width;
  p.n_pages = cache->n_pages;
  p.heads_kv = cache->heads;
  p.group = q_heads / cache->heads;
  p.page_shift = page_shift_of(cache->page_size);
  p.causal = causal;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.tok_blk = p.group <= chitu::kTileRows ? chitu::kTileRows / p.group : 0;
  p.out_aligned32 = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
  p.count = static_cast<int*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kHeaderBytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool fp16 = dtype == CHITU_DTYPE_FP16, eight = es == 1;
  cudaError_t e;
  const bool tile = takes_tile_kernel(max_q, p.group);
  const int box = std::min(cache->page_size, tile ? 128 : eight ? chitu::RowsShape<true>::keys : chitu::RowsShape<false>::keys);
  CUtensorMap tk, tv;
  if (int rc = make_cache_map(&tk, cache, cache->k, cache->k_strides, box, !(tile && eight), "k_cache")) return rc;
  if (int rc = make_cache_map(&tv, cache, cache->v, cache->v_strides, box, !(tile && eight), "v_cache")) return rc;
  if (tile) {
    p.min_tiles = kTileMinTiles;
    e = fp16 ? (eight ? launch_tile<true, true>(tk, tv, p, st) : launch_tile<true, false>(tk, tv, p, st))
             : (eight ? launch_tile<false, true>(tk, tv, p, st) : launch_tile<false, false>(tk, tv, p, st));
    return e == cudaSuccess ? CHITU_OK : cuda_fail(e, "attn_fwd_cache: launch");
  }
  e = fp16 ? (eight ? launch_rows<true, true>(tk, tv, p, max_q, max_kv, st) : launch_rows<true, false>(tk, tv, p, max_q, max_kv, st))
           : (eight ? launch_rows<false, true>(tk, tv, p, max_q, max_kv, st) : launch_rows<false, false>(tk, tv, p, max_q, max_kv, st));
  return e == cudaSuccess ? CHITU_OK : cuda_fail(e, "attn_fwd_cache: launch");
}

}  // extern "C"
