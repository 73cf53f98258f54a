// Attention of packed queries over a paged key/value cache, head_dim 128: what is common to its kernels, and the kernel
// for few query rows per sequence and key head (single tokens, a few of them).
//
//   out_i = sum_j softmax_j(scale q_i . K_j) V_j,   j < lens[b], with `causal` j <= lens[b] - n_b + i
//
// Query row r of sequence b and key head h is token r / group, query head h * group + r % group: the heads that share keys
// are rows of one tile, so keys and values are read once for all of them.
//
// 8-bit pages hold e4m3 codes k8, v8 with scales ks, vs for each page and head.  Codes are exact in fp16, so they are
// widened to fp16 and never rounded; scales enter in fp32:
//   score  s = (scale ks) (q . k8);   p = 2^(s log2e + log2 vs - m);   o = sum p v8,   l = sum p / vs
// The value scale sits in the exponent, so the running maximum m is that of p itself and the 16-bit probabilities use their
// range whatever the scales are.  A bf16 query row is brought to fp16 by a power of two of its own (bf16 values of one row are
// 2^-24 of its largest before fp16 drops any of their bits), which goes into the score's factor.
#pragma once

#include <cfloat>

#include "attn_persist.cuh"
#include "kv_cache.cuh"

namespace chitu {

struct CacheAttnParams {
  const void* q;  // [tokens, heads_q, 128], element strides
  long long q_token, q_head;
  void* out;      // [tokens, heads_q, 128] contiguous
  float* lse;     // [heads_q, tokens] fp32 natural log, or nullptr
  const float* scale[2];                       // 8-bit pages: one fp32 per page and head
  long long s_page[2], s_head[2];              // strides, elements
  const int* block_table;
  long long table_stride;
  const int* lens;
  const int* cu;
  int* status;
  int batch, tokens, width, n_pages, heads_kv, group, page_shift, causal;
  float scale_log2;  // softmax_scale * log2(e)
  // work split over the grid (see each kernel) and scratch for pieces of a row's keys
  int min_tiles;
  int tok_blk;        // tokens of a 256-row block (tile kernel)
  int out_aligned32;
  int* count;
  float* part;
};

// Lengths of one sequence, brought into what the table and the packed queries can hold.
struct SeqInfo {
  int tok0, n_new, len, first;  // first packed token, tokens, keys, position of the first token
};
__device__ __forceinline__ SeqInfo seq_info(const CacheAttnParams& p, int b) {
  SeqInfo s;
  s.tok0 = min(max(__ldg(p.cu + b), 0), p.tokens);
  s.n_new = min(max(__ldg(p.cu + b + 1), s.tok0), p.tokens) - s.tok0;
  const int raw = max(__ldg(p.lens + b), -(1 << 30));
  s.len = static_cast<int>(min(static_cast<long long>(max(raw, 0)), static_cast<long long>(p.width) << p.page_shift));
  s.first = raw - s.n_new;
  return s;
}

// probabilities are kept at up to 2^(kProbShift + kRescaleThreshold) in fp16, whose range would otherwise end 2^-24 below
// the row's maximum
constexpr float kProbShift = 7.f;
// A value scale of zero has no logarithm: it counts as the smallest normal number.  l = sum p / vs has to stay finite, so the
// running maximum takes scales below 2^-82 for 2^-82: a weight p / vs is then at most 2^(15 + 82), and a sequence has at most
// 2^30 keys.  Probabilities keep the true scale, so where all scales of a row are below 2^-82 by 2^x, its largest ones come to
// 2^(7 - x) and end in fp16's last steps of 2^-24: weights of values of 2^-92 have all their 11 bits, of 2^-105 none.
constexpr float kMinValueScale = FLT_MIN;
constexpr float kLowValueLog2 = -82.f;

__device__ __forceinline__ void mma_16816_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool kHalf>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kHalf)
    mma_16816_f16(d, a, b0, b1);
  else
    mma_16816_bf16(d, a, b0, b1);
}
__device__ __forceinline__ uint32_t widen_e4m3x2(uint32_t two_codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two_codes)));
  return h;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// ----------------------------------------------------------------------------
// rows kernel: 16 query rows of one key head per unit, warp-level matrix instructions
// ----------------------------------------------------------------------------
//
// Memory bound: a key and a value byte are read once for at most 16 rows.  The grid's CTAs share all (sequence, 16 rows, key
// head, tile of keys) steps evenly, in that order: CTA c takes the c-th of gridDim.x equal runs, whatever the lengths are.  A
// run that ends inside an item (sequence, rows, head) leaves the item's fp32 piece in scratch, and the CTA that completes the
// item's count merges its pieces in order; nobody waits.
//
// 64 sequences of 3 to 16300 keys, one token each, 32 query heads over 8, 8-bit pages of 64: 198 us, 5.4 TB/s of keys and values, one pass
// behind the other, 215 us among other work (four times as long: 6.5 TB/s, the rate of a copy); two of 125000 in pages of 16: 99 and
// 106 us (a merge of 28 pieces in four turns rather than two costs 5 more); 16-bit pages of 32, 16 sequences of 500 to 8191: 108 us,
// 5.3 TB/s.  The first version, a block per 256 keys and loads through registers, took 329, 183 and 178.
//
// A warp takes 32 (16-bit pages: 16) of a tile's keys and keeps its own softmax.  The matrix instructions' sum over channels and the
// output's channels may be numbered as is convenient, so a lane's fragments are whole 16-byte pieces of cache rows: for q k^T, of
// key lane / 4, the pieces lane % 4 (and every fourth further); for p v, of four keys, the piece lane / 4.  Each warp has a ring of
// its own that one lane fills by tensor copies (a box is 16 or 32 tokens of a page; a page that does not exist reads zeros), over
// item borders, so the warps need no barrier inside a run.
constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
template <bool kEightBit>
struct RowsShape {
  static constexpr int ctas_per_sm = kEightBit ? 3 : 2;
  static constexpr int stages = kEightBit ? 2 : 3;
  static constexpr int keys = kEightBit ? 32 : 16;            // of a warp's step
  static constexpr int tile = keys * kRowsWarps;
  static constexpr int step_bytes = 8192;                     // keys, then values; also a warp's accumulators
  static constexpr int ring = kRowsWarps * stages * step_bytes;
  static constexpr int meta_at = ring;                        // per warp and stage: scales of both halves, whether they have a page
  static constexpr int q_at = meta_at + kRowsWarps * stages * 32;  // query fragments: 8 steps of 16 channels, 32 lanes
  static constexpr int stat_at = q_at + 8 * 32 * 16;
  static constexpr int bar_at = stat_at + kRowsWarps * 16 * 8;
  static constexpr int smem = bar_at + kRowsWarps * stages * 8 + 16 + 1024;
};
// scratch of one piece: [rows g, rows g + 8][16 accumulators][32 lanes] float2, then (maximum, sum) of 16 rows
constexpr int kRowsPieceFloats = 2 * 16 * 32 * 2 + 32;

// Position in the order of steps.
struct RowsCursor {
  int b, rb, h, tile;   // sequence, 16-row block, key head, tile of keys
  int n_rb, n_tiles;    // of the sequence
  SeqInfo seq;
  template <int kTile>
  __device__ __forceinline__ void measure(const CacheAttnParams& p) {
    seq = seq_info(p, b);
    n_rb = (seq.n_new * p.group + 15) >> 4;
    n_tiles = max((seq.len + kTile - 1) / kTile, 1);
  }
  template <int kTile>
  __device__ __forceinline__ void next_item(const CacheAttnParams& p) {
    tile = 0;
    if (++h < p.heads_kv) return;
    h = 0;
    if (++rb < n_rb) return;
    rb = 0;
    while (++b < p.batch) {
      measure<kTile>(p);
      if (n_rb > 0) return;
    }
  }
};
template <int kTile>
__device__ __forceinline__ long long rows_steps(const CacheAttnParams& p, int b, int& tiles) {
  const SeqInfo s = seq_info(p, b);
  const long long n_rb = (static_cast<long long>(s.n_new) * p.group + 15) >> 4;
  tiles = max((s.len + kTile - 1) / kTile, 1);
  return n_rb * p.heads_kv * tiles;
}

// Query rows g and g + 8 as matrix fragments: for 8-bit pages piece j (64 channels), step k (16 of them) is channels
// 64 j + 16 c + 4 k + {0, 1, 2, 3} of lane c; for 16-bit pages 32 j + 8 c + 4 k + ....
template <bool kFp16, bool kEightBit>
__device__ __forceinline__ void rows_load_q(const CacheAttnParams& p, const RowsCursor& cur, int g, int c, uint32_t (&qf)[8][4], float (&factor)[2]) {
  constexpr int kPieces = kEightBit ? 2 : 4, kSteps = kEightBit ? 4 : 2;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = cur.rb * 16 + g + 8 * i;
    const int tok = r / p.group, hq = cur.h * p.group + r - tok * p.group;
    const bool live = tok < cur.seq.n_new;
    uint4 w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = make_uint4(0, 0, 0, 0);
    if (live) {
      const uint16_t* row = static_cast<const uint16_t*>(p.q) + (cur.seq.tok0 + tok) * p.q_token + hq * p.q_head;
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
#pragma unroll
        for (int k = 0; k < kSteps / 2; ++k) w[j * (kSteps / 2) + k] = __ldg(reinterpret_cast<const uint4*>(row + j * (128 / kPieces) + c * (32 / kPieces) + 8 * k));
    }
    factor[i] = p.scale_log2;
    uint32_t v[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[4 * k] = w[k].x;
      v[4 * k + 1] = w[k].y;
      v[4 * k + 2] = w[k].z;
      v[4 * k + 3] = w[k].w;
    }
    if constexpr (kEightBit && !kFp16) {
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(v[k] << 16)), fabsf(__uint_as_float(v[k] & 0xffff0000u))));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // row / 2^(exponent of its largest): below 2, exact in fp16 down to 2^-24
      const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 1), 253);
      const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
      factor[i] *= __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = pack2<true>(__uint_as_float(v[k] << 16) * down, __uint_as_float(v[k] & 0xffff0000u) * down);
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      qf[s][i] = v[2 * s];
      qf[s][2 + i] = v[2 * s + 1];
    }
  }
}

template <bool kFp16, bool kEightBit>
__global__ void __launch_bounds__(kRowsThreads, RowsShape<kEightBit>::ctas_per_sm)
attn_cache_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CacheAttnParams p) {
  using Shape = RowsShape<kEightBit>;
  constexpr int kStages = Shape::stages, kKeys = Shape::keys, kTile = Shape::tile;
  constexpr int kHalves = kKeys / 16;
  constexpr bool kHalf = kEightBit || kFp16;  // fp16 products
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_base + warp * kStages * Shape::step_bytes;
  const uint32_t meta_ring = smem_base + Shape::meta_at + warp * kStages * 32;
  const uint32_t bars = smem_base + Shape::bar_at + warp * kStages * 8;
  float2* join_stat = reinterpret_cast<float2*>(smem + Shape::stat_at);
  volatile int* last_flag = reinterpret_cast<volatile int*>(smem + Shape::bar_at + kRowsWarps * kStages * 8);
  volatile int* abort_flag = last_flag + 1;
  if (lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    *abort_flag = 0;
    // a step's copies, and four lanes' of the scales
    for (int s = 0; s < kStages; ++s) mbar_init(bars + 8 * s, kEightBit ? 5 : 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __syncwarp();

  // all steps, and where this CTA's run begins (each warp finds out by itself)
  long long total = 0;
  int longest = 1;  // tiles of an item
  for (int b = lane; b < p.batch; b += 32) {
    int tiles;
    total += rows_steps<kTile>(p, b, tiles);
    longest = max(longest, tiles);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
  }
  // A run costs about a microsecond a step, a piece of an item that is merged a fifth of one: n tiles are best cut into runs of
  // sqrt(n / 5), where the grid does not ask for longer ones (32 tiles, 8 heads: runs of one 18.7 us, of two 12.8).
  const int per = static_cast<int>(max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(max(1.f, sqrtf(0.2f * longest)))));
  const long long lo = static_cast<long long>(blockIdx.x) * per;
  if (lo >= total) return;
  const int n_steps = static_cast<int>(min(static_cast<long long>(per), total - lo));
  RowsCursor cur;
  long long at = 0;  // steps before sequence cur.b
  for (cur.b = 0;; cur.b += 32) {
    const int b = cur.b + lane;
    int tiles;
    const long long mine = b < p.batch ? rows_steps<kTile>(p, b, tiles) : 0;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, at + upto > lo);
    if (past != 0) {
      const int i = __ffs(past) - 1;
      at += __shfl_sync(0xffffffffu, upto - mine, i);
      cur.b += i;
      break;
    }
    at += __shfl_sync(0xffffffffu, upto, 31);
  }
  cur.measure<kTile>(p);
  {
    const long long item = (lo - at) / cur.n_tiles;
    cur.rb = static_cast<int>(item / p.heads_kv);
    cur.h = static_cast<int>(item - static_cast<long long>(cur.rb) * p.heads_kv);
    cur.tile = static_cast<int>(lo - at - item * cur.n_tiles);
  }
  RowsCursor ahead = cur;  // what is copied next
  int copied = 0;
  // Table entries of the keys that are copied next, loaded a step before they are looked at: entry(0) and, where pages are
  // smaller than a step, entry(1).
  const int* table = p.block_table + ahead.b * p.table_stride;
  auto entry = [&](int half) {
    const int key = ahead.tile * kTile + warp * kKeys + half * 16;
    int id = -1;
    if (key < ahead.seq.len) id = __ldg(table + (key >> p.page_shift));
    return id;
  };
  const bool small_pages = kHalves == 2 && p.page_shift == 4;
  int entry0 = entry(0), entry1 = small_pages ? entry(1) : 0;
  auto copy_step = [&](int stage) {
    const uint32_t bar = bars + 8 * stage;
    const uint32_t meta = meta_ring + stage * 32;
    const int page0 = static_cast<unsigned>(entry0) < static_cast<unsigned>(p.n_pages) ? entry0 : -1;
    const int page1 = small_pages ? (static_cast<unsigned>(entry1) < static_cast<unsigned>(p.n_pages) ? entry1 : -1) : page0;
    if (lane == 0) {
      asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(meta + 16), "r"(page0 >= 0 ? 1 : 0), "r"(page1 >= 0 ? 1 : 0) : "memory");
      mbar_arrive_expect_tx(bar, Shape::step_bytes);
      const uint32_t dst = ring + stage * Shape::step_bytes;
      const int token = (ahead.tile * kTile + warp * kKeys) & ((1 << p.page_shift) - 1);
      if constexpr (kEightBit) {
        tma_load_4d(dst, &tm_k, bar, 0, ahead.h, token, page0);
        tma_load_4d(dst + 4096, &tm_v, bar, 0, ahead.h, token, page0);
        if (small_pages) {
          tma_load_4d(dst + 2048, &tm_k, bar, 0, ahead.h, token, page1);
          tma_load_4d(dst + 6144, &tm_v, bar, 0, ahead.h, token, page1);
        }
      } else {
        tma_load_4d(dst, &tm_k, bar, 0, ahead.h, token, page0);
        tma_load_4d(dst + 2048, &tm_k, bar, 64, ahead.h, token, page0);
        tma_load_4d(dst + 4096, &tm_v, bar, 0, ahead.h, token, page0);
        tma_load_4d(dst + 6144, &tm_v, bar, 64, ahead.h, token, page0);
      }
    }
    if (kEightBit && lane < 4) {
      const int page = lane < 2 ? page0 : page1, kv = lane & 1;
      if (page >= 0) cp_async4(meta + 4 * lane, p.scale[kv] + page * p.s_page[kv] + ahead.h * p.s_head[kv]);
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    }
    if (++ahead.tile == ahead.n_tiles) {
      ahead.next_item<kTile>(p);
      table = p.block_table + ahead.b * p.table_stride;
    }
    if (++copied < n_steps) {
      entry0 = entry(0);
      if (small_pages) entry1 = entry(1);
    }
  };
#pragma unroll 1
  for (int s = 0; s < kStages; ++s)
    if (copied < n_steps) copy_step(s);

  // A row's probabilities are 2^(score + shift), shift = kProbShift - m; the largest score so far may pass m by kRescaleThreshold
  // before the shift moves.  A row that has seen no key has no limit to pass.
  constexpr float kTop = kProbShift + kRescaleThreshold;
  const uint32_t q_frag = smem_base + Shape::q_at + lane * 16;
  float factor[2], o[16][4], shift[2], l[2], ceiling[2];
  int limit[2], unmasked = 0;  // keys that a row, that all rows see
  int stage = 0, phase = 0;
  bool fresh = true;
#pragma unroll 1
  for (int step = 0; step < n_steps; ++step) {
    if (fresh) {
      {
        uint32_t qf[8][4];
        rows_load_q<kFp16, kEightBit>(p, cur, g, c, qf, factor);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k >> 1 == warp) asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(q_frag + k * 512), "r"(qf[k][0]), "r"(qf[k][1]), "r"(qf[k][2]), "r"(qf[k][3]) : "memory");
        __syncthreads();  // (each warp has written a quarter of the fragments that all of them read)
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = cur.rb * 16 + g + 8 * i;
        limit[i] = p.causal ? min(cur.seq.first + r / p.group + 1, cur.seq.len) : cur.seq.len;
        shift[i] = 0.f;
        ceiling[i] = -INFINITY;
        l[i] = 0.f;
      }
      unmasked = p.causal ? min(cur.seq.first + cur.rb * 16 / p.group + 1, cur.seq.len) : cur.seq.len;
#pragma unroll
      for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][e] = 0.f;
      fresh = false;
    }
    const int key0 = cur.tile * kTile + warp * kKeys;
    mbar_wait(bars + 8 * stage, phase, abort_flag, p.status, kDevTimeoutSoftmax);
    __syncwarp();
    const uint32_t src = ring + stage * Shape::step_bytes;
    const uint4 scales = ld_shared16(meta_ring + stage * 32);
    const uint4 there = ld_shared16(meta_ring + stage * 32 + 16);
    const bool border = key0 + kKeys > unmasked || there.x == 0 || there.y == 0;  // (the same for the whole warp)
    if (border) {
      // what a page holds behind the sequence's end may be anything: no weight is not enough
      const int left = cur.seq.len - key0;
      if constexpr (kEightBit) {
        if (lane >= left) {
#pragma unroll
          for (int i = 0; i < 8; ++i) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(src + 4096 + lane * 128 + i * 16), "r"(0) : "memory");
        }
      } else {
        if ((lane & 15) >= left) {
#pragma unroll
          for (int i = 0; i < 8; ++i) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(src + 4096 + lane * 128 + i * 16), "r"(0) : "memory");
        }
      }
      fence_proxy_async_smem();  // (before the next copy into this stage)
      __syncwarp();
    }
    // rows of 128 bytes, their 16-byte pieces exchanged by row & 7
    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    const uint32_t k_row = src + g * 128;
#pragma unroll
    for (int j = 0; j < (kEightBit ? 2 : 4); ++j) {
      const uint32_t at = k_row + (kEightBit ? 0 : (j >> 1) * 2048) + ((((j & 1) * 4 + c) ^ g) << 4);
      uint4 w[kKeys / 8];
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) w[n] = ld_shared16(at + n * 1024);
#pragma unroll
      for (int k = 0; k < (kEightBit ? 4 : 2); ++k) {
        const uint4 qv = ld_shared16(q_frag + (j * (kEightBit ? 4 : 2) + k) * 512);
        const uint32_t qf[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
        for (int n = 0; n < kKeys / 8; ++n) {
          if constexpr (kEightBit) {
            const uint32_t codes = k == 0 ? w[n].x : k == 1 ? w[n].y : k == 2 ? w[n].z : w[n].w;
            mma_16816_f16(s[n], qf, widen_e4m3x2(codes), widen_e4m3x2(codes >> 16));
          } else {
            mma_16816<kHalf>(s[n], qf, k == 0 ? w[n].x : w[n].z, k == 0 ? w[n].y : w[n].w);
          }
        }
      }
    }
    // scores of rows g (e = 0, 1) and g + 8 (e = 2, 3), keys key0 + 8 n + 2 c + (e & 1), in units of log2 and shifted
    float v_inv[kHalves];
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int half = 0; half < kHalves; ++half) {
      float k_scale = 1.f, v_log2 = 0.f, lift = 0.f;
      v_inv[half] = 1.f;
      if constexpr (kEightBit) {
        k_scale = __uint_as_float(half ? scales.z : scales.x);
        const float vs = fmaxf(__uint_as_float(half ? scales.w : scales.y), kMinValueScale);
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(v_log2) : "f"(vs));
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(v_inv[half]) : "f"(vs));
        if (border && (half ? there.y : there.x) == 0) {  // (no scales either)
          k_scale = v_inv[half] = 1.f;
          v_log2 = 0.f;
        }
        lift = fmaxf(kLowValueLog2 - v_log2, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = factor[i] * k_scale, add = v_log2 + shift[i];
#pragma unroll
        for (int n = 2 * half; n < 2 * half + 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[n][2 * i + e] = fmaf(s[n][2 * i + e], f, add);
        if (border) {
          asm volatile("" ::: "memory");  // (a branch that is rarely taken, not selections that always are)
#pragma unroll
          for (int n = 2 * half; n < 2 * half + 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if ((half ? there.y : there.x) == 0 || key0 + 8 * n + 2 * c + e >= limit[i]) s[n][2 * i + e] = -INFINITY;
        }
        top[i] = fmaxf(top[i], fmaxf(max3(s[2 * half][2 * i], s[2 * half][2 * i + 1], s[2 * half + 1][2 * i]), s[2 * half + 1][2 * i + 1]) + lift);
      }
    }
    if (__any_sync(0xffffffffu, top[0] > ceiling[0] || top[1] > ceiling[1])) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float t = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
        if (t > ceiling[i]) {
          const float down = kProbShift - t;  // the new shift, from the old one
          const float f = ceiling[i] == -INFINITY ? 0.f : fast_exp2(down);
          shift[i] += down;
          ceiling[i] = kTop;
          l[i] *= f;
#pragma unroll
          for (int tt = 0; tt < 16; ++tt) {
            o[tt][2 * i] *= f;
            o[tt][2 * i + 1] *= f;
          }
#pragma unroll
          for (int n = 0; n < kKeys / 8; ++n) {
            s[n][2 * i] += down;
            s[n][2 * i + 1] += down;
          }
        }
      }
    }
    uint32_t pf[kHalves][4];
#pragma unroll
    for (int half = 0; half < kHalves; ++half)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float a = fast_exp2(s[2 * half + n][2 * i]), b = fast_exp2(s[2 * half + n][2 * i + 1]);
          sum = n == 0 ? a + b : sum + (a + b);
          pf[half][n * 2 + i] = pack2<kHalf>(a, b);
        }
        l[i] = fmaf(sum, v_inv[half], l[i]);
      }
    // o += p v: lane's channels 16 g + t, t = 0 .. 15, of keys 16 half + 2 c, + 1, + 8, + 9
#pragma unroll
    for (int half = 0; half < kHalves; ++half)
#pragma unroll
      for (int j = 0; j < (kEightBit ? 1 : 2); ++j) {
        uint4 w[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int key = 2 * c + (n & 1);  // (+ 8 does not change key & 7)
          const uint32_t row = src + 4096 + (kEightBit ? 0 : (g >> 2) * 2048) + key * 128 + half * 2048 + (n >> 1) * 1024;
          w[n] = ld_shared16(row + (((kEightBit ? g : (g & 3) * 2 + j) ^ (key & 7)) << 4));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t r0 = q == 0 ? w[0].x : q == 1 ? w[0].y : q == 2 ? w[0].z : w[0].w;
          const uint32_t r1 = q == 0 ? w[1].x : q == 1 ? w[1].y : q == 2 ? w[1].z : w[1].w;
          const uint32_t r2 = q == 0 ? w[2].x : q == 1 ? w[2].y : q == 2 ? w[2].z : w[2].w;
          const uint32_t r3 = q == 0 ? w[3].x : q == 1 ? w[3].y : q == 2 ? w[3].z : w[3].w;
          if constexpr (kEightBit) {
            const uint32_t lo01 = __byte_perm(r0, r1, 0x5140), hi01 = __byte_perm(r0, r1, 0x7362);
            const uint32_t lo23 = __byte_perm(r2, r3, 0x5140), hi23 = __byte_perm(r2, r3, 0x7362);
            mma_16816_f16(o[4 * q], pf[half], widen_e4m3x2(lo01), widen_e4m3x2(lo23));
            mma_16816_f16(o[4 * q + 1], pf[half], widen_e4m3x2(lo01 >> 16), widen_e4m3x2(lo23 >> 16));
            mma_16816_f16(o[4 * q + 2], pf[half], widen_e4m3x2(hi01), widen_e4m3x2(hi23));
            mma_16816_f16(o[4 * q + 3], pf[half], widen_e4m3x2(hi01 >> 16), widen_e4m3x2(hi23 >> 16));
          } else {
            mma_16816<kHalf>(o[8 * j + 2 * q], pf[half], __byte_perm(r0, r1, 0x5410), __byte_perm(r2, r3, 0x5410));
            mma_16816<kHalf>(o[8 * j + 2 * q + 1], pf[half], __byte_perm(r0, r1, 0x7632), __byte_perm(r2, r3, 0x7632));
          }
        }
      }
    __syncwarp();  // every lane has read the stage
    const bool leaves = cur.tile + 1 == cur.n_tiles || step + 1 == n_steps;
    if (leaves) {
      // The run leaves this item.  The warps' accumulators meet in the stages that the step has just read; warp w sums
      // accumulators 4 w .. 4 w + 3 of all of them and takes these to the end.
      const int n_halves = min(cur.seq.n_new * p.group - cur.rb * 16, 16) > 8 ? 2 : 1;  // rows g + 8 in use?
      const uint32_t mine = src + lane * 8;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= n_halves) break;
#pragma unroll
        for (int t = 0; t < 16; ++t) asm volatile("st.shared.v2.f32 [%0], {%1,%2};" ::"r"(mine + (i * 16 + t) * 256), "f"(o[t][2 * i]), "f"(o[t][2 * i + 1]) : "memory");
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (c == 0) join_stat[warp * 16 + g + 8 * i] = make_float2(ceiling[i] == -INFINITY ? -INFINITY : kProbShift - shift[i], l[i]);
      }
      __syncthreads();
      float2 r[2][4];
      float m_row[2] = {-INFINITY, -INFINITY}, l_row[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i >= n_halves) break;
        float f[kRowsWarps];
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) m_row[i] = fmaxf(m_row[i], join_stat[w * 16 + g + 8 * i].x);
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
          const float2 st = join_stat[w * 16 + g + 8 * i];
          f[w] = st.x == -INFINITY ? 0.f : fast_exp2(st.x - m_row[i]);
          l_row[i] = fmaf(st.y, f[w], l_row[i]);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          r[i][t] = make_float2(0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kRowsWarps; ++w) {
            float x, y;
            asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(x), "=f"(y) : "r"(smem_base + (w * kStages + stage) * Shape::step_bytes + (i * 16 + 4 * warp + t) * 256 + lane * 8) : "memory");
            r[i][t].x = fmaf(x, f[w], r[i][t].x);
            r[i][t].y = fmaf(y, f[w], r[i][t].y);
          }
        }
      }
      fence_proxy_async_smem();  // (before the next copies into these stages)
      // CTAs that have a share of this item, which began at step `begun` of this one's run (or before it)
      const int begun = step - cur.tile, last_step = begun + cur.n_tiles - 1;
      const int cta = blockIdx.x;
      const int c_first = begun >= 0 ? cta : cta - (per - 1 - begun) / per, c_last = cta + last_step / per;
      bool write = true;
      if (c_first == c_last) {
        __syncthreads();
      } else {
        auto piece = [&](int c) {  // an item starts a CTA's run, or is the last of it
          return p.part + static_cast<long long>(2 * c + (c == c_first && begun - (c - cta) * per > 0 ? 1 : 0)) * kRowsPieceFloats;
        };
        float* out_piece = piece(cta);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i >= n_halves) break;
#pragma unroll
          for (int t = 0; t < 4; ++t) reinterpret_cast<float2*>(out_piece)[(i * 16 + 4 * warp + t) * 32 + lane] = r[i][t];
          if (warp == 0 && c == 0) reinterpret_cast<float2*>(out_piece + 2048)[g + 8 * i] = make_float2(m_row[i], l_row[i]);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
          // (the barrier has ordered the CTA's stores before this release, and orders its loads behind the acquire)
          int before;
          asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.count + c_first) : "memory");
          const int last = before == c_last - c_first;
          if (last) p.count[c_first] = 0;
          *last_flag = last;
        }
        __syncthreads();
        write = *last_flag != 0;
        if (write) {
          // Pieces in their order through the warp's stage (in registers they cost the main loop its own: spills, half the speed),
          // or all of its stages where the run is over: this warp's accumulators of a piece, then its 16 rows' statistics.
          const int n_pieces = c_last - c_first + 1;
          const int region = n_halves * 1024 + 128;
          const uint32_t room = step + 1 == n_steps ? ring : src;
          const int at_once = (step + 1 == n_steps ? kStages : 1) * Shape::step_bytes / region;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            m_row[i] = -INFINITY;
            l_row[i] = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t) r[i][t] = make_float2(0.f, 0.f);
          }
#pragma unroll 1
          for (int k0 = 0; k0 < n_pieces; k0 += at_once) {
            const int n = min(at_once, n_pieces - k0);
#pragma unroll 1
            for (int k = 0; k < n; ++k) {
              const float* from = piece(c_first + k0 + k);
              const uint32_t to = room + k * region;
#pragma unroll 1
              for (int part = lane; part < n_halves * 64; part += 32)  // 16 bytes: two lanes' pairs of one accumulator
                cp_async16(to + part * 16, from + (part >> 6) * 1024 + warp * 256 + (part & 63) * 4);
              if (lane < 8) cp_async16(to + region - 128 + lane * 16, from + 2048 + lane * 4);
            }
            cp_async_commit();
            cp_async_wait<0>();
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (i >= n_halves) break;
#pragma unroll 1
              for (int k = 0; k < n; ++k) {
                const uint32_t at = room + k * region;
                float2 st;
                asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(st.x), "=f"(st.y) : "r"(at + region - 128 + (g + 8 * i) * 8) : "memory");
                const float top = fmaxf(m_row[i], st.x);
                const float mine = m_row[i] == -INFINITY ? 0.f : fast_exp2(m_row[i] - top), theirs = st.x == -INFINITY ? 0.f : fast_exp2(st.x - top);
                m_row[i] = top;
                l_row[i] = fmaf(st.y, theirs, l_row[i] * mine);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                  float x, y;
                  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(x), "=f"(y) : "r"(at + (i * 4 + t) * 256 + lane * 8) : "memory");
                  r[i][t] = make_float2(fmaf(x, theirs, r[i][t].x * mine), fmaf(y, theirs, r[i][t].y * mine));
                }
              }
            }
            __syncwarp();
          }
          fence_proxy_async_smem();  // (before the next copy into the stage)
          __syncwarp();
        }
      }
      if (write) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row_i = cur.rb * 16 + g + 8 * i;
          const int tok = row_i / p.group, hq = cur.h * p.group + row_i - tok * p.group;
          if (i < n_halves && tok < cur.seq.n_new) {
            const float inv = l_row[i] == 0.f ? 0.f : 1.f / l_row[i];
            const size_t row = static_cast<size_t>(cur.seq.tok0 + tok);
            uint16_t* dst = static_cast<uint16_t*>(p.out) + (row * (static_cast<size_t>(p.heads_kv) * p.group) + hq) * 128 + 4 * warp;
            // (accumulator t, column 2 c + e: channel 16 (2 c + e) + t)
            *reinterpret_cast<uint2*>(dst + 32 * c) = make_uint2(pack2<kFp16>(r[i][0].x * inv, r[i][1].x * inv), pack2<kFp16>(r[i][2].x * inv, r[i][3].x * inv));
            *reinterpret_cast<uint2*>(dst + 32 * c + 16) = make_uint2(pack2<kFp16>(r[i][0].y * inv, r[i][1].y * inv), pack2<kFp16>(r[i][2].y * inv, r[i][3].y * inv));
            if (p.lse != nullptr && warp == 0 && c == 0)
              p.lse[static_cast<size_t>(hq) * p.tokens + row] = l_row[i] == 0.f ? -INFINITY : (m_row[i] - kProbShift + log2f(l_row[i])) * 0.6931471805599453f;
          }
        }
      }
      if (step + 1 < n_steps) {
        cur.next_item<kTile>(p);
        fresh = true;
      }
    } else {
      ++cur.tile;
    }
    if (copied < n_steps) copy_step(stage);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  if (*abort_flag && lane == 0) {
    // A wait has run out: nothing of ours may still be landing when the CTA retires (bounded polls on the last copies).
    for (int i = max(0, n_steps - kStages); i < n_steps; ++i)
      for (int spin = 0; spin < (1 << 20) && !mbar_try_wait(bars + 8 * (i % kStages), (i / kStages) & 1); ++spin) {
      }
  }
}

}  // namespace chitu
