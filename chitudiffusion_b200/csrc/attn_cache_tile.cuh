// Attention over a paged key/value cache for chunks of queries: 256-row query blocks on the tensor core (tcgen05, accumulators
// in tensor memory).
//
// Query block: two tiles of 128 rows, row r = token r / group, query head r % group of the key head, so that heads which share
// keys share a block.  Tensor bound; the layout is that of attn_persist_kernel - S | P0 | P1 | O0 | O1, one set of score
// columns that leaves for registers at once, three issuing warps - with what a paged 8-bit cache adds:
//
//   warps 0-3 / 4-7  softmax of tile 0 / 1 (a thread is a row); they also bring the block's query rows to shared memory
//   warps 8-11       widen e4m3 codes to fp16 in the swizzled layout of the matrix operands (16-bit pages: only clear the rows of
//                    values behind the sequence's end)
//   warps 12-14      issue QK^T, PV of tile 0, PV of tile 1
//   warp  15         walks the CTA's share of the work and publishes it block by block (TileSeg); tensor copies of pages (a box is a
//                    page, or 128 rows of one; page numbers are the outermost coordinate, and one outside the pool reads
//                    zeros) and the scales of a tile's sixteen-key groups
//
// Measured: 4680 queries over 32760 keys, 12 heads, 8-bit pages of 128: 773 us, 1218 TFLOP/s on a cool card, 898 us and 1049 under the
// power cap (attn_persist_kernel on the same keys in 16 bits: 706, 831); four causal chunks of 389 to 512 tokens over up to 8100
// keys, 32 query heads over 8, pages of 64: 150 us, 969 TFLOP/s, among other work 162 us, 897.  16-bit pages, cool card: 904 us and,
// for chunks of like sizes, 140 us where 8-bit ones take 140 as well.  A block of one tile's rows has one chain of scores,
// exponentials and products, and the SM waits for it: split over both halves of the CTA (every second key tile each) 64 such blocks of
// 16000 keys took 746 us instead of 823, but the code that it needs cost the cases above 0.5 %, and a form of its own with more
// copies in flight (673) cost shorter ones 3 to 7 %.
//
// Widening costs the SM sub-partitions' issue slots (about 100 instructions per warp and tile) rather than a pass over
// memory: read back from a 16-bit copy of the cache, three frames over 21 would move 200 MB more.
//
// Work.  A block's share of the work is the keys it sees, K = the last row's, and kBlockKeys for what a block costs besides (its
// queries, the first scores, its result).  All blocks in the order (sequence, key head, block) are a line of such keys; CTA c
// takes the c-th of gridDim.x equal runs of it, and of a block those 128-key tiles whose first key (behind the block's
// kBlockKeys) lies in its run.  So ragged lengths, causal blocks and few long blocks alike finish together.
// (Dealing out whole blocks first, so that CTAs walk the same keys at the same time, gained nothing: 790 us against 770 for
// three frames over 21.)  A block that a run's border cuts leaves fp32 pieces in scratch; attn_cache_join_kernel, launched
// behind, merges them with all SMs (the CTA that comes last would have up to 148 pieces of 128 KB to itself).
#pragma once

#include "attn_cache.cuh"

namespace chitu {

constexpr int kTileThreads = 512;
constexpr int kTileRows = 2 * kTileM;    // rows of a block
constexpr int kCoefStages = 8;           // tiles whose scales are kept: the copies run at most five ahead of the softmax
constexpr int kSegStages = 8;            // blocks whose description is kept (each has a tile at least)
template <bool kEightBit>
struct TileShape {
  static constexpr int slots = kEightBit ? 4 : 5;       // 16-bit operand tiles, keys and values in turn
  static constexpr int raw_slots = kEightBit ? 2 : 5;   // as copied (16-bit pages are copied into their operand slot)
  static constexpr int raw_bytes = kEightBit ? kTileBytes / 2 : 0;
  static constexpr int coef_at = 2 * kTileBytes + slots * kTileBytes + raw_slots * raw_bytes;
  static constexpr int bar_at = coef_at + kCoefStages * 8 * 16;
  static constexpr int seg_at = bar_at + 496;
  static constexpr int smem = seg_at + kSegStages * 48 + 1024;
};
// What the join kernel needs to know of a block whose first tile is in a CTA's run and whose last one is not.
struct TileJoin {
  int n_pieces;          // 0: there is no such block
  int first;             // where the first piece is; the others are 2 (CTA + 1), 2 (CTA + 2), ...
  int row, n_rows;       // first packed token, query rows
  int h, pad[3];
};
// scratch of one piece: per tile [32 column groups][128 rows] float4, then (maximum, sum) of 128 rows
constexpr int kTilePieceFloats = 2 * (32 * kTileM * 4 + 2 * kTileM);

struct TileBlock {
  int b, h, blk;       // sequence, key head, block
  int n_blk;           // blocks of the sequence
  int keys, n_tiles;   // K of the block, kBlockKeys included; its tiles
  long long start;     // first key on the line
  SeqInfo seq;
};
// (four causal chunks, one to nine blocks a CTA: CTAs end between 125 and 185 us without it)
constexpr int kBlockKeys = 512;

// What the warps of a CTA need to know of a block that they work on.
struct TileSeg {
  int n;                        // its key tiles t0 ... t0 + n - 1; 0: there is no more work
  int t0;
  int tok0, n_new, len, first;  // of the sequence
  int h, blk, rows;             // key head, block, query rows
  int piece;                    // where its fp32 piece goes, -1: the result itself
  int pad[2];
};
static_assert(sizeof(TileSeg) == 48, "control block");
struct TileLine {
  long long total, per;  // keys, keys of a run
};

// Blocks of a sequence hold whole tokens: tok_blk = 256 / group each.  The blocks' K are first + tok_blk, first + 2 tok_blk, ...,
// all of the sequence's keys for the last one; where nothing is masked by position, or lengths do not fit (more queries than keys,
// more keys than the table holds), it is all keys for every block.
__device__ __forceinline__ bool tile_steps_grow(const CacheAttnParams& p, const SeqInfo& s) { return p.causal && s.first >= 0 && s.len == s.first + s.n_new; }
__device__ __forceinline__ int tile_blocks(const CacheAttnParams& p, const SeqInfo& s) { return (s.n_new + p.tok_blk - 1) / p.tok_blk; }
__device__ __forceinline__ int tile_keys(const CacheAttnParams& p, const SeqInfo& s, int blk) {
  return (tile_steps_grow(p, s) ? min(s.first + p.tok_blk * (blk + 1), s.len) : s.len) + kBlockKeys;
}
// keys of blocks [0, blk) of one head
__device__ __forceinline__ long long tile_keys_before(const CacheAttnParams& p, const SeqInfo& s, int blk, int n_blk) {
  if (!tile_steps_grow(p, s)) return static_cast<long long>(blk) * (s.len + kBlockKeys);
  if (n_blk == 0) return 0;
  const long long n = min(blk, n_blk - 1);  // (the last block ends with the sequence)
  const long long sum = n * (s.first + kBlockKeys) + p.tok_blk * (n * (n + 1) / 2);
  return blk == n_blk ? sum + s.len + kBlockKeys : sum;
}
__device__ __forceinline__ long long tile_keys_of(const CacheAttnParams& p, int b) {
  const SeqInfo s = seq_info(p, b);
  const int n_blk = tile_blocks(p, s);
  return tile_keys_before(p, s, n_blk, n_blk) * p.heads_kv;
}

__device__ __forceinline__ void tile_measure(const CacheAttnParams& p, TileBlock& w) {
  w.keys = tile_keys(p, w.seq, w.blk);
  w.n_tiles = max((w.keys - kBlockKeys + kTileN - 1) / kTileN, 1);
}
__device__ __forceinline__ void tile_next_block(const CacheAttnParams& p, TileBlock& w) {
  w.start += w.keys;
  if (++w.blk == w.n_blk) {
    w.blk = 0;
    if (++w.h == p.heads_kv) {
      w.h = 0;
      while (++w.b < p.batch) {
        w.seq = seq_info(p, w.b);
        w.n_blk = tile_blocks(p, w.seq);
        if (w.n_blk > 0) break;
      }
      if (w.b >= p.batch) return;
    }
  }
  tile_measure(p, w);
}

// The line, by a whole warp.
__device__ __forceinline__ TileLine tile_line(const CacheAttnParams& p, int lane, int ctas) {
  TileLine line;
  line.total = 0;
  for (int b = lane; b < p.batch; b += 32) line.total += tile_keys_of(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) line.total += __shfl_xor_sync(0xffffffffu, line.total, o);
  line.per = max((line.total + ctas - 1) / ctas, static_cast<long long>(p.min_tiles) * kTileN);
  return line;
}
// The block that key `pos` of the line (< total) belongs to, by a whole warp.
__device__ __forceinline__ TileBlock tile_locate(const CacheAttnParams& p, int lane, long long pos) {
  TileBlock w;
  long long at = 0;
  for (w.b = 0;; w.b += 32) {
    const int b = w.b + lane;
    const long long mine = b < p.batch ? tile_keys_of(p, b) : 0;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, at + upto > pos);
    if (past != 0) {
      const int i = __ffs(past) - 1;
      at += __shfl_sync(0xffffffffu, upto - mine, i);
      w.b += i;
      break;
    }
    at += __shfl_sync(0xffffffffu, upto, 31);
  }
  w.seq = seq_info(p, w.b);
  w.n_blk = tile_blocks(p, w.seq);
  const long long per_head = tile_keys_before(p, w.seq, w.n_blk, w.n_blk);
  w.h = static_cast<int>((pos - at) / per_head);
  const long long in_head = pos - at - w.h * per_head;
  int lo = 0, hi = w.n_blk - 1;  // the last block that starts at or before in_head
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tile_keys_before(p, w.seq, mid, w.n_blk) <= in_head)
      lo = mid;
    else
      hi = mid - 1;
  }
  w.blk = lo;
  w.start = at + w.h * per_head + tile_keys_before(p, w.seq, lo, w.n_blk);
  tile_measure(p, w);
  return w;
}

// The blocks of a CTA's run one after the other, each with its tiles [t0, t0 + n).
struct TileWalk {
  TileBlock w;
  long long lo, end;  // the run
  bool begun;
  __device__ __forceinline__ void begin(const CacheAttnParams& p, int lane, int cta, int ctas) {
    const TileLine line = tile_line(p, lane, ctas);
    lo = cta * line.per;
    end = min(lo + line.per, line.total);
    if (lo < end) w = tile_locate(p, lane, lo);
    begun = false;
  }
  __device__ __forceinline__ bool next(const CacheAttnParams& p, int& t0, int& n) {
    if (lo >= end) return false;
    long long pos = lo;
    while (true) {
      if (begun) {
        pos = w.start + w.keys;
        if (pos >= end) return false;
        tile_next_block(p, w);
      }
      begun = true;
      // (tile i's place on the line: kBlockKeys + 128 i)
      auto first_at = [](long long at) { return static_cast<int>((max(at - kBlockKeys, 0ll) + kTileN - 1) / kTileN); };
      t0 = first_at(pos - w.start);
      n = (end - w.start >= w.keys ? w.n_tiles : end - w.start <= kBlockKeys ? 0 : first_at(end - w.start)) - t0;
      if (n > 0) return true;
    }
  }
};

__device__ __forceinline__ void st_global32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// mbar_wait with its loop in a few instructions: the roles' hot loops share the instruction cache.  As there, a wait ends when
// the barrier's phase is complete, when another role has given up, or after about a second (2^24 polls of at least 100 cycles).
__device__ __forceinline__ bool tile_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n, a;\n\tmov.u32 n, 0;\n"
      "POLL:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE;\n\t"
      "ld.volatile.shared.u32 a, [%3];\n\tsetp.ne.u32 q, a, 0;\n\t@q bra DONE;\n\t"
      "add.u32 n, n, 1;\n\tsetp.lt.u32 q, n, 16777216;\n\t@q bra POLL;\n"
      "DONE:\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(smem_u32(const_cast<const int*>(abort_flag)))
      : "memory");
  if (ok == 0 && *abort_flag == 0) {
    *abort_flag = 1;
    record_status(status, code);
  }
  return ok != 0;
}

// One softmax step (thread = one row, 128 scores): scores in, probabilities out.  As persist_softmax_step, with a factor and an
// addend for each sixteen keys (coef: key scale, log2 of the value scale, the scale's inverse, the logarithm as the maximum takes
// it) and, in a form of its own that keeps the other one short, `valid` keys visible to this row.  m is the largest (score factor +
// addend) so far in log2 units, moved only when it has grown by more than 2^8.  Hidden scores are -inf before they meet their
// factor, which therefore may not vanish: a row of zeros has 2^-126 of its own, and a small key scale would take it to 0 and the
// score to NaN.
template <bool kHalf, bool kMasked>
__device__ __forceinline__ void tile_softmax_step(const TileRefs& r, int step, bool first, int valid, float row_factor, const float4* coef,
                                                  float& m, float& l_sum, volatile int* abort_flag, int* status) {
  uint32_t s[4][32];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld32(r.t_s + c * 32, s[c]);
  tmem_wait_ld();
  tc_fence_before_sync();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(r.bar_s_empty);
  if constexpr (kMasked) {
#pragma unroll
    for (int i = 0; i < 128; ++i)
      if (i >= valid) s[i >> 5][i & 31] = 0xff800000u;  // -inf
  }
  auto factor = [&](const float4& k) {
    const float f = row_factor * k.x;
    return kMasked ? fmaxf(f, FLT_MIN) : f;
  };
  float mx = -INFINITY;
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t* x = &s[c >> 1][(c & 1) * 16];
    float a = max3(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
    float b = max3(__uint_as_float(x[3]), __uint_as_float(x[4]), __uint_as_float(x[5]));
    a = max3(a, __uint_as_float(x[6]), __uint_as_float(x[7]));
    b = max3(b, __uint_as_float(x[8]), __uint_as_float(x[9]));
    a = max3(a, __uint_as_float(x[10]), __uint_as_float(x[11]));
    b = max3(b, __uint_as_float(x[12]), __uint_as_float(x[13]));
    a = max3(a, __uint_as_float(x[14]), __uint_as_float(x[15]));
    const float4 k = coef[c];
    mx = fmaxf(mx, fmaf(fmaxf(a, b), factor(k), k.w));
  }
  if (first) {
    m = mx;
  } else {
    const bool need = mx > m + kRescaleThreshold;
    if (__any_sync(0xffffffffu, need)) {
      tile_wait(r.bar_pv, (step - 1) & 1, abort_flag, status, kDevTimeoutSoftmax);
      __syncwarp();
      tc_fence_after_sync();
      const float f = need ? fast_exp2(m - mx) : 1.0f;
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        uint32_t o[16];
        tmem_ld16(r.t_o + c * 16, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tmem_st16(r.t_o + c * 16, o);
      }
      l_sum *= f;
      if (need) m = mx;
    }
  }
  // (looked at early, so that the answer is there when the first probabilities are stored)
  const bool pv_done = step == 0 || mbar_try_wait(r.bar_pv, (step - 1) & 1);
  const float shift = m == -INFINITY ? 0.f : kProbShift - m;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t pk[32];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = half * 4 + q;
      const float4 k = coef[c];
      const float f = factor(k), add = k.y + shift;
      const float2 f2 = make_float2(f, f), add2 = make_float2(add, add);
      const uint32_t* x = &s[c >> 1][(c & 1) * 16];
      float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        float2 x0 = __ffma2_rn(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), f2, add2);
        float2 x1 = __ffma2_rn(make_float2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), f2, add2);
        x0.x = fast_exp2(x0.x);
        x0.y = fast_exp2(x0.y);
        x1.x = fast_exp2(x1.x);
        x1.y = fast_exp2(x1.y);
        la = __fadd2_rn(la, x0);
        lb = __fadd2_rn(lb, x1);
        pk[q * 8 + (i >> 1)] = pack2<kHalf>(x0.x, x0.y);
        pk[q * 8 + (i >> 1) + 1] = pack2<kHalf>(x1.x, x1.y);
      }
      la = __fadd2_rn(la, lb);
      l_sum = fmaf(la.x + la.y, k.z, l_sum);
    }
    // 64 probabilities done: hand this half to the issuing warp
    if (half == 0) {
      if (!pv_done) tile_wait(r.bar_pv, (step - 1) & 1, abort_flag, status, kDevTimeoutSoftmax);
      __syncwarp();  // (lanes may have found out on their own; the store below is the warp's)
      tc_fence_after_sync();
    }
    tmem_st32(r.t_p + half * 32, pk);
    tmem_wait_st();
    tc_fence_before_sync();
    mbar_arrive(r.bar_p + 8 * half);
  }
}

template <bool kFp16, bool kEightBit>
__global__ void __launch_bounds__(kTileThreads, 1)
attn_cache_tile_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CacheAttnParams p) {
  using Shape = TileShape<kEightBit>;
  constexpr int kSlots = Shape::slots, kRaw = Shape::raw_slots;
  constexpr bool kHalf = kEightBit || kFp16;  // fp16 products
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t q_smem = smem_base;                      // 2 tiles
  const uint32_t kv_smem = smem_base + 2 * kTileBytes;    // kSlots operand tiles
  const uint32_t raw_smem = kv_smem + kSlots * kTileBytes;
  float4* coef_ring = reinterpret_cast<float4*>(smem_gen + Shape::coef_at);
  uint8_t* ctl = smem_gen + Shape::bar_at;
  const uint32_t bars = smem_u32(ctl);
  const uint32_t bar_raw_full = bars;                     // [kRaw] copies have landed
  const uint32_t bar_raw_empty = bar_raw_full + 8 * 5;    // [kRaw] codes have been widened (8-bit pages)
  const uint32_t bar_kv_full = bar_raw_empty + 8 * 5;     // [kSlots]
  const uint32_t bar_kv_empty = bar_kv_full + 8 * 5;      // [kSlots]
  const uint32_t bar_coef = bar_kv_empty + 8 * 5;         // [kCoefStages]
  const uint32_t bar_q_ready = bar_coef + 8 * kCoefStages;  // [2]
  const uint32_t bar_s_full = bar_q_ready + 16;           // [2]
  const uint32_t bar_p_full = bar_s_full + 16;            // [2][2]
  const uint32_t bar_pv = bar_p_full + 32;                // [2]
  const uint32_t bar_s_empty = bar_pv + 16;
  const uint32_t bar_drain = bar_s_empty + 8;             // [3]
  const uint32_t bar_seg = bar_drain + 24;                // [kSegStages] a block is described
  const uint32_t bar_seg_empty = bar_seg + 8 * kSegStages;  // [kSegStages] and has been read
  int* raw_rows = reinterpret_cast<int*>(ctl + 464);       // [kRaw] rows of the copy that exist, -1: no more
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 484);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctl + 488);
  TileSeg* segs = reinterpret_cast<TileSeg*>(smem_gen + Shape::seg_at);
  static_assert(8 * (20 + kCoefStages + 2 * kSegStages) + 16 + 16 + 32 + 16 + 8 + 24 <= 464 && kRaw <= 5 && kSlots <= 5, "control block");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 32) {
    *abort_flag = 0;
    for (int s = 0; s < kRaw; ++s) {
      mbar_init(bar_raw_full + 8 * s, 1);
      mbar_init(bar_raw_empty + 8 * s, 4);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(bar_kv_full + 8 * s, 4);
      mbar_init(bar_kv_empty + 8 * s, 2);
    }
    for (int s = 0; s < kCoefStages; ++s) mbar_init(bar_coef + 8 * s, 1);
    for (int s = 0; s < kSegStages; ++s) {
      mbar_init(bar_seg + 8 * s, 1);
      mbar_init(bar_seg_empty + 8 * s, 11);  // the issuing and the softmax warps
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_q_ready + 8 * t, kTileM);
      mbar_init(bar_s_full + 8 * t, 1);
      mbar_init(bar_p_full + 16 * t, kTileM);
      mbar_init(bar_p_full + 16 * t + 8, kTileM);
      mbar_init(bar_pv + 8 * t, 1);
    }
    mbar_init(bar_s_empty, 4);
    for (int i = 0; i < 3; ++i) mbar_init(bar_drain + 8 * i, 1);
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  if (warp == 15 && lane == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int n_segs = 0;  // blocks that this warp has taken up
  // the next of them (n 0: there is none; the warp decides as one)
  auto next_seg = [&](TileSeg& seg) {
    const int e = n_segs % kSegStages;
    if (!__all_sync(0xffffffffu, tile_wait(bar_seg + 8 * e, (n_segs / kSegStages) & 1, abort_flag, p.status, kDevTimeoutMma))) return false;
    ++n_segs;
    seg = segs[e];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_seg_empty + 8 * e);
    return seg.n > 0;
  };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 15) {
      // ---------------------------------------------------------------- copies of pages, scales
      const int box_shift = min(p.page_shift, 7);
      const int boxes = kTileN >> box_shift;
      int slot = 0, phase = 0, tiles = 0;  // ring position, tiles so far
      bool given_up = false;
      TileWalk walk;
      TileJoin join = {};
      walk.begin(p, lane, blockIdx.x, gridDim.x);
      int t0, n;
      // lane l < boxes: the table's entry for the tile's l-th box, -1 where there is none
      auto entry = [&](int tile) {
        const int key = tile * kTileN + (lane << box_shift);
        int id = -1;
        if (lane < boxes && key < walk.w.seq.len) id = __ldg(p.block_table + walk.w.b * p.table_stride + (key >> p.page_shift));
        return id;
      };
      while (!given_up && walk.next(p, t0, n)) {
        tile_wait(bar_seg_empty + 8 * (n_segs % kSegStages), (n_segs / kSegStages & 1) ^ 1, abort_flag, p.status, kDevTimeoutLoad);
        if (lane == 0) {
          TileSeg& seg = segs[n_segs % kSegStages];
          const TileBlock& w = walk.w;
          seg.n = n;
          seg.t0 = t0;
          seg.tok0 = w.seq.tok0;
          seg.n_new = w.seq.n_new;
          seg.len = w.seq.len;
          seg.first = w.seq.first;
          seg.h = w.h;
          seg.blk = w.blk;
          seg.rows = min(p.tok_blk, w.seq.n_new - w.blk * p.tok_blk) * p.group;
          seg.piece = n == w.n_tiles ? -1 : 2 * static_cast<int>(blockIdx.x) + (w.start > walk.lo ? 1 : 0);
          if (t0 == 0 && n < w.n_tiles) {
            const long long last_tile = w.start + kBlockKeys + static_cast<long long>(w.n_tiles - 1) * kTileN;
            const long long per = walk.end - walk.lo;  // (a run that a block outlasts is a whole one)
            join = {static_cast<int>(last_tile / per) - static_cast<int>(blockIdx.x) + 1, seg.piece, seg.tok0 + w.blk * p.tok_blk, seg.rows, w.h, {}};
          }
          mbar_arrive(bar_seg + 8 * (n_segs % kSegStages));
        }
        ++n_segs;
        int next = entry(t0);
        for (int j = 0; j < n && !given_up; ++j, ++tiles) {
          const int tile = t0 + j;
          const int page = static_cast<unsigned>(next) < static_cast<unsigned>(p.n_pages) ? next : -1;
          if (j + 1 < n) next = entry(tile + 1);
          // scales of the tile's sixteen-key groups (the entry's last reader is eight tiles back)
          {
            const int from = __shfl_sync(0xffffffffu, page, (lane * 16 >> box_shift) & 31);
            if (lane < 8) {
              const float hidden = from < 0 ? -INFINITY : 0.f;
              float4 k = make_float4(1.f, hidden, 1.f, hidden);
              if (kEightBit && from >= 0) {
                const float ks = __ldg(p.scale[0] + from * p.s_page[0] + walk.w.h * p.s_head[0]);
                const float vs = fmaxf(__ldg(p.scale[1] + from * p.s_page[1] + walk.w.h * p.s_head[1]), kMinValueScale);
                const float log2_vs = __log2f(vs);
                k = make_float4(ks, log2_vs, __fdividef(1.f, vs), fmaxf(log2_vs, kLowValueLog2));
              }
              coef_ring[(tiles % kCoefStages) * 8 + lane] = k;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_coef + 8 * (tiles % kCoefStages));
          }
          for (int kv = 0; kv < 2; ++kv) {
            const bool ok = tile_wait((kEightBit ? bar_raw_empty : bar_kv_empty) + 8 * slot, phase ^ 1, abort_flag, p.status, kDevTimeoutLoad);
            given_up = given_up || !__all_sync(0xffffffffu, ok);
            const uint32_t bar = bar_raw_full + 8 * slot;
            if (lane == 0) {
              raw_rows[slot] = min(walk.w.seq.len - tile * kTileN, kTileN);
              mbar_arrive_expect_tx(bar, kEightBit ? kTileBytes / 2 : kTileBytes);
            }
            __syncwarp();
            if (lane < boxes) {
              const CUtensorMap* tm = kv ? &tm_v : &tm_k;
              const int token = (tile * kTileN + (lane << box_shift)) & ((1 << p.page_shift) - 1);
              const uint32_t at = (lane << box_shift) * 128;
              if constexpr (kEightBit) {
                tma_load_4d(raw_smem + slot * Shape::raw_bytes + at, tm, bar, 0, walk.w.h, token, page);
              } else {
                tma_load_4d(kv_smem + slot * kTileBytes + at, tm, bar, 0, walk.w.h, token, page);
                tma_load_4d(kv_smem + slot * kTileBytes + kHalfTileBytes + at, tm, bar, 64, walk.w.h, token, page);
              }
            }
            __syncwarp();
            if (++slot == kRaw) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
      }
      // no more: everybody goes home
      tile_wait(bar_seg_empty + 8 * (n_segs % kSegStages), (n_segs / kSegStages & 1) ^ 1, abort_flag, p.status, kDevTimeoutLoad);
      if (lane == 0) {
        reinterpret_cast<TileJoin*>(p.part + 2ll * gridDim.x * kTilePieceFloats)[blockIdx.x] = join;
        segs[n_segs % kSegStages].n = 0;
        mbar_arrive(bar_seg + 8 * (n_segs % kSegStages));
      }
      tile_wait((kEightBit ? bar_raw_empty : bar_kv_empty) + 8 * slot, phase ^ 1, abort_flag, p.status, kDevTimeoutLoad);
      if (lane == 0) {
        raw_rows[slot] = -1;
        mbar_arrive(bar_raw_full + 8 * slot);
        // Should a role have given up, nothing of ours may still be landing when the CTA retires (bounded polls on the last
        // copy into every slot, this one's arrival among them; a slot that was never filled counts as complete in its phase before the first).
        for (int i = 0; i < kRaw; ++i)
          for (int spin = 0; spin < (1 << 20) && !mbar_try_wait(bar_raw_full + 8 * i, i <= slot ? phase : phase ^ 1); ++spin) {
          }
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------------- matrix issuers
      const bool leader = elect_one();
      const int role = warp - 12;  // 0 scores; 1, 2 PV of tile 0, 1
      int slot = 0, phase = 0;     // the next key (role 0) or value tile
      auto advance = [&] {
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      if (role > 0) advance();
      if (role == 0) {
        constexpr uint32_t kIdescQK = umma_idesc(1, kHalf ? 0 : 1, kHalf ? 0 : 1, 0, kTileM, kTileN);
        const uint64_t q_desc0 = umma_smem_desc_sw128(q_smem, 16, 1024);
        const uint64_t k_desc0 = umma_smem_desc_sw128(kv_smem, 16, 1024);
        int q_uses[2] = {0, 0}, scores = 0;
        TileSeg seg;
        while (next_seg(seg)) {
          const int n = seg.n, n_qt = seg.rows > kTileM ? 2 : 1;
          for (int j = 0; j < n; ++j) {
            tile_wait(bar_kv_full + 8 * slot, phase, abort_flag, p.status, kDevTimeoutMma);
            for (int t = 0; t < n_qt; ++t) {
              if (j == 0) {
                tile_wait(bar_q_ready + 8 * t, q_uses[t] & 1, abort_flag, p.status, kDevTimeoutMma);
                ++q_uses[t];
              }
              // the columns of the scores are free once the softmax warps have the previous ones in registers
              if (scores > 0) tile_wait(bar_s_empty, (scores - 1) & 1, abort_flag, p.status, kDevTimeoutMma);
              ++scores;
              __syncwarp();
              tc_fence_after_sync();
              if (leader) {
                const uint64_t a0 = q_desc0 + static_cast<uint64_t>((t * kTileBytes) >> 4);
                const uint64_t b0 = k_desc0 + static_cast<uint64_t>((slot * kTileBytes) >> 4);
#pragma unroll
                for (int k = 0; k < kHeadDim / 16; ++k) {
                  const uint64_t off = static_cast<uint64_t>(((k >> 2) * kHalfTileBytes + (k & 3) * 32) >> 4);
                  umma_ss_f16(tmem_base, a0 + off, b0 + off, kIdescQK, k > 0);
                }
                umma_commit(bar_s_full + 8 * t);
              }
              __syncwarp();
            }
            if (leader) {  // (a slot is released by two arrivals: values have two readers)
              umma_commit(bar_kv_empty + 8 * slot);
              umma_commit(bar_kv_empty + 8 * slot);
            }
            __syncwarp();
            advance();
            advance();
          }
        }
      } else {
        constexpr uint32_t kIdescPV = umma_idesc(1, kHalf ? 0 : 1, kHalf ? 0 : 1, 1, kTileM, kHeadDim);
        const int t = role - 1;
        const uint64_t v_desc0 = umma_smem_desc_sw128(kv_smem, kHalfTileBytes, 1024);
        const uint32_t t_p = tmem_base + kTileN + t * 64;
        const uint32_t t_o = tmem_base + 2 * kTileN + t * kHeadDim;
        int steps = 0;  // the tile's steps so far
        TileSeg seg;
        while (next_seg(seg)) {
          const int n = seg.n, n_qt = seg.rows > kTileM ? 2 : 1;
          for (int j = 0; j < n; ++j) {
            tile_wait(bar_kv_full + 8 * slot, phase, abort_flag, p.status, kDevTimeoutMma);
            if (t < n_qt) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                tile_wait(bar_p_full + 16 * t + 8 * h, steps & 1, abort_flag, p.status, kDevTimeoutMma);
                __syncwarp();
                tc_fence_after_sync();
                if (leader) {
                  const uint64_t b0 = v_desc0 + static_cast<uint64_t>((slot * kTileBytes + h * 8192) >> 4);
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    umma_ts_f16(t_o, t_p + h * 32 + k * 8, b0 + static_cast<uint64_t>((k * 2048) >> 4), kIdescPV, (h > 0 || k > 0 || j > 0) ? 1u : 0u);
                  if (h == 1) umma_commit(bar_pv + 8 * t);
                }
                __syncwarp();
              }
              ++steps;
            }
            if (leader) umma_commit(bar_kv_empty + 8 * slot);
            __syncwarp();
            advance();
            advance();
          }
        }
      }
      // One more commit and a bounded poll on it: every arrival of this warp's commits has landed, and nothing writes tensor
      // memory after it has been freed below.
      if (leader) umma_commit(bar_drain + 8 * role);
      __syncwarp();
      for (int spin = 0; spin < (1 << 20) && !mbar_try_wait(bar_drain + 8 * role, 0); ++spin) {
      }
      __syncwarp();
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------------ codes to operands
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int tid = threadIdx.x - 256;
    int slot = 0, phase = 0, raw = 0, raw_phase = 0;
    bool values = false;
    while (true) {
      bool ok = tile_wait(bar_raw_full + 8 * raw, raw_phase, abort_flag, p.status, kDevTimeoutMma);
      if (!__all_sync(0xffffffffu, ok)) break;
      const int rows = reinterpret_cast<volatile int*>(raw_rows)[raw];
      if (rows < 0) break;
      if constexpr (kEightBit) {
        ok = tile_wait(bar_kv_empty + 8 * slot, phase ^ 1, abort_flag, p.status, kDevTimeoutMma);
        if (!__all_sync(0xffffffffu, ok)) break;
        // thread: channels 16 c .. 16 c + 15 of rows r, r + 16, ...; two 16-byte pieces of a swizzled row, the second panel's
        // threads in the other order (a quarter warp then covers all banks)
        const int c = tid & 7, r = tid >> 3;
        const uint32_t from = raw_smem + raw * Shape::raw_bytes + r * 128 + c * 16;
        const uint32_t to = kv_smem + slot * kTileBytes + (c >> 2) * kHalfTileBytes + r * 128;
        const int sw = r & 7, first = c >> 2;
        const uint32_t at0 = to + ((((c & 3) * 2 + first) ^ sw) << 4), at1 = to + ((((c & 3) * 2 + 1 - first) ^ sw) << 4);
        if (values && rows < kTileN) {
          // what the page holds behind the sequence's end may be anything: no weight is not enough
#pragma unroll 1
          for (int i = 0; i < 8; ++i)
            if (r + i * 16 >= rows) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(from + i * 2048), "r"(0) : "memory");
        }
#pragma unroll 1  // (the hot loops of all roles together should stay in the instruction cache: unrolled, 3 % slower)
        for (int half = 0; half < 2; ++half) {
          uint4 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = ld_shared16(from + (half * 4 + i) * 2048);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = first ? w[i].z : w[i].x, a1 = first ? w[i].w : w[i].y;
            const uint32_t b0 = first ? w[i].x : w[i].z, b1 = first ? w[i].y : w[i].w;
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at0 + (half * 4 + i) * 2048), "r"(widen_e4m3x2(a0)),
                         "r"(widen_e4m3x2(a0 >> 16)), "r"(widen_e4m3x2(a1)), "r"(widen_e4m3x2(a1 >> 16))
                         : "memory");
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at1 + (half * 4 + i) * 2048), "r"(widen_e4m3x2(b0)),
                         "r"(widen_e4m3x2(b0 >> 16)), "r"(widen_e4m3x2(b1)), "r"(widen_e4m3x2(b1 >> 16))
                         : "memory");
          }
        }
      } else if (values && rows < kTileN) {
        const uint32_t to = kv_smem + raw * kTileBytes + tid * 128;
        if (tid >= rows) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(to + i * 16), "r"(0) : "memory");
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(to + kHalfTileBytes + i * 16), "r"(0) : "memory");
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (kEightBit) mbar_arrive(bar_raw_empty + 8 * raw);
        mbar_arrive(bar_kv_full + 8 * (kEightBit ? slot : raw));
      }
      values = !values;
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
      if (++raw == kRaw) {
        raw = 0;
        raw_phase ^= 1;
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax, queries in, results out
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int t = warp >> 2, quad = warp & 3;
    const int row_in_tile = quad * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_o = tmem_base + lane_base + 2 * kTileN + t * kHeadDim;
    const TileRefs refs{tmem_base + lane_base, tmem_base + lane_base + kTileN + t * 64, t_o, bar_s_empty, bar_p_full + 16 * t, bar_pv + 8 * t};
    int steps = 0, tiles = 0;  // this tile's steps, the CTA's key tiles so far
    // A block's queries are fetched before the previous block's result is written, so that its first scores are formed
    // meanwhile.
    bool held = false;  // a result waits in tensor memory: the row's
    bool live = false;
    int row = 0, hq = 0, piece = 0;
    float m = -INFINITY, l_sum = 0.f;
    while (true) {
      TileSeg seg;
      bool more;
      while ((more = next_seg(seg)) && t * kTileM >= seg.rows) tiles += seg.n;
      const int r = t * kTileM + row_in_tile;
      const int in_blk = more ? r / p.group : 0;
      const int tok = seg.blk * p.tok_blk + in_blk;
      const int next_row = seg.tok0 + tok, next_hq = seg.h * p.group + r - in_blk * p.group;
      const bool next_live = more && r < seg.rows;
      float row_factor = p.scale_log2;
      if (more) {
        // The warp's 32 rows to shared memory, two at a time in whole lines (a row per thread was 4096 L1 accesses, 2 us): the last
        // QK^T that read this tile's rows is complete, its scores have been waited for.
        const unsigned long long src = next_live ? reinterpret_cast<unsigned long long>(static_cast<const uint16_t*>(p.q) + next_row * p.q_token + next_hq * p.q_head) : 0ull;
        const int half = lane >> 4, piece16 = lane & 15;
        uint4 v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const unsigned long long from = __shfl_sync(0xffffffffu, src, 2 * i + half);
          v[i] = from != 0ull ? __ldg(reinterpret_cast<const uint4*>(from) + piece16) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = quad * 32 + 2 * i + half;
          if constexpr (kEightBit && !kFp16) {
            uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            uint32_t top = 0;  // largest magnitude of the row, as bits (they order like the values)
#pragma unroll
            for (int k = 0; k < 4; ++k) top = max(top, max((x[k] << 16) & 0x7fff0000u, x[k] & 0x7fff0000u));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = min(max(static_cast<int>(top >> 23), 1), 253);
            const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = pack2<true>(__uint_as_float(x[k] << 16) * down, __uint_as_float(x[k] & 0xffff0000u) * down);
            v[i] = make_uint4(x[0], x[1], x[2], x[3]);
            const int mine = __shfl_sync(0xffffffffu, e, (lane & 1) * 16);
            if (lane >> 1 == i) row_factor *= __uint_as_float(static_cast<uint32_t>(mine) << 23);
          }
          *reinterpret_cast<uint4*>(smem_gen + t * kTileBytes + (piece16 >> 3) * kHalfTileBytes + r * 128 + (((piece16 & 7) ^ (r & 7)) << 4)) = v[i];
        }
        fence_proxy_async_smem();
        mbar_arrive(bar_q_ready + 8 * t);
      }
      if (held) {
        tile_wait(bar_pv + 8 * t, (steps - 1) & 1, abort_flag, p.status, kDevTimeoutEpilogue);
        __syncwarp();
        tc_fence_after_sync();
        if (piece < 0) {
          const float inv = l_sum == 0.f ? 0.f : 1.f / l_sum;
          uint16_t* dst = static_cast<uint16_t*>(p.out) + (row * (static_cast<size_t>(p.heads_kv) * p.group) + hq) * 128;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + c * 32, o);
            tmem_wait_ld();
            if (live) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = pack2<kFp16>(__uint_as_float(o[16 * h + 2 * i]) * inv, __uint_as_float(o[16 * h + 2 * i + 1]) * inv);
                if (p.out_aligned32) {
                  st_global32(dst + c * 32 + h * 16, v);
                } else {
                  uint4* d = reinterpret_cast<uint4*>(dst + c * 32 + h * 16);
                  d[0] = make_uint4(v[0], v[1], v[2], v[3]);
                  d[1] = make_uint4(v[4], v[5], v[6], v[7]);
                }
              }
            }
            __syncwarp();
          }
          if (live && p.lse != nullptr)
            p.lse[static_cast<size_t>(hq) * p.tokens + row] = l_sum == 0.f ? -INFINITY : (m - kProbShift + log2f(l_sum)) * 0.6931471805599453f;
        } else {
          // a piece: rows as they are, the maximum and the sum with them
          float* to = p.part + static_cast<long long>(piece) * kTilePieceFloats + t * (kTilePieceFloats / 2);
          float4* mine = reinterpret_cast<float4*>(to) + row_in_tile;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              mine[(c * 8 + (i >> 2)) * kTileM] = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
          }
          reinterpret_cast<float2*>(to + 32 * kTileM * 4)[row_in_tile] = make_float2(m, l_sum);
        }
        tc_fence_before_sync();
      }
      if (!more) break;
      held = true;
      live = next_live;
      row = next_row;
      hq = next_hq;
      piece = seg.piece;
      // keys visible to the row, from the block's first tile on
      int left = (live && p.causal ? min(seg.first + tok + 1, seg.len) : seg.len) - seg.t0 * kTileN;
      m = -INFINITY;
      l_sum = 0.f;
      for (int j = 0; j < seg.n; ++j, ++steps, ++tiles, left -= kTileN) {
        tile_wait(bar_s_full + 8 * t, steps & 1, abort_flag, p.status, kDevTimeoutSoftmax);
        // (complete by now, and only now its own phase: warps without rows in a block run ahead of the copies)
        tile_wait(bar_coef + 8 * (tiles % kCoefStages), (tiles / kCoefStages) & 1, abort_flag, p.status, kDevTimeoutSoftmax);
        __syncwarp();
        tc_fence_after_sync();
        const float4* coef = coef_ring + (tiles % kCoefStages) * 8;
        if (__any_sync(0xffffffffu, left < kTileN))
          tile_softmax_step<kHalf, true>(refs, steps, j == 0, left, row_factor, coef, m, l_sum, abort_flag, p.status);
        else
          tile_softmax_step<kHalf, false>(refs, steps, j == 0, left, row_factor, coef, m, l_sum, abort_flag, p.status);
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

// Merges the pieces of the blocks that runs' borders have cut: blockIdx.x is the run that has a block's first tile (of at most one
// block that ends behind it), blockIdx.y a group of 32 rows.  Eight warps, 16 channels each; a lane is a row.  Launched
// while attn_cache_tile_kernel still runs; its CTAs come to the SMs that have finished.
template <bool kFp16>
__global__ void __launch_bounds__(256)
attn_cache_join_kernel(const __grid_constant__ CacheAttnParams p, int ctas) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4* at = reinterpret_cast<const int4*>(reinterpret_cast<const TileJoin*>(p.part + 2ll * ctas * kTilePieceFloats) + blockIdx.x);
  const int4 d0 = __ldcg(at), d1 = __ldcg(at + 1);
  const TileJoin join = {d0.x, d0.y, d0.z, d0.w, d1.x, {}};
  const int r = blockIdx.y * 32 + lane;
  const bool live = r < join.n_rows;
  if (join.n_pieces == 0 || !__any_sync(0xffffffffu, live)) return;
  const int in_blk = r / p.group, hq = join.h * p.group + r - in_blk * p.group;
  const int t = r >> 7, row_in_tile = r & 127;
  const float* part = p.part + t * (kTilePieceFloats / 2);
  float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
#pragma unroll 2
  for (int i = 0; i < join.n_pieces; ++i) {
    const float* from = part + static_cast<long long>(i == 0 ? join.first : 2 * (blockIdx.x + i)) * kTilePieceFloats;
    const float2 st = __ldcg(reinterpret_cast<const float2*>(from + 32 * kTileM * 4) + row_in_tile);
    const float4* src = reinterpret_cast<const float4*>(from) + warp * 4 * kTileM + row_in_tile;
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __ldcg(src + j * kTileM);
    const float top = fmaxf(m, st.x);
    const float mine = m == -INFINITY ? 0.f : fast_exp2(m - top), theirs = st.x == -INFINITY ? 0.f : fast_exp2(st.x - top);
    m = top;
    l = l * mine + st.y * theirs;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[4 * j] = o[4 * j] * mine + v[j].x * theirs;
      o[4 * j + 1] = o[4 * j + 1] * mine + v[j].y * theirs;
      o[4 * j + 2] = o[4 * j + 2] * mine + v[j].z * theirs;
      o[4 * j + 3] = o[4 * j + 3] * mine + v[j].w * theirs;
    }
  }
  if (!live) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const size_t row = static_cast<size_t>(join.row + in_blk);
  uint16_t* dst = static_cast<uint16_t*>(p.out) + (row * (static_cast<size_t>(p.heads_kv) * p.group) + hq) * 128 + warp * 16;
  uint32_t v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = pack2<kFp16>(o[2 * i] * inv, o[2 * i + 1] * inv);
  uint4* d = reinterpret_cast<uint4*>(dst);
  d[0] = make_uint4(v[0], v[1], v[2], v[3]);
  d[1] = make_uint4(v[4], v[5], v[6], v[7]);
  if (warp == 0 && p.lse != nullptr)
    p.lse[static_cast<size_t>(hq) * p.tokens + row] = l == 0.f ? -INFINITY : (m - kProbShift + log2f(l)) * 0.6931471805599453f;
}

}  // namespace chitu
