// Rotary positions and the paged key/value cache's write side: what fills the cache that attn_cache.cuh reads.
//
// Rotation of a head's first `rot` channels by the factors (cos, sin) of the token's position, from an fp32 table
// [rows][rot / 2]: pairs are adjacent channels (2j, 2j + 1) or the two halves (j, j + rot / 2); channels from rot on pass,
// and so does a token whose position lies outside the table.  Products and sums are rounded one by one (no fused
// multiply-add), so that the result is that of the elementary operations.
#pragma once

#include "elementwise.cuh"

namespace chitu {

// A thread's piece of a head: 16 channels as two vectors of eight.  In the rotated part, piece u holds vectors u and
// u + rot / 16, so that both partners of a half-layout pair meet in one thread; behind it vectors rot / 8 + u' and half the
// rest further.  Neighbouring pieces are neighbouring 16 bytes in both vectors.
__device__ __forceinline__ void piece_vectors(int u, int rot16, int n_pieces, int& v0, int& v1) {
  if (u < rot16) {
    v0 = u;
    v1 = u + rot16;
  } else {
    v0 = rot16 + u;
    v1 = v0 + n_pieces - rot16;
  }
}

// (cos, sin) of a piece's eight pairs.  Half layout: pairs 8u .. 8u + 7.  Adjacent: 4u .. 4u + 3 (first vector) and
// 4 (u + rot / 16) .. + 3 (second).
__device__ __forceinline__ void load_factors(const float2* row, int u, int rot16, bool interleaved, float (&c)[8], float (&s)[8]) {
  const float4* a = reinterpret_cast<const float4*>(row + (interleaved ? 4 * u : 8 * u));
  const float4* b = reinterpret_cast<const float4*>(row + (interleaved ? 4 * (u + rot16) : 8 * u + 4));
  const float4 f[4] = {__ldg(a), __ldg(a + 1), __ldg(b), __ldg(b + 1)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[2 * i] = f[i].x;
    s[2 * i] = f[i].y;
    c[2 * i + 1] = f[i].z;
    s[2 * i + 1] = f[i].w;
  }
}

__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
  a = x;
}
__device__ __forceinline__ void rotate_piece(float (&x)[8], float (&y)[8], bool interleaved, const float (&c)[8], const float (&s)[8]) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      rotate_pair(x[2 * i], x[2 * i + 1], c[i], s[i]);
      rotate_pair(y[2 * i], y[2 * i + 1], c[4 + i], s[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) rotate_pair(x[i], y[i], c[i], s[i]);
  }
}

template <int kDtype>
__device__ __forceinline__ void store8(void* p, size_t i, const float (&v)[8]) {
  if constexpr (kDtype == kFP32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 o;
    o.x = pack16(v[0], v[1], kDtype);
    o.y = pack16(v[2], v[3], kDtype);
    o.z = pack16(v[4], v[5], kDtype);
    o.w = pack16(v[6], v[7], kDtype);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = o;
  }
}

// ----------------------------------------------------------------------------
// rotary: up to three tensors of the same tokens
// ----------------------------------------------------------------------------
struct RotaryJob {
  const void* x;
  void* out;
  long long x_token, x_head, out_token, out_head;  // element strides
  int heads;
};
struct RotaryParams {
  RotaryJob job[3];
  int chunk_end[3];       // blockIdx.y of a tensor's last group of heads, plus one
  const void* positions;  // [tokens] int32 or int64
  int wide_positions;
  const float2* table;    // [rows][rot / 2]
  long long table_rows;
  int tokens, head_dim, rot, heads_each;
};

constexpr int kRotaryThreads = 256;

// Memory bound.  A thread owns a piece of a token's heads: the factors are read once and stay in registers while it walks
// heads_each heads of a tensor (blockIdx.y picks which), four of them in flight.  The first ones are asked for before the
// position is known, whose factors are two loads away.  32760 tokens, 24 heads of 128: 72 us, 5.9 TB/s (one head in flight 78).
template <int kDtype, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int kBatch = kDtype == kFP32 ? 2 : 4;
  const int pieces = p.head_dim >> 4, rot16 = p.rot >> 4;
  const int per_block = kRotaryThreads / pieces;
  const int local = threadIdx.x / pieces, u = threadIdx.x - local * pieces;
  const int t = blockIdx.x * per_block + local;
  if (local >= per_block || t >= p.tokens) return;
  const int y = blockIdx.y;
  const int j = (y >= p.chunk_end[0]) + (y >= p.chunk_end[1]);
  const RotaryJob& jb = p.job[j];
  int v0, v1;
  piece_vectors(u, rot16, pieces, v0, v1);
  int h = (y - (j == 0 ? 0 : p.chunk_end[j - 1])) * p.heads_each;
  const int h_end = min(h + p.heads_each, jb.heads);
  const size_t x0 = static_cast<size_t>(t * jb.x_token), o0 = static_cast<size_t>(t * jb.out_token);
  RawVec8<kDtype> ra[kBatch], rb[kBatch];
  auto load = [&] {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (h + i < h_end) {
        ra[i] = ld_raw8<kDtype>(jb.x, x0 + (h + i) * jb.x_head + v0 * 8);
        rb[i] = ld_raw8<kDtype>(jb.x, x0 + (h + i) * jb.x_head + v1 * 8);
      }
  };
  load();
  const long long pos = p.wide_positions ? static_cast<const long long*>(p.positions)[t] : static_cast<const int*>(p.positions)[t];
  const bool turns = u < rot16 && pos >= 0 && pos < p.table_rows;
  float c[8], s[8];
  if (turns) load_factors(p.table + pos * (p.rot >> 1), u, rot16, kInterleaved, c, s);
  while (true) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (h + i >= h_end) break;
      float a[8], b[8];
      unpack8<kDtype>(ra[i], a);
      unpack8<kDtype>(rb[i], b);
      if (turns) rotate_piece(a, b, kInterleaved, c, s);
      const size_t oi = o0 + (h + i) * jb.out_head;
      store8<kDtype>(jb.out, oi + v0 * 8, a);
      store8<kDtype>(jb.out, oi + v1 * 8, b);
    }
    h += kBatch;
    if (h >= h_end) break;
    load();
  }
}

// ----------------------------------------------------------------------------
// append: rotated keys and plain values into pages, queries rotated on the way
// ----------------------------------------------------------------------------
//
// Token i of sequence b (packed: tokens cu[b] .. cu[b + 1]) takes position lens[b] - n_b + i, that is slot pos % page of
// page table[b][pos / page].  16-bit pages take the value as it is rounded.  An 8-bit page holds e4m3 codes and one
// scale for each head:
//   scale = max(the page's scale if it holds earlier tokens, 2^ceil(log2(max |x| / 448)) over the new ones)
//   code  = e4m3(x / scale), earlier codes: e4m3(code * old scale / scale) when the scale has grown.
// A power of two costs an e4m3 value nothing (its error is relative) and makes both divisions exact, so that raising a
// page's scale later only touches codes at the bottom of the range.
struct AppendParams {
  const void* src[3];           // k, v, q (nullptr: none)
  long long src_token[3], src_head[3];
  void* cache[2];
  long long c_page[2], c_token[2], c_head[2];  // strides, bytes
  float* scale[2];
  long long s_page[2], s_head[2];              // strides, elements
  void* q_out;                  // [tokens, heads_q, 128] contiguous
  const int* block_table;
  long long table_stride;       // entries from one sequence's row to the next
  const int* lens;
  const int* cu;
  const void* positions;        // [tokens] rows of the rotary table, or nullptr: the position in the sequence
  int wide_positions;
  const float2* rope;           // [rows][rot / 2] or nullptr
  long long rope_rows;
  int rot, interleaved;
  int batch, tokens, width, n_pages, heads_kv, heads_q, page, page_shift, slots, turns, kv_blocks;
};

__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
__device__ __forceinline__ float2 unpack_e4m3x2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// smallest power of two that brings amax to at most 448 = 1.75 * 2^8 (of nothing: the smallest normal number)
__device__ __forceinline__ float power_of_two_scale(float amax) {
  const uint32_t bits = __float_as_uint(fminf(amax, 3.4e38f));
  int e = static_cast<int>(bits >> 23) - 8;                  // biased exponent of 2^(floor(log2 amax) - 8)
  if ((bits & 0x7fffffu) > 0x600000u) ++e;                   // mantissa above 1.75
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);
}

// rotation of a piece by its position, where it has one
__device__ __forceinline__ void turn_piece(const AppendParams& p, int kind, int u, int rot16, long long pos, float (&x)[8], float (&y)[8]) {
  if (kind == 1 || u >= rot16 || pos < 0 || pos >= p.rope_rows) return;
  float c[8], s[8];
  load_factors(p.rope + pos * (p.rot >> 1), u, rot16, p.interleaved, c, s);
  if (p.interleaved)
    rotate_piece(x, y, true, c, s);
  else
    rotate_piece(x, y, false, c, s);
}
__device__ __forceinline__ long long rope_row(const AppendParams& p, int first, int c0, int tok) {
  if (p.positions == nullptr) return first + tok;
  return p.wide_positions ? static_cast<const long long*>(p.positions)[c0 + tok] : static_cast<const int*>(p.positions)[c0 + tok];
}
__device__ __forceinline__ float piece_max(const float (&x)[8], const float (&y)[8], float m) {
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, fmaxf(fabsf(x[e]), fabsf(y[e])));
  return m;
}
__device__ __forceinline__ void store_codes(uint8_t* at, const float (&f)[8], float inv) {
  uint2 w;
  w.x = pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
  w.y = pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
  *reinterpret_cast<uint2*>(at) = w;
}
__device__ __forceinline__ void rescale_codes(uint8_t* p8, float ratio) {
  uint2* at = reinterpret_cast<uint2*>(p8);
  uint2 w = *at;
  const float2 a = unpack_e4m3x2(w.x), b = unpack_e4m3x2(w.x >> 16), c = unpack_e4m3x2(w.y), d = unpack_e4m3x2(w.y >> 16);
  w.x = pack_e4m3x4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
  w.y = pack_e4m3x4(c.x * ratio, c.y * ratio, d.x * ratio, d.y * ratio);
  *at = w;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory");
}

// Many tokens.  A block takes a run of rows - an 8-bit page, whose maximum has to be known before anything is stored; elsewhere 64
// rows of a page or of the queries - of `turns` groups of heads one after the other, 4 threads per row and head, each with two rows'
// pieces.  The rows' factors stay in registers; values come through a ring of copies, each thread reading what it copied, so
// that a block has 48 KB on their way while it computes.  Memory bound: 12 prompts of 61 to 2603 tokens, 48 heads, 8-bit pages
// of 64: 76 us, 5.0 TB/s; with a group of heads per block and loads to registers 122.  blockIdx.x is (sequence, run of rows), y
// the heads: k, v, q.
template <int kThreads>
struct AppendShape {
  static constexpr int stages = kThreads == 256 ? 4 : kThreads == 512 ? 3 : 2;
  static constexpr int smem = stages * kThreads * 64;
};
template <bool kFp16, bool kEightBit, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 256 ? 2 : 1)
kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kIn = kFp16 ? kFP16 : kBF16;
  constexpr int kStages = AppendShape<kThreads>::stages;
  constexpr bool kKeep = kThreads <= 512;  // room for the factors
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float red[2][32];
  const int b = blockIdx.x / p.slots, slot0 = blockIdx.x - b * p.slots;
  const int c0 = min(max(__ldg(p.cu + b), 0), p.tokens), c1 = min(max(__ldg(p.cu + b + 1), c0), p.tokens);
  const int n_new = c1 - c0;
  if (n_new == 0) return;
  const int first = max(__ldg(p.lens + b), -(1 << 30)) - n_new;  // position of the first new token
  const int kind = static_cast<int>(blockIdx.y) < p.kv_blocks ? 0 : static_cast<int>(blockIdx.y) < 2 * p.kv_blocks ? 1 : 2;  // (kv_blocks 0: queries only)
  if (kind != 2 && first + n_new <= 0) return;  // (no token has a place)
  const int shift = kEightBit && kind != 2 ? p.page_shift : min(p.page_shift, 6);  // rows of a run
  const int group_threads = 4 << shift;
  const int sub = threadIdx.x / group_threads, tid = threadIdx.x - sub * group_threads;
  const int heads_each = kThreads / group_threads;
  const int heads = kind == 2 ? p.heads_q : p.heads_kv;
  const int head0 = (blockIdx.y - kind * p.kv_blocks) * p.turns * heads_each;
  const int n_turns = min(p.turns, (heads - head0 + heads_each - 1) / heads_each);
  const int u = tid & 7, r0 = tid >> 3;
  const int rot16 = p.rope != nullptr ? p.rot >> 4 : 0;
  int v0, v1;
  piece_vectors(u, rot16, 8, v0, v1);
  const uint32_t slot_smem = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + threadIdx.x * 16;
  const int run0 = kind == 2 ? 0 : max(first, 0) >> shift;
  const int n_runs = kind == 2 ? ((n_new - 1) >> shift) + 1 : ((first + n_new - 1) >> shift) - run0 + 1;
  for (int slot = slot0; slot < n_runs; slot += p.slots) {
    const int base = ((run0 + slot) << shift) - (kind == 2 ? 0 : first);  // token of row 0
    int page_id = 0, in_page = 0;
    if (kind != 2) {
      const int pos = (run0 + slot) << shift, entry = pos >> p.page_shift;
      in_page = pos & (p.page - 1);
      if (entry >= p.width) continue;
      page_id = __ldg(p.block_table + b * p.table_stride + entry);
      if (page_id < 0 || page_id >= p.n_pages) continue;
    }
    const int held = max(-base, 0);  // rows that hold earlier tokens
    bool there[2];
    const uint16_t* src[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tok = base + r0 + i * (1 << (shift - 1));
      there[i] = tok >= 0 && tok < n_new;
      src[i] = static_cast<const uint16_t*>(p.src[kind]) + (c0 + tok) * p.src_token[kind] + (head0 + sub) * p.src_head[kind];
    }
    auto copy = [&](int turn) {
      if (turn < n_turns && head0 + turn * heads_each + sub < heads) {
        const uint32_t dst = slot_smem + (turn % kStages) * (kThreads * 64);
        const long long off = turn * heads_each * p.src_head[kind];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (there[i]) {
            cp_async16(dst + (2 * i) * (kThreads * 16), src[i] + off + v0 * 8);
            cp_async16(dst + (2 * i + 1) * (kThreads * 16), src[i] + off + v1 * 8);
          }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) copy(s);
    float c[2][8], s[2][8];
    bool turns[2];
    const float2* factors[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      turns[i] = false;
      factors[i] = nullptr;
      if (!there[i] || kind == 1 || u >= rot16) continue;
      const long long pos = rope_row(p, first, c0, base + r0 + i * (1 << (shift - 1)));
      if (pos < 0 || pos >= p.rope_rows) continue;
      turns[i] = true;
      factors[i] = p.rope + pos * (p.rot >> 1);
      if constexpr (kKeep) load_factors(factors[i], u, rot16, p.interleaved, c[i], s[i]);
    }
#pragma unroll 1
    for (int turn = 0; turn < n_turns; ++turn) {
      const int head = head0 + turn * heads_each + sub;
      const bool live = head < heads;
      float old = 0.f;
      float* scale = nullptr;
      if (kEightBit && kind != 2 && live) {
        // (read by every thread before the barrier below, written by one behind it)
        scale = p.scale[kind] + page_id * p.s_page[kind] + head * p.s_head[kind];
        old = *reinterpret_cast<volatile float*>(scale);
      }
      cp_async_wait<kStages - 2>();
      const uint32_t from = slot_smem + (turn % kStages) * (kThreads * 64);
      float x[2][2][8];
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!live || !there[i]) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          RawVec8<kIn> raw;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(raw.a.x), "=r"(raw.a.y), "=r"(raw.a.z), "=r"(raw.a.w) : "r"(from + (2 * i + k) * (kThreads * 16)) : "memory");
          unpack8<kIn>(raw, x[i][k]);
        }
        if (turns[i]) {
          if constexpr (!kKeep) load_factors(factors[i], u, rot16, p.interleaved, c[i], s[i]);
          if (p.interleaved)
            rotate_piece(x[i][0], x[i][1], true, c[i], s[i]);
          else
            rotate_piece(x[i][0], x[i][1], false, c[i], s[i]);
        }
        if (kEightBit) amax = piece_max(x[i][0], x[i][1], amax);
      }
      float inv = 1.f;
      if (kEightBit && kind != 2) {
        // the page's maximum over its threads (whole warps: 4 * page is a multiple of 64)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int warps = group_threads >> 5, parity = turn & 1;
        if ((threadIdx.x & 31) == 0) red[parity][threadIdx.x >> 5] = amax;
        __syncthreads();  // (two buffers in turn: nobody is two groups ahead)
        for (int w = 0; w < warps; ++w) amax = fmaxf(amax, red[parity][sub * warps + w]);
        float now = power_of_two_scale(amax);
        if (held > 0) now = fmaxf(now, old);
        inv = __frcp_rn(now);
        if (live && held > 0 && now > old) {
          const float ratio = __fdiv_rn(old, now);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = r0 + i * (1 << (shift - 1));
            if (r >= held) continue;
            uint8_t* row = static_cast<uint8_t*>(p.cache[kind]) + page_id * p.c_page[kind] + r * p.c_token[kind] + head * p.c_head[kind];
            rescale_codes(row + v0 * 8, ratio);
            rescale_codes(row + v1 * 8, ratio);
          }
        }
        if (live && now != old && tid == 0) *scale = now;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!live || !there[i]) continue;
        const int r = r0 + i * (1 << (shift - 1));
        if (kind == 2) {
          const size_t at = (static_cast<size_t>(c0 + base + r) * p.heads_q + head) * 128;
          store8<kIn>(p.q_out, at + v0 * 8, x[i][0]);
          store8<kIn>(p.q_out, at + v1 * 8, x[i][1]);
          continue;
        }
        uint8_t* row = static_cast<uint8_t*>(p.cache[kind]) + page_id * p.c_page[kind] + (in_page + r) * p.c_token[kind] + head * p.c_head[kind];
        if constexpr (kEightBit) {
          store_codes(row + v0 * 8, x[i][0], inv);
          store_codes(row + v1 * 8, x[i][1], inv);
        } else {
          store8<kIn>(row, v0 * 8, x[i][0]);
          store8<kIn>(row, v1 * 8, x[i][1]);
        }
      }
      copy(turn + kStages - 1);
    }
    cp_async_wait<0>();
    if (kEightBit && kind != 2) __syncthreads();  // (the next run starts with the first buffer of maxima again)
  }
}

// A token or a few of each sequence: eight threads per sequence and head walk its new tokens, one page after the other
// (latency bound: 64 sequences, a token each, 48 heads: 3.0 us; a block for each of their pages and heads took 13.4).
template <bool kFp16, bool kEightBit>
__global__ void __launch_bounds__(256)
kv_append_few_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kIn = kFp16 ? kFP16 : kBF16;
  const int plane = blockIdx.y * 32 + (threadIdx.x >> 3), u = threadIdx.x & 7;
  const int kind = plane < p.heads_kv ? 0 : plane < 2 * p.heads_kv ? 1 : 2;
  const int head = plane - kind * p.heads_kv;
  if (kind == 2 && head >= p.heads_q) return;
  const unsigned mates = 0xffu << (threadIdx.x & 24);  // the head's eight lanes
  const int b = blockIdx.x;
  const int c0 = min(max(__ldg(p.cu + b), 0), p.tokens), c1 = min(max(__ldg(p.cu + b + 1), c0), p.tokens);
  const int n_new = c1 - c0;
  if (n_new == 0) return;
  const int first = max(__ldg(p.lens + b), -(1 << 30)) - n_new;
  const int rot16 = p.rope != nullptr ? p.rot >> 4 : 0;
  int v0, v1;
  piece_vectors(u, rot16, 8, v0, v1);
  RawVec8<kIn> ra, rb;
  auto load = [&](int tok) {
    const size_t at = static_cast<size_t>((c0 + tok) * p.src_token[kind] + head * p.src_head[kind]);
    ra = ld_raw8<kIn>(p.src[kind], at + v0 * 8);
    rb = ld_raw8<kIn>(p.src[kind], at + v1 * 8);
  };
  int tok = 0;
  if (kind != 2) tok = max(0, -first);  // (positions before the sequence's begin have no place)
  while (tok < n_new) {
    // tokens [tok, end) share a page
    const int pos0 = first + tok, slot = pos0 >> p.page_shift;
    const int end = kind == 2 ? n_new : min(n_new, ((slot + 1) << p.page_shift) - first);
    load(tok);
    int page_id = 0;
    if (kind != 2) {
      if (slot >= p.width) return;
      page_id = __ldg(p.block_table + b * p.table_stride + slot);
      if (page_id < 0 || page_id >= p.n_pages) {
        tok = end;
        continue;
      }
    }
    uint8_t* page = kind == 2 ? nullptr : static_cast<uint8_t*>(p.cache[kind]) + page_id * p.c_page[kind] + head * p.c_head[kind];
    float x[8], y[8], inv = 1.f;
    if (kEightBit && kind != 2) {
      float* scale = p.scale[kind] + page_id * p.s_page[kind] + head * p.s_head[kind];
      const float old = *reinterpret_cast<volatile float*>(scale);
      float amax = 0.f;
      for (int i = tok; i < end; ++i) {
        if (i > tok) load(i);
        unpack8<kIn>(ra, x);
        unpack8<kIn>(rb, y);
        turn_piece(p, kind, u, rot16, rope_row(p, first, c0, i), x, y);
        amax = piece_max(x, y, amax);
      }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mates, amax, o));
      const int held = pos0 & ((1 << p.page_shift) - 1);  // earlier tokens in the page
      float now = power_of_two_scale(amax);
      if (held > 0) now = fmaxf(now, old);
      inv = __frcp_rn(now);
      if (held > 0 && now > old) {
        const float ratio = __fdiv_rn(old, now);
#pragma unroll 4
        for (int r = 0; r < held; ++r) {
          rescale_codes(page + r * p.c_token[kind] + v0 * 8, ratio);
          rescale_codes(page + r * p.c_token[kind] + v1 * 8, ratio);
        }
      }
      __syncwarp(mates);  // (all eight have read the scale)
      if (now != old && u == 0) *scale = now;
      if (end - tok == 1) {  // (still in hand)
        uint8_t* row = page + held * p.c_token[kind];
        store_codes(row + v0 * 8, x, inv);
        store_codes(row + v1 * 8, y, inv);
        tok = end;
        continue;
      }
    }
    for (int i = tok; i < end; ++i) {
      if (i > tok || (kEightBit && kind != 2)) load(i);
      unpack8<kIn>(ra, x);
      unpack8<kIn>(rb, y);
      turn_piece(p, kind, u, rot16, rope_row(p, first, c0, i), x, y);
      if (kind == 2) {
        const size_t at = (static_cast<size_t>(c0 + i) * p.heads_q + head) * 128;
        store8<kIn>(p.q_out, at + v0 * 8, x);
        store8<kIn>(p.q_out, at + v1 * 8, y);
      } else {
        uint8_t* row = page + ((first + i) & ((1 << p.page_shift) - 1)) * p.c_token[kind];
        if constexpr (kEightBit) {
          store_codes(row + v0 * 8, x, inv);
          store_codes(row + v1 * 8, y, inv);
        } else {
          store8<kIn>(row, v0 * 8, x);
          store8<kIn>(row, v1 * 8, y);
        }
      }
    }
    tok = end;
  }
}

}  // namespace chitu
