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
  int n_jobs;
  const void* positions;  // [tokens] int32 or int64
  int wide_positions;
  const float2* table;    // [rows][rot / 2]
  long long table_rows;
  int tokens, head_dim, rot, heads_total, heads_each;
};

constexpr int kRotaryThreads = 256;

// Memory bound.  A thread owns a piece of a token's heads: the factors are read once and stay in registers while it walks
// heads_each heads of the tensors laid end to end (blockIdx.y picks which).
template <int kDtype, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(const __grid_constant__ RotaryParams p) {
  const int pieces = p.head_dim >> 4, rot16 = p.rot >> 4;
  const int per_block = kRotaryThreads / pieces;
  const int local = threadIdx.x / pieces, u = threadIdx.x - local * pieces;
  const int t = blockIdx.x * per_block + local;
  if (local >= per_block || t >= p.tokens) return;
  const long long pos = p.wide_positions ? static_cast<const long long*>(p.positions)[t] : static_cast<const int*>(p.positions)[t];
  const bool turns = u < rot16 && pos >= 0 && pos < p.table_rows;
  float c[8], s[8];
  if (turns) load_factors(p.table + pos * (p.rot >> 1), u, rot16, kInterleaved, c, s);
  int v0, v1;
  piece_vectors(u, rot16, pieces, v0, v1);
  int h = blockIdx.y * p.heads_each;
  const int h_end = min(h + p.heads_each, p.heads_total);
  int base = 0;
  for (int j = 0; j < p.n_jobs; ++j) {
    const RotaryJob& jb = p.job[j];
    const int end = min(h_end, base + jb.heads);
    const size_t x0 = static_cast<size_t>(t * jb.x_token), o0 = static_cast<size_t>(t * jb.out_token);
#pragma unroll 4
    for (; h < end; ++h) {
      const size_t xi = x0 + (h - base) * jb.x_head, oi = o0 + (h - base) * jb.out_head;
      const RawVec8<kDtype> ra = ld_raw8<kDtype>(jb.x, xi + v0 * 8), rb = ld_raw8<kDtype>(jb.x, xi + v1 * 8);
      float a[8], b[8];
      unpack8<kDtype>(ra, a);
      unpack8<kDtype>(rb, b);
      if (turns) rotate_piece(a, b, kInterleaved, c, s);
      store8<kDtype>(jb.out, oi + v0 * 8, a);
      store8<kDtype>(jb.out, oi + v1 * 8, b);
    }
    base += jb.heads;
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
  int batch, tokens, width, n_pages, heads_kv, heads_q, page, page_shift, heads_each, slots;
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

// Block: 4 * page threads for each of heads_each heads; a thread holds two rows' pieces (32 values), so a page is read once
// and its maximum is known before anything is stored.  blockIdx.x: (sequence, page of its new tokens), y: heads of k, then v,
// then q.
template <bool kFp16, bool kEightBit>
__global__ void __launch_bounds__(1024)
kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int kIn = kFp16 ? kFP16 : kBF16;
  __shared__ float red[32];
  const int group_threads = p.page * 4;
  const int sub = threadIdx.x / group_threads;
  const int tid = threadIdx.x - sub * group_threads;
  const int plane = blockIdx.y * p.heads_each + sub;
  const int planes = 2 * p.heads_kv + (p.src[2] != nullptr ? p.heads_q : 0);
  const bool live = plane < planes;
  const int kind = plane < p.heads_kv ? 0 : plane < 2 * p.heads_kv ? 1 : 2;
  const int head = plane - kind * p.heads_kv;
  const int b = blockIdx.x / p.slots, slot0 = blockIdx.x - b * p.slots;
  const int c0 = min(max(__ldg(p.cu + b), 0), p.tokens), c1 = min(max(__ldg(p.cu + b + 1), c0), p.tokens);
  const int n_new = c1 - c0;
  if (n_new == 0) return;
  const int first = __ldg(p.lens + b) - n_new;  // position of the first new token
  const int u = tid & 7, r0 = tid >> 3;
  const int rot16 = p.rope != nullptr ? p.rot >> 4 : 0;
  int v0, v1;
  piece_vectors(u, rot16, 8, v0, v1);
  const int page0 = max(first, 0) >> p.page_shift;
  const int n_slots = max((first + n_new - 1 - (page0 << p.page_shift)) >> p.page_shift, (n_new - 1) >> p.page_shift) + 1;
  for (int slot = slot0; slot < n_slots; slot += p.slots) {
    // rows of this block: positions of page page0 + slot (keys, values), or that many tokens (queries)
    const int base = kind == 2 ? slot << p.page_shift : ((page0 + slot) << p.page_shift) - first;  // token of row 0
    int page_id = 0;
    bool stored = live;
    if (kind != 2) {
      stored = stored && page0 + slot < p.width;
      if (stored) page_id = __ldg(p.block_table + b * p.table_stride + page0 + slot);
      stored = stored && page_id >= 0 && page_id < p.n_pages;
    }
    float x[2][2][8];
    bool here[2];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int tok = base + r0 + i * (p.page >> 1);
      here[i] = stored && tok >= 0 && tok < n_new;
      if (!here[i]) continue;
      const size_t at = static_cast<size_t>((c0 + tok) * p.src_token[kind] + head * p.src_head[kind]);
      const RawVec8<kIn> ra = ld_raw8<kIn>(p.src[kind], at + v0 * 8), rb = ld_raw8<kIn>(p.src[kind], at + v1 * 8);
      long long pos = first + tok;
      if (p.positions != nullptr)
        pos = p.wide_positions ? static_cast<const long long*>(p.positions)[c0 + tok] : static_cast<const int*>(p.positions)[c0 + tok];
      unpack8<kIn>(ra, x[i][0]);
      unpack8<kIn>(rb, x[i][1]);
      if (kind != 1 && u < rot16 && pos >= 0 && pos < p.rope_rows) {
        float c[8], s[8];
        load_factors(p.rope + pos * (p.rot >> 1), u, rot16, p.interleaved, c, s);
        if (p.interleaved)
          rotate_piece(x[i][0], x[i][1], true, c, s);
        else
          rotate_piece(x[i][0], x[i][1], false, c, s);
      }
      if constexpr (kEightBit) {
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(fabsf(x[i][0][e]), fabsf(x[i][1][e])));
      }
    }
    float inv = 1.f;
    if constexpr (kEightBit) {
      // (read by every thread before the barriers below, written by one behind them)
      float* scale = p.scale[kind == 1] + page_id * p.s_page[kind == 1] + head * p.s_head[kind == 1];
      const float old = stored && kind != 2 ? *reinterpret_cast<volatile float*>(scale) : 0.f;
      // the page's maximum over its threads (whole warps: 4 * page is a multiple of 64)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const int warp = threadIdx.x >> 5, warps = group_threads >> 5;
      __syncthreads();  // (an earlier round's maxima have been read)
      if ((threadIdx.x & 31) == 0) red[warp] = amax;
      __syncthreads();
      for (int w = 0; w < warps; ++w) amax = fmaxf(amax, red[sub * warps + w]);
      if (stored && kind != 2) {
        float now = power_of_two_scale(amax);
        const int held = max(-base, 0);  // rows of the page that hold earlier tokens
        if (held > 0) now = fmaxf(now, old);
        inv = __frcp_rn(now);
        if (held > 0 && now > old) {
          const float ratio = __fdiv_rn(old, now);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = r0 + i * (p.page >> 1);
            if (r >= held) continue;
            uint8_t* row = static_cast<uint8_t*>(p.cache[kind]) + page_id * p.c_page[kind] + r * p.c_token[kind] + head * p.c_head[kind];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint2* at = reinterpret_cast<uint2*>(row + (half ? v1 : v0) * 8);
              uint2 w = *at;
              const float2 a = unpack_e4m3x2(w.x), bb = unpack_e4m3x2(w.x >> 16), cc = unpack_e4m3x2(w.y), d = unpack_e4m3x2(w.y >> 16);
              w.x = pack_e4m3x4(a.x * ratio, a.y * ratio, bb.x * ratio, bb.y * ratio);
              w.y = pack_e4m3x4(cc.x * ratio, cc.y * ratio, d.x * ratio, d.y * ratio);
              *at = w;
            }
          }
        }
        if (now != old && tid == 0) *scale = now;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!here[i]) continue;
      const int r = r0 + i * (p.page >> 1);
      if (kind == 2) {
        const size_t at = (static_cast<size_t>(c0 + base + r) * p.heads_q + head) * 128;
        store8<kIn>(p.q_out, at + v0 * 8, x[i][0]);
        store8<kIn>(p.q_out, at + v1 * 8, x[i][1]);
        continue;
      }
      uint8_t* row = static_cast<uint8_t*>(p.cache[kind]) + page_id * p.c_page[kind] + r * p.c_token[kind] + head * p.c_head[kind];
      if constexpr (kEightBit) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float (&f)[8] = x[i][half];
          uint2 w;
          w.x = pack_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
          w.y = pack_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
          *reinterpret_cast<uint2*>(row + (half ? v1 : v0) * 8) = w;
        }
      } else {
        store8<kIn>(row, v0 * 8, x[i][0]);
        store8<kIn>(row, v1 * 8, x[i][1]);
      }
    }
  }
}

}  // namespace chitu
