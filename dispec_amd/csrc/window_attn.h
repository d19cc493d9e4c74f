// What the kernels of dsp_paged_window_attention share (window_attn.hip, window_prefill.hip,
// window_stream.h).
#pragma once

#include <float.h>

#include <algorithm>

#include "dsp_common.h"
#include "dsp_internal.h"
#include "dsp_mfma.h"
#include "dsp_quant.h"
#include "dsp_tile32.h"

namespace dsp_window {

using namespace dsp_mfma;
using dsp_quant::kFp4;
using dsp_quant::kFp8;
using dsp_quant::kNone;

// The 16-bit operands that hold a probability where q has 16 bits.
template <int D>
constexpr int prob_terms() {
  return D > 128 ? 3 : 1;
}
// By how much, in powers of two, a score may exceed the running maximum before it moves.  (fp16 in three
// operands: by little, so that a row's largest probability is 2^13 or more and what pack8 keeps above 0
// in the second and third, 2^-24 each, is 2^-36 of it: fp32's last bit after 4096 such keys)
template <typename Tag, int kTerms>
constexpr float lag() {
  return std::is_same<Tag, F16Tag>::value && kTerms == 3 ? 2.f : 8.f;
}

constexpr int kWholeWindow = 1 << 30;  // a window that no context reaches the end of

struct WinArgs {
  const void* q;
  int64_t qst, qsh;                // elements
  const char* kc;
  const char* vc;
  const uint8_t* ks;               // scales of a quantised cache
  const uint8_t* vs;
  uint32_t num_blocks;
  int64_t slot_bytes, head_bytes;  // of kc and vc
  int64_t scale_slot, scale_head;  // of ks and vs
  const int32_t* bt;
  int64_t bt_stride;
  int32_t log2_bs;
  const int32_t* cu_q;             // null: one query a sequence
  const int32_t* ctx_lens;
  int32_t B, KVH, G, max_q_len, max_ctx, window, sinks;
  float scale_log2;
  // tile kernel: tiles of a (sequence, KV head), parts of a tile, chunks of a part
  int32_t tiles, parts, part_chunks;
  // stream kernel: KV heads of a workgroup; runs that the list of chunks is cut into, the least units
  // of one, what a tile's start counts as; 2^16 / G, rounded up
  int32_t heads, runs, least, start, inv_g;
  int32_t* desc;
  float* ws_acc;
  float* ws_ml;
  void* out;
  int64_t ost, osh;
  int32_t vec_out;
  int32_t* err;
};

// A number that every lane of the wave reads alike, by a scalar load.
__device__ __forceinline__ int32_t scalar_load(const int32_t* p) {
  return *reinterpret_cast<__attribute__((address_space(4))) const int32_t*>(
      reinterpret_cast<uintptr_t>(p));
}

struct Seq {
  int q0, n, ctx;
  bool bad;   // lengths that are none: counted, rows of zeros
  int queries, rows;   // queries that are computed, and their packed rows
};
__device__ __forceinline__ Seq sequence(const WinArgs& a, int b) {
  Seq s;
  s.ctx = scalar_load(a.ctx_lens + b);
  s.q0 = a.cu_q ? scalar_load(a.cu_q + b) : b;
  s.n = a.cu_q ? scalar_load(a.cu_q + b + 1) - s.q0 : 1;
  s.bad = s.n > 0 && (s.ctx < s.n || s.ctx > a.max_ctx);
  s.queries = min(s.n, a.max_q_len);
  s.rows = s.queries * a.G;
  return s;
}

__device__ __forceinline__ int wave_incl_scan(int v) {
  const int lane = __lane_id();
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Chunks of kSize keys of a tile whose rows are those of queries at positions pf .. pl: `sink` from key
// 0 on, then those from key kSize * first on, n in all.
struct Span {
  int lo, hi;      // keys of the window: lo .. hi - 1
  int sink, first, n;
};
template <int kSize>
__device__ __forceinline__ Span span_of(int pf, int pl, int window, int sinks) {
  Span s;
  s.hi = pl + 1;
  s.lo = max(pf - window + 1, 0);
  s.first = s.lo / kSize;
  s.sink = min((sinks + kSize - 1) / kSize, s.first);
  s.n = s.sink + (s.hi + kSize - 1) / kSize - s.first;
  return s;
}

template <typename Tag>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same<Tag, Bf16Tag>::value)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// Of each of two operands' 16-bit numbers, not negative (or NaN, the largest here), the larger.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t not_below(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

// Four elements of the output, from element `at` on.
template <typename Tag, bool kF32>
__device__ __forceinline__ void store4(const WinArgs& a, int64_t at, f32x4 v) {
  if constexpr (kF32) {
    float* p = static_cast<float*>(a.out) + at;
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = v[j];
  } else {
    uint16_t* p = static_cast<uint16_t*>(a.out) + at;
    const uint32_t lo = narrow2<Tag>(v[0], v[1]), hi = narrow2<Tag>(v[2], v[3]);
    if (a.vec_out) {
      *reinterpret_cast<dsp_u32x2*>(p) = dsp_u32x2{lo, hi};
    } else {
      p[0] = uint16_t(lo);
      p[1] = uint16_t(lo >> 16);
      p[2] = uint16_t(hi);
      p[3] = uint16_t(hi >> 16);
    }
  }
}

// One row's np parts merged: workspace row row0, then those from row1 on, `stride` rows apart.  Dims d .. d
// + 3, 8 parts loaded at a time; packed row r of KV head kvh.
template <typename Tag, int D, bool kF32>
__device__ __forceinline__ void merge_row(const WinArgs& a, int q0, int64_t row0, int64_t row1,
                                          int stride, int np, int r, int kvh, int d) {
  constexpr int kBatch = 8;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  float M = -INFINITY, L = 0.f;
  f32x4 A = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < np; p0 += kBatch) {
    f32x4 va[kBatch];
    f32x2 ml[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      va[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      ml[i] = f32x2{-INFINITY, 0.f};
      if (p0 + i < np) {
        const int64_t row = p0 + i == 0 ? row0 : row1 + int64_t(p0 + i - 1) * stride;
        va[i] = *reinterpret_cast<const f32x4*>(a.ws_acc + row * D + d);
        ml[i] = *reinterpret_cast<const f32x2*>(a.ws_ml + 2 * row);
      }
    }
    float bm = M;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) bm = fmaxf(bm, ml[i][0]);
    const float Mu = bm == -INFINITY ? 0.f : bm;
    const float keep = dsp_weight(M - Mu);
    L *= keep;
    A *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float x = dsp_weight(ml[i][0] - Mu);
      L = fmaf(ml[i][1], x, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = fmaf(va[i][e], x, A[e]);
    }
    M = bm;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int qi = r / a.G;
  const int64_t o = int64_t(q0 + qi) * a.ost + int64_t(kvh * a.G + r - qi * a.G) * a.osh + d;
  A *= inv;
  store4<Tag, kF32>(a, o, A);
}

// ---- which launch a shape takes
struct WinPlan {
  bool tile;    // the tile or the stream kernel (else, with a cache in q's type, the general one)
  bool stream;
  int rows, tiles, parts, part_chunks;
  int heads, runs, least, start;  // stream (WinArgs)
  bool once;    // ... K and V by non-temporal loads
};

// The stream kernel over caches of each format (window_stream_*.hip).
int stream_plain(int32_t D, int32_t dtype, const WinPlan& p, const WinArgs& a, hipStream_t s);
int stream_fp8(int32_t D, int32_t dtype, const WinPlan& p, const WinArgs& a, hipStream_t s);
int stream_fp4(int32_t D, int32_t dtype, const WinPlan& p, const WinArgs& a, hipStream_t s);

// Tiles of 256 rows (window_prefill.hip): q in 16 bits, D 64 or 128.
int wide_tiles(int D, int fmt, bool f16, unsigned grid, const WinArgs& a, hipStream_t s);

constexpr int kChunk = 64;  // keys per chunk of the tile kernels
// Chunks of the stream kernel, in keys, and waves of its workgroups: one workgroup fills a CU.
constexpr int kStreamChunk = 32;
constexpr int stream_block(int D) { return D > 128 ? 4 : 8; }
constexpr int kDesc = 8;  // ints that describe a run's merge: pieces, q0, rows, first row, first head

}  // namespace dsp_window
