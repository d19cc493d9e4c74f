// Attention of a drafted tree over the paged cache (speculative decoding with trees; the reference
// verifies chains, dispec/engine/model_runner.py:160-185).
//
//     o[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_ih . k_j),
//     j over the context before the tree and the nodes whose bit is set in node i's mask.
//
// All rows of a sequence see the whole context before the tree, so what a tile of rows costs is
// the same for all its tiles: ceil(ctx / 64) chunks of 64 keys.  The masks matter in the chunks
// that hold nodes only, the last one to few.
//
// Tile (16-bit caches): NW waves of 32 packed rows each (row r: query r / G of head kvh G + r % G)
// share 64-key chunks of K and V that the LDS DMA brings in; S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_32x32x16, with P in registers (dsp_tile32.h), a row's running maximum that moves when it
// is exceeded by 2^8, sums and accumulators in fp32.  Up to 128 dims the probabilities enter P V as
// one 16-bit operand (rounded to nearest; the sum takes the unrounded ones): half a step of the
// type, as much as the output's own rounding, as on the 16- and 128-row tiles of the multi-query
// attention (its ragged verify batches and decode of more than 8 heads a KV head hold more).  At 256
// dims they are three operands, all 24 bits, as in the other attention of such heads, which a
// tree's batch takes over from: 12 sequences of 16 nodes (G 2, 500 to 4000 tokens) 91 us, with one
// operand 68.5.
//  * Two workgroups of 4 waves (128 rows) to a CU for up to 128 rows a KV head, one of 8 waves (256
//    rows, a chunk loaded once for twice the rows) above.
//  * The list of (sequence, KV head, tile, chunk) units is cut into as many equal runs as there are
//    workgroups resident on the chip, computed on the device from the lengths; a tile's start counts
//    as kStart chunks.  A tile inside a run is written; a tile that runs cut leaves its rows'
//    maximum, sum and accumulator per piece, and the second launch merges them.
//  * What bounds it, heads of 128 in bf16: 32 trees of 16 nodes (G 2, 500 to 4000 tokens, 321 MB) 63
//    us and 5 of merge: 5.1 TB/s, 5 us of it until the first keys are there.  4 trees of 64 (G 4,
//    32768 tokens) 170 us and 8 of merge, 810 TFLOP/s (205 to 223 after a millisecond: the clock
//    falls): the matrix cores are busy for 37 % of the cycles, and two waves a SIMD, which issue in
//    order, spend 26 % of theirs waiting to issue and 34 % on barriers, loads and LDS.  24 trees of
//    1 to 33 nodes (40 to 3001 tokens) 26 us and 6: 5 chunks of 1.8 us a workgroup behind the chain
//    lengths, block ids, first keys.
// Everything else (fp32 caches, other head dims, blocks of fewer than 16 tokens, rows off 16 bytes,
// a scale that is not positive) runs on the kernels of generic_attn.hip with the same masks.
#include <float.h>

#include <algorithm>

#include "dsp_common.h"
#include "dsp_internal.h"
#include "dsp_mfma.h"
#include "dsp_tile32.h"

namespace {

using namespace dsp_mfma;

constexpr int kChunk = 64;     // keys per chunk
// A workgroup gets at least this many chunks: 4 heads of 63 26 us (29 with 1, 25.9 with 4), 2 of 16 13.2
// (12.3 with 1, 15.1 with 4).
constexpr int kMinChunks = 2;
// What a run spends on a tile beside its chunks (ids, q, the pipeline's first loads, a partial result
// or the output), in chunks: every tile counts as so many more when the list is cut.  32 sequences
// of 500 to 4000 tokens, 8 KV heads, D 128, 256 and 512 rows a head: 160 and 269 us (counted as
// nothing: 171 and 288); 4 to 8 pieces of equal tiles, where each has one start: 73 us (71).
constexpr int kStart = 4;
// K and V of a call that take so many bytes bypass the caches' replacement order (non-temporal loads):
// half of the last-level cache, behind which the next call finds little of its own anyway.  321 MB
// in 32 sequences 71.8 us (81.9 without), 130 MB in 6 35.5 (40.0); 42 MB that a call before left
// there 36.2 (33.7).
constexpr int64_t kStream = int64_t(128) << 20;
constexpr int kBlocks = 2048;  // block ids of a piece held in LDS
constexpr int kDesc = 8;       // ints that describe a run's merge: pieces, q0, rows, KV head, tile
constexpr int kMaskThreads = 256;

// One thread a node: its mask row is its own bit and its ancestors'.  Parents come before their
// children, so the chain up ends; a node whose parent is not an earlier one is a root.
__global__ __launch_bounds__(kMaskThreads) void tree_mask_kernel(
    const int32_t* __restrict__ parents, const int32_t* __restrict__ cu_q, int64_t rows,
    int32_t max_q_len, int32_t words, uint32_t* __restrict__ mask) {
  const int b = blockIdx.y, i = blockIdx.x * kMaskThreads + threadIdx.x;
  const int at = cu_q[b], n = min(cu_q[b + 1] - at, max_q_len);
  if (at < 0 || i >= n || int64_t(at) + i >= rows) return;
  uint32_t* row = mask + (int64_t(at) + i) * words;
  int a = i, w = i >> 5;
  uint32_t bits = 0;
  for (int x = words - 1; x > w; --x) row[x] = 0u;
  while (a >= 0) {
    for (; (a >> 5) < w; --w) {
      row[w] = bits;
      bits = 0;
    }
    bits |= 1u << (a & 31);
    const int p = parents ? parents[at + a] : a - 1;
    a = p < a ? p : -1;
  }
  for (; w >= 0; --w) {
    row[w] = bits;
    bits = 0;
  }
}

// a / b for 0 <= a < 2^24, 0 < b < 2^24: a reciprocal (to 24 bits, so that a times it is off by
// less than 1) and one correction, where the compiler's division is tens of instructions (a
// workgroup runs a chain of them before its first load).
struct Div {
  int b;
  float inv;
  __device__ __forceinline__ explicit Div(int d) : b(d) {
    const float f = float(d), x = __builtin_amdgcn_rcpf(f);
    inv = fmaf(fmaf(-f, x, 1.f), x, x);
  }
  __device__ __forceinline__ int operator()(int a) const {
    const int q = int(float(a) * inv), r = a - q * b;
    return r < 0 ? q - 1 : (r >= b ? q + 1 : q);
  }
};

// One sequence: `tiles` of TR packed rows (its first max_q_len nodes'), each of `chunks` units (one
// unit a tile where the tiles stay whole).
struct TreeSeq {
  int q0, n, ctx, rows, tiles, chunks, per_tile, units;
};
__device__ __forceinline__ bool tree_bad(int n, int ctx, int max_ctx) {
  return n > 0 && (ctx < n || ctx > max_ctx);
}
template <int TR>
__device__ __forceinline__ TreeSeq tree_seq(int q0, int q1, int ctx, int G, int max_q_len,
                                            int max_ctx, bool whole) {
  TreeSeq s;
  s.q0 = q0;
  s.n = q1 - q0;
  s.ctx = ctx;
  const bool none = s.n <= 0 || tree_bad(s.n, ctx, max_ctx);
  s.rows = none ? 0 : min(s.n, max_q_len) * G;
  s.tiles = (s.rows + TR - 1) / TR;
  s.chunks = none ? 0 : (ctx + kChunk - 1) / kChunk;
  s.per_tile = whole ? 1 : kStart + s.chunks;
  s.units = s.tiles * s.per_tile;
  return s;
}
__device__ __forceinline__ TreeSeq lane_seq(const TreeSeq& s, int l) {
  TreeSeq r;
  r.q0 = __builtin_amdgcn_readlane(s.q0, l);
  r.n = __builtin_amdgcn_readlane(s.n, l);
  r.ctx = __builtin_amdgcn_readlane(s.ctx, l);
  r.rows = __builtin_amdgcn_readlane(s.rows, l);
  r.tiles = __builtin_amdgcn_readlane(s.tiles, l);
  r.chunks = __builtin_amdgcn_readlane(s.chunks, l);
  r.per_tile = __builtin_amdgcn_readlane(s.per_tile, l);
  r.units = __builtin_amdgcn_readlane(s.units, l);
  return r;
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

// The shape of a tile: kNW waves of 32 rows, and buffers of a chunk's K and V: 128 KiB of them on a
// CU, for kPerCU workgroups.
template <int kNW, int kPerCU>
struct Shape {
  static constexpr int NW = kNW, TR = 32 * kNW;
  static constexpr int bufs(int D) { return 128 * 1024 / (4 * kChunk * D) / kPerCU; }
};

// Waits until at most n chunks' loads (kLoads each) of this wave are out, n <= kMost.
template <int kMost, int kLoads>
__device__ __forceinline__ void wait_chunks(int n) {
  if constexpr (kMost > 0) {
    if (n >= kMost) {
      __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<kMost * kLoads>());
      return;
    }
    wait_chunks<kMost - 1, kLoads>(n);
  } else {
    __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<0>());
  }
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

template <typename Tag>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same<Tag, Bf16Tag>::value)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// Of each of two operands' 16-bit numbers, not negative (or NaN, the largest here), the larger and
// the smaller.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t not_below(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t not_above(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

template <typename Tag>
__device__ __forceinline__ float low(uint32_t two) {
  return std::is_same<Tag, Bf16Tag>::value ? dsp_bf16lo(two) : dsp_f16lo(two);
}
template <typename Tag>
__device__ __forceinline__ float high(uint32_t two) {
  return std::is_same<Tag, Bf16Tag>::value ? dsp_bf16hi(two) : dsp_f16hi(two);
}

template <typename Tag, int D, typename S>
__global__ __launch_bounds__(64 * S::NW) __attribute__((amdgpu_waves_per_eu(D > 128 ? 1 : 2))) void
tree_tile_kernel(
    const uint16_t* __restrict__ q, int64_t qst, int64_t qsh, const uint16_t* __restrict__ kc,
    const uint16_t* __restrict__ vc, uint32_t num_blocks, int32_t kvs_slot, int64_t kvs_head,
    const int32_t* __restrict__ bt, int64_t bt_stride, int32_t log2_bs,
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ ctx_lens,
    const uint32_t* __restrict__ mask, int32_t words, int32_t B, int32_t KVH, int32_t G,
    int32_t max_q_len, int32_t max_ctx, float scale_log2, int32_t whole, int32_t least,
    int32_t stream_units, int32_t tiles_max, float* __restrict__ ws_acc, float* __restrict__ ws_ml,
    int32_t* __restrict__ ws_desc, uint16_t* __restrict__ out, int64_t ost, int64_t osh,
    int32_t vec_out, int32_t* __restrict__ err_count) {
  constexpr int NW = S::NW, TR = S::TR, NB = S::bufs(D);
  constexpr int NKS = D / 16, NDT = D / 32;      // 16-dim steps of K Q^T, 32-dim tiles of V^T P^T
  constexpr int CPR = D / 8, ROWB = 2 * D;       // 16-byte pieces and bytes of a K or V row
  constexpr int SLAB = kChunk * ROWB;            // a chunk of K (or V)
  constexpr int RPI = 1024 / ROWB;               // rows per 1-KiB DMA load
  constexpr int LPW = SLAB / 1024 / NW;          // loads per wave and slab
  constexpr int RPW = kChunk / NW;               // rows per wave: one block's
  constexpr int kTerms = D > 128 ? 3 : 1;        // operands that hold a probability
  static_assert(LPW >= 1 && LPW * RPI == RPW && RPW <= 16, "a wave's rows lie in one block");
  // Stage c of a piece is V of its chunk c and K of chunk c + 1, what one turn of the loop needs.
  // [buffer][K | V]
  __shared__ __attribute__((aligned(1024))) char lds[NB][2][SLAB];
  // of a stage, bit 2 wave: a wave's rows of K have a bad block id, 2 wave + 1: its rows of V hold
  // infinities or NaN.  Set before the stage's barrier, cleared after the next one's.
  __shared__ int32_t s_flag[4];
  __shared__ int32_t s_blk[kBlocks + 16];        // block ids of a piece (16: read ahead, not used)

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, col = lane & 31;
  const int lin = blockIdx.x;

  // ---- this workgroup's run.  Lane l holds sequence first + l of the 64 the wave looks at.
  int first = 0;
  TreeSeq mine;
  int incl = 0;
  auto look = [&](int f) {
    first = f;
    const int b = min(f + lane, B - 1);
    mine = tree_seq<TR>(cu_q[b], cu_q[b + 1], ctx_lens[b], G, max_q_len, max_ctx, whole != 0);
    if (f + lane >= B) mine.units = 0;
    incl = wave_incl_scan(mine.units);
  };
  int total = 0;  // units per KV head
  for (int f = 0; f < B; f += 64) {
    look(f);
    total += __builtin_amdgcn_readlane(incl, 63);
    // bad lengths (rare): counted once, the rows written as zeros, one sequence per workgroup
    uint64_t bad = __ballot(f + lane < B && tree_bad(mine.n, mine.ctx, max_ctx));
    for (; bad; bad &= bad - 1) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(bad)) - 1);
      if ((f + l) % int(gridDim.x) != lin) continue;
      if (threadIdx.x == 0 && err_count) atomicAdd(err_count, 1);
      const TreeSeq s = lane_seq(mine, l);
      const int row = KVH * G * D, n = min(s.n, max_q_len);
      for (int i = 0; i < n; ++i)
        for (int e = threadIdx.x; e < row; e += 64 * NW)
          out[int64_t(s.q0 + i) * ost + int64_t(e / D) * osh + e % D] = 0;
    }
  }
  const int C = total * KVH;
  const int W = min(C / least + (C % least != 0), int(gridDim.x));
  if (lin >= W) {
    if (!whole && tiles_max == 0 && threadIdx.x == 0) ws_desc[kDesc * lin] = 0;
    return;
  }
  // workgroup lin runs on XCD lin % 8: each XCD takes a contiguous part of the list, so that the
  // tiles and pieces of one (sequence, KV head) share an L2
  const int q8 = W / 8, r8 = W % 8, xcd = lin % 8, pos = lin / 8;
  const int w = xcd < r8 ? xcd * (q8 + 1) + pos : r8 * (q8 + 1) + (xcd - r8) * q8 + pos;
  const bool stream = C > stream_units;
  const Div by_w(W);
  const int share = C / W, extra = C - share * W;  // (C: of any size)
  int b = 0, kvh = 0, tile = 0, x = 0;   // where the run stands: unit x of a tile
  int base = 0;                          // units (of all KV heads) before sequence b
  TreeSeq sq;
  // unit u -> (b, kvh, tile, x); u < C
  auto locate = [&](int u) {
    for (int f = 0, pre = 0; f < B; f += 64) {
      if (f != first || B > 64) look(f);
      const uint64_t hit = __ballot(KVH * (pre + incl) > u);
      if (hit) {
        const int l = __builtin_amdgcn_readfirstlane(
            __ffsll(static_cast<unsigned long long>(hit)) - 1);
        sq = lane_seq(mine, l);
        b = f + l;
        base = KVH * (pre + __builtin_amdgcn_readlane(incl, l) - sq.units);
        break;
      }
      pre += __builtin_amdgcn_readlane(incl, 63);
    }
    int rest = u - base;
    kvh = __builtin_amdgcn_readfirstlane(Div(sq.units)(rest));
    rest -= kvh * sq.units;
    tile = __builtin_amdgcn_readfirstlane(Div(sq.per_tile)(rest));
    x = rest - tile * sq.per_tile;
  };
  // the tile after this one (there is one)
  auto next_tile = [&]() {
    x = 0;
    if (++tile < sq.tiles) return;
    tile = 0;
    if (++kvh < KVH) return;
    kvh = 0;
    base += KVH * sq.units;
    do {
      ++b;
      sq = tree_seq<TR>(cu_q[b], cu_q[b + 1], ctx_lens[b], G, max_q_len, max_ctx, whole != 0);
    } while (sq.units <= 0);
  };
  // Run v begins at unit floor(v C / W), or at the tile's first where that is one of its kStart.
  auto begin_of = [&](int v) {
    return __builtin_amdgcn_readfirstlane(v * share + by_w(v * extra));
  };
  int end = C;
  if (w + 1 < W) {
    end = begin_of(w + 1);
    if (!whole) {
      locate(end);
      if (x <= kStart) end -= x;
    }
  }
  int left = end - begin_of(w);
  locate(begin_of(w));
  if (!whole && x <= kStart) {
    left += x;
    x = 0;
  }

  // ---- its pieces: chunks c0 .. c1 of a tile
  auto kswz = [](int row) { return row & (CPR - 1); };
  auto vswz = [](int row) { return D >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); };
  const int bmask = (1 << log2_bs) - 1;
  const uint32_t slot_bytes = uint32_t(kvs_slot) * 2, blk_bytes = slot_bytes << log2_bs;
  uint32_t koff[LPW], voff[LPW];
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    const int rw = j * RPI + lane / CPR, row = RPW * wave + rw, sl = lane % CPR;
    koff[j] = uint32_t(rw) * slot_bytes + 16 * (sl ^ kswz(row));
    voff[j] = uint32_t(rw) * slot_bytes + 16 * (sl ^ vswz(row));
  }
  const uint32_t lds_base = uint32_t(reinterpret_cast<uintptr_t>((lds_void_t*)&lds[0][0][0]));
  int32_t d_np = 0, d_q0 = 0, d_rows = 0, d_kvh = 0, d_tile = 0;
  bool any_bad = false;
  for (bool again = false; left > 0; again = true) {
    const int nch = sq.chunks, c0 = x == 0 ? 0 : x - kStart;
    const int took = min(sq.per_tile - x, left);
    const int c1 = x + took == sq.per_tile ? nch : x + took - kStart;
    const int kbeg = c0 * kChunk, kfin = min(c1 * kChunk, sq.ctx), tree0 = sq.ctx - sq.n;
    const int r0 = tile * TR + 32 * wave;   // this wave's first row
    const int64_t bt_row = int64_t(b) * bt_stride;
    const bool wave_has_rows = r0 < sq.rows;
    const int r = r0 + col;
    const bool row_ok = r < sq.rows;
    const int qi = row_ok ? r / G : 0, tok = sq.q0 + qi;
    const int head = kvh * G + (row_ok ? r - qi * G : 0);
    dsp_u32x4 qop[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
      qop[ks] = row_ok ? *reinterpret_cast<const dsp_u32x4*>(q + int64_t(tok) * qst +
                                                             int64_t(head) * qsh + 16 * ks + 8 * hl)
                       : dsp_u32x4{0u, 0u, 0u, 0u};
    float m = -INFINITY, lpart = 0.f;
    f32x16 acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[dt][j] = 0.f;
    int blk0 = 0;                   // the first block id in s_blk
    // the block ids from the one that holds key t0 on, as many as fit; every wave is done with the
    // buffers and the ids
    auto stage_ids = [&](int t0) {
      blk0 = t0 >> log2_bs;
      const int n = min(kBlocks, ((kfin - 1) >> log2_bs) - blk0 + 1);
      for (int i = threadIdx.x; i < n; i += 64 * NW) s_blk[i] = bt[bt_row + blk0 + i];
      __syncthreads();
    };
    // This wave's RPW rows of a chunk lie in one block.  A chunk's K is sent for one stage ahead of
    // its V: the rows' offset is kept in between, the next chunk's id read from LDS a stage ahead.
    // (All uniform.)
    const char* const kbase = reinterpret_cast<const char*>(kc + int64_t(kvh) * kvs_head);
    const char* const vbase = reinterpret_cast<const char*>(vc + int64_t(kvh) * kvs_head);
    uint64_t rows_off = 0;          // of the chunk whose K was sent for last; its id is bad
    bool rows_bad = false;
    uint32_t bad_k = 0, bad_v = 0;  // buffers whose rows of this wave have a bad block id
    int32_t id_next = 0;
    auto first_key = [&](int c) { return min(kbeg + c * kChunk + RPW * wave, kfin - 1); };
    auto read_id = [&](int c) { id_next = s_blk[(first_key(c) >> log2_bs) - blk0]; };
    // rows from `rows` on into a slab; those past kfin as the last key's (a stale row may hold
    // anything)
    auto fetch = [&](const char* rows, int c, uint32_t m0, bool is_v) {
      if (kbeg + (c + 1) * kChunk > kfin) {
        const int room = kfin - 1 - first_key(c);
#pragma unroll
        for (int j = 0; j < LPW; ++j) {
          const int rw = j * RPI + lane / CPR, row = RPW * wave + rw, sl = lane % CPR;
          dma16<true>(rows, uint32_t(min(rw, room)) * slot_bytes +
                                16 * (sl ^ (is_v ? vswz(row) : kswz(row))), m0 + j * 1024);
        }
        return;
      }
      if (stream) {
#pragma unroll
        for (int j = 0; j < LPW; ++j) dma16<true>(rows, is_v ? voff[j] : koff[j], m0 + j * 1024);
      } else {
#pragma unroll
        for (int j = 0; j < LPW; ++j) dma16<false>(rows, is_v ? voff[j] : koff[j], m0 + j * 1024);
      }
    };
    auto slab_of = [&](int buf, int plane) {
      return lds_base + uint32_t((2 * buf + plane) * SLAB + wave * LPW * 1024);
    };
    auto send_k = [&](int c, int buf) {
      const uint32_t id = __builtin_amdgcn_readfirstlane(id_next);
      rows_bad = id >= num_blocks;   // (its rows: slots 0 ..)
      rows_off = rows_bad ? 0 : uint64_t(id) * blk_bytes +
                                    uint32_t(first_key(c) & bmask) * uint64_t(slot_bytes);
      any_bad |= rows_bad && kbeg + c * kChunk + RPW * wave < kfin;
      bad_k = (bad_k & ~(1u << buf)) | uint32_t(rows_bad) << buf;
      fetch(kbase + rows_off, c, slab_of(buf, 0), false);
      read_id(c + 1);
    };
    auto send_stage = [&](int c) {
      const int buf = c & (NB - 1);
      bad_v = (bad_v & ~(1u << buf)) | uint32_t(rows_bad) << buf;
      fetch(vbase + rows_off, c, slab_of(buf, 1), true);
      send_k(c + 1, buf);
    };
    if (again) __syncthreads();  // every wave is done with the previous piece's buffers, ids, flags
    if (threadIdx.x < 4) s_flag[threadIdx.x] = 0;
    stage_ids(kbeg);
    // the wait for the ids was one for the q rows too (issued before them): none is left to the
    // loop, whose loads the compiler cannot count
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) asm volatile("" : "+v"(qop[ks]));
    const int nc = c1 - c0;
    // stages whose ids are held: for those past them the ids are staged once the loads are done
    const int fit = int(min(int64_t(nc) + 1, (int64_t(kBlocks - 1) << log2_bs) / kChunk));
    int held = fit > nc ? nc : fit - 1;
    int sent = 0;           // stages sent for
    read_id(0);
    send_k(0, NB - 1);
    for (; sent < min(held, NB - 1); ++sent) send_stage(sent);
    __builtin_amdgcn_sched_barrier(0);
    wait_chunks<NB - 1, 2 * LPW>(sent);
    if ((bad_k >> (NB - 1)) & 1u && lane == 0) atomicOr(&s_flag[3], 1 << 2 * wave);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kBadK = 0x5555, kOddV = 0xaaaa;
    // Stage c is in LDS, for every wave: its loads are waited for, its flags (of every wave's rows)
    // returned.
    auto arrive = [&](int c) -> int {
      const int buf = c & (NB - 1);
      if (c == sent) {  // (a piece longer than the ids held)
        __syncthreads();
        stage_ids(kbeg + c * kChunk);
        held = nc - c < fit ? nc : c + fit - 1;
        read_id(c + 1);
        for (; sent < min(held, c + NB - 1); ++sent) send_stage(sent);
      }
      __builtin_amdgcn_sched_barrier(0);
      wait_chunks<NB - 2, 2 * LPW>(sent - c - 1);
      char* const my_v = &lds[buf][1][wave * LPW * 1024];  // the V rows this wave loaded
      int flag = (bad_k >> buf) & 1u;
      if ((bad_v >> buf) & 1u) zero_rows<CPR, LPW>(my_v, 0);
      if (kbeg + (c + 1) * kChunk > tree0) {
        __builtin_amdgcn_sched_barrier(0);
        flag |= any_nonfinite<Tag, LPW>(my_v) ? 2 : 0;
      }
      if (flag != 0 && lane == 0) atomicOr(&s_flag[c & 3], flag << 2 * wave);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      if (threadIdx.x == 0) s_flag[(c + 3) & 3] = 0;
      return s_flag[c & 3];
    };
    // The stage NB - 1 further on, into the buffer of stage c - 1, which every wave is done with.
    auto send_next = [&](int c) {
      if (sent < min(held, c + NB)) send_stage(sent++);
    };
    // ---- operands from LDS.  K: row 32*x + col of buffer buf, 16-byte piece 2*ks + hl, which lies at
    // piece (2*ks + hl) ^ kswz(row): the bits that ks sets are XORed into the address.  V^T: as in
    // load_vt, the bits of dt XORed likewise; 16-key steps and halves of them by whole rows.
    typedef __attribute__((address_space(3))) const dsp_u32x4 lds_u32x4_t;
    const uint32_t k_lane = lds_base + uint32_t(col * ROWB + 16 * (hl ^ kswz(col)));
    const uint32_t v_lane = lds_base + uint32_t(
        SLAB + (4 * hl + ((lane & 15) >> 2)) * ROWB +
        16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vswz((lane & 15) >> 2)) + 8 * (lane & 1));
    auto read_k = [&](uint32_t at, int x, int ks) {
      return *reinterpret_cast<lds_u32x4_t*>(((k_lane + at) ^ uint32_t(32 * ks)) +
                                             uint32_t(32 * x * ROWB));
    };
    auto read_v = [&](uint32_t at, int x, int ps, int dt) {
      v4i16 vh[2];
#pragma unroll
      for (int inst = 0; inst < 2; ++inst)
        vh[inst] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(
            ((v_lane + at) ^ uint32_t(64 * dt)) + uint32_t((32 * x + 16 * ps + 8 * inst) * ROWB)));
      return __builtin_bit_cast(dsp_u32x4, vh);
    };
    static_assert(D >= 64, "row strides of 128 bytes or more: the XORed bits lie inside a row");
    // Scores S^T (keys x rows) of half x of the chunk in buffer buf: sc[j] is key 32*x + 8*(j/4) +
    // 4*hl + j%4 of row col.
    auto scores = [&](int buf, int x, f32x16& sc) {
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        sc = mfma32x32<Tag>(read_k(buf * 2 * SLAB, x, ks), qop[ks], sc);
    };
    // The probabilities of a half that wait for their P V: as operands (P^T of two 16-key steps: step
    // ps takes registers j = 8*ps .. 8*ps + 7, i.e. keys 16*ps + 4*hl + {0..3, 8..11}), or, where
    // three operands hold one, in fp32 until their step (the operands of both would take 24
    // registers).
    dsp_u32x4 pop[2];
    f32x16 pend;
    auto operands = [&](int ps, dsp_u32x4 (&t)[kTerms]) {
      if constexpr (kTerms == 1) {
        t[0] = pop[ps];
      } else {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = pend[8 * ps + i];
        pack8<Tag, kTerms>(p, t);
      }
    };
    // O^T += V^T . P^T over half x of the chunk in buffer buf.
    auto add_pv = [&](int buf, int x) {
#pragma unroll
      for (int ps = 0; ps < 2; ++ps) {
        dsp_u32x4 t[kTerms];
        operands(ps, t);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          __builtin_amdgcn_sched_barrier(0);  // (registers)
          const dsp_u32x4 v = read_v(buf * 2 * SLAB, x, ps, dt);
#pragma unroll
          for (int k = 0; k < kTerms; ++k) acc[dt] = mfma32x32<Tag>(v, t[k], acc[dt]);
        }
      }
    };
    // Which keys of half x of chunk c the row sees, in a chunk that holds nodes (bit i: key 32*x +
    // 4*hl + i of it).
    auto window = [&](int c, int x) {
      return dsp_tree_window(mask + int64_t(tok) * words, words, sq.n,
                             kbeg + c * kChunk + 32 * x - tree0) >> (4 * hl);
    };
    // Half x of chunk c: keys that count for nothing (kflags: the flags that came with its K), and
    // whether a row's probabilities would exceed 2^(kRef + kLag); top: the largest score.
    // What m holds is the running maximum (base 2) less kRef: fp16's least number is 2^-24, bf16's
    // far below, so fp16 operands go up to 2^15 and end at 2^-31 of a row's largest probability
    // (without it a tail of keys below 2^-25 of a row's first key counted for nothing), three
    // operands at 2^-37.  Differences to m are one fma each, here as in prob, and the largest is
    // looked at before it is used: at 2^25 a step of fp32 is 4, and an fp16 operand could overflow.
    constexpr bool kF16 = std::is_same<Tag, F16Tag>::value;
    constexpr float kLag = kF16 && kTerms == 3 ? 2.f : 8.f, kRef = kF16 ? 15.f - kLag : 0.f;
    float top = 0.f;
    auto exceeds = [&] { return fmaf(top, scale_log2, -m) > kRef + kLag; };  // (-inf, -inf: no)
    auto settle = [&](int c, int x, int kflags, f32x16& sc) -> bool {
      if (kbeg + (c + 1) * kChunk > tree0) {
        const uint32_t seen = window(c, x);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sc[j] = (seen >> (8 * (j >> 2) + (j & 3))) & 1u ? sc[j] : -INFINITY;
      }
      if (const uint32_t bad = __builtin_amdgcn_readfirstlane(kflags) & kBadK; bad != 0) {
        // sc[j] lies in the chunk's 16-key group 2*x + j/8, whose id the wave that loaded it found
        // bad
#pragma unroll
        for (int g = 0; g < 2; ++g)
          if ((bad >> (2 * (((2 * x + g) * NW) / 4))) & 1u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) sc[8 * g + j] = -INFINITY;
          }
      }
      top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, sc[j]);
      top = fmaxf(top, dsp_shfl_xor(top, 32));
      return __builtin_amdgcn_ballot_w64(exceeds()) != 0;
    };
    // The running maximum of such a row moves: the sum and the accumulators
    // share it, so the result is the same.  Other rows of the wave keep theirs: what a row gives
    // does not depend on its neighbours.  The factor stays above 0: the accumulators may hold an
    // infinity, also of a key whose score is yet to come (take_odd), and 0 * inf is NaN.
    auto rescale = [&]() -> float {
      const bool moves = exceeds();
      float m_new = moves ? fmaf(top, scale_log2, -kRef) : m;
      if (moves && fmaf(top, scale_log2, -m_new) > 15.f)  // (steps of 16 and more: the next one up)
        m_new = __uint_as_float(__float_as_uint(m_new) + (m_new > 0.f ? 1 : -1));
      const float alpha = moves ? fmaxf(dsp_exp2(m - m_new), 0x1p-126f) : 1.f;
      m = m_new;
      lpart *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) acc[dt] *= alpha;
      return alpha;
    };
    auto prob = [&](const f32x16& sc, int j, float neg_m) {
      const float p = dsp_exp2(fmaf(sc[j], scale_log2, neg_m));
      lpart += p;
      return p;
    };
    // Of a chunk before the tree, which every row sees, an operand is kept above 0 (one: 2^-31 of the
    // row's largest probability in fp16, 2^-126 in bf16; three: pack8 keeps those of what is not
    // below kLeastP), so that an infinity in V meets a positive factor.  (Keys with a bad block id:
    // V is zeros.  A chunk that holds nodes: take_odd.)
    constexpr uint32_t kLeast = kF16 ? 0x00010001u : 0x00800080u;
    constexpr float kLeastP = kF16 ? 0x1p-24f : 0x1p-126f;
    auto before_tree = [&](int c) { return kbeg + (c + 1) * kChunk <= tree0; };
    // Exponentials e .. e + n of the half sc (n even) of chunk c (before: before_tree(c)), and their
    // operands.
    auto take_probs = [&](f32x16& sc, int e, int n, float neg_m, bool before, dsp_u32x4 (&to)[2]) {
#pragma unroll
      for (int j = e; j < e + n; ++j) {
        sc[j] = prob(sc, j, neg_m);
        if constexpr (kTerms == 1) {
          if (j & 1)
            to[j >> 3][(j >> 1) & 3] =
                not_below(narrow2<Tag>(sc[j - 1], sc[j]), before ? kLeast : 0u);
        } else {
          sc[j] = fmaxf(sc[j], before ? kLeastP : 0.f);  // (NaN: the sum has it)
        }
      }
    };
    // (rare) infinities and NaN of V of chunk c, in buffer buf, to the rows that see them; then they
    // are cleared
    auto take_odd = [&](int c, int buf) {
      if (wave_has_rows)
#pragma unroll 1
        for (int y = 0; y < 4; ++y) {
          const int x = y >> 1, ps = y & 1;
          const uint32_t seen = window(c, x);
          {
            dsp_u32x4 huge;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t two = seen >> (16 * ps + 8 * (i >> 1) + 2 * (i & 1));
              huge[i] = (two & 1u ? kHuge : 0u) | (two & 2u ? kHuge << 16 : 0u);
            }
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
              __builtin_amdgcn_sched_barrier(0);  // one tile's operands at a time: registers
              const dsp_u32x4 v = read_v(buf * 2 * SLAB, x, ps, dt);
              acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, false), huge, acc[dt]);
              acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, true), huge, acc[dt]);
            }
          }
        }
      __syncthreads();  // every wave has taken them
      clear_nonfinite<Tag, LPW>(&lds[buf][1][wave * LPW * 1024]);
      __syncthreads();
    };
    constexpr int kFirst = NB - 1;  // the buffer of K of chunk 0
    constexpr int kAhead = NDT < 3 ? NDT : 3;  // operands read ahead of their MFMAs
    constexpr int kSendAt = 1;  // the step of a chunk's first half in which the next stage is sent for
    static_assert(NKS <= 16 && NKS == 2 * NDT, "a step has one exponential or more");
    int kflags = s_flag[3];  // (in a vector register until it is looked at)
    // Half by half, a pipeline in which the MFMAs of one half's scores and of another's P V have
    // the exponentials of a third beside them, instruction by instruction (a wave issues in order:
    // MFMAs in a row, each after the wait for its operands, left the chip 67 % idle).  half(x): the
    // probabilities of cur; of half x of a stage, next = the scores and acc += P V with the
    // probabilities before (pop).
    f32x16 s0, s1;
    auto half = [&](auto xc, int c, int cx, int buf, int kfl, f32x16& cur, f32x16& next) {
      constexpr int x = decltype(xc)::value;
      const uint32_t at = uint32_t(buf * 2 * SLAB);
      dsp_u32x4 kop[NKS], vop[2 * NDT];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        kop[i] = read_k(at, x, i);
        vop[i] = read_v(at, x, i / NDT, i % NDT);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (settle(c, cx, kfl, cur)) {
        // the probabilities that still wait for their P V move along (one operand: rounded once
        // more, but the factor is below 2^-8 where it is not 1, and so is what that adds to the
        // row's error)
        const float alpha = rescale();
        if constexpr (kTerms == 1) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t two = pop[i >> 2][i & 3];
            pop[i >> 2][i & 3] =
                not_below(narrow2<Tag>(low<Tag>(two) * alpha, high<Tag>(two) * alpha),
                          not_above(two, kLeast));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) pend[j] = fmaxf(pend[j] * alpha, fminf(pend[j], kLeastP));
        }
      }
      const float neg_m = m == -INFINITY ? 0.f : -m;
      const bool before = before_tree(c);
      dsp_u32x4 fresh[2], t[kTerms];
#pragma unroll
      for (int j = 0; j < 16; ++j) next[j] = 0.f;
#pragma unroll
      for (int i = 0; i < NKS; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        if (i + kAhead < NKS) {
          kop[i + kAhead] = read_k(at, x, i + kAhead);
          vop[i + kAhead] = read_v(at, x, (i + kAhead) / NDT, (i + kAhead) % NDT);
        }
        next = mfma32x32<Tag>(kop[i], qop[i], next);
        if (x == 0 && i == kSendAt) send_next(c);
        take_probs(cur, 16 / NKS * i, 16 / NKS, neg_m, before, fresh);
        if (i % NDT == 0) operands(i / NDT, t);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < kTerms; ++k) acc[i % NDT] = mfma32x32<Tag>(vop[i], t[k], acc[i % NDT]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kTerms == 1) {
        pop[0] = fresh[0];
        pop[1] = fresh[1];
      } else {
        pend = cur;
      }
    };
    if (wave_has_rows) {
      scores(kFirst, 0, s0);
      if (settle(0, 0, kflags, s0)) rescale();
      take_probs(s0, 0, 16, m == -INFINITY ? 0.f : -m, before_tree(0), pop);
      if constexpr (kTerms > 1) pend = s0;
      scores(kFirst, 1, s1);
    }
    for (int c = 0; c < nc; ++c) {
      const int buf = c & (NB - 1);
      const int flags = arrive(c);
      if (kbeg + (c + 1) * kChunk > tree0 && (__builtin_amdgcn_readfirstlane(flags) & kOddV))
        take_odd(c, buf);
      if (wave_has_rows) {
        half(std::integral_constant<int, 0>{}, c, 1, buf, kflags, s1, s0);
        if (c + 1 < nc) half(std::integral_constant<int, 1>{}, c + 1, 0, buf, flags, s0, s1);
      } else {
        send_next(c);  // (it only loads)
      }
      kflags = flags;
    }
    if (wave_has_rows) add_pv((nc - 1) & (NB - 1), 1);
    // ---- the piece's rows: acc[dt][j] = O[row col][dim 32*dt + 8*(j/4) + 4*hl + j%4]
    lpart += dsp_shfl_xor(lpart, 32);
    const bool complete = c0 == 0 && c1 == nch;
    if (row_ok) {
      if (complete) {
        const float inv = lpart == 0.f ? 0.f : 1.f / lpart;  // (0: the row sees no key; NaN stays)
        uint16_t* o = out + int64_t(tok) * ost + int64_t(head) * osh;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int j4 = 0; j4 < 4; ++j4) {
            const f32x16& a = acc[dt];
            const uint32_t lo = narrow2<Tag>(a[4 * j4] * inv, a[4 * j4 + 1] * inv);
            const uint32_t hi = narrow2<Tag>(a[4 * j4 + 2] * inv, a[4 * j4 + 3] * inv);
            uint16_t* const at = o + 32 * dt + 8 * j4 + 4 * hl;
            if (vec_out) {
              *reinterpret_cast<dsp_u32x2*>(at) = dsp_u32x2{lo, hi};
            } else {
              at[0] = uint16_t(lo);
              at[1] = uint16_t(lo >> 16);
              at[2] = uint16_t(hi);
              at[3] = uint16_t(hi >> 16);
            }
          }
      } else {
        const int64_t wrow = int64_t(2 * w + (c0 == 0 ? 1 : 0)) * TR + 32 * wave + col;
        float* dst = ws_acc + wrow * D;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int j4 = 0; j4 < 4; ++j4)
            *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * j4 + 4 * hl) =
                f32x4{acc[dt][4 * j4], acc[dt][4 * j4 + 1], acc[dt][4 * j4 + 2],
                      acc[dt][4 * j4 + 3]};
        if (hl == 0) {
          ws_ml[2 * wrow] = m;
          ws_ml[2 * wrow + 1] = lpart;
        }
      }
    }
    if (c0 == 0 && !whole) {
      // this run began the tile: its merge is described here.  Pieces: up to the last run that
      // begins before the tile's end.
      int np = 0;
      if (!complete) {
        const int upto = base + (kvh * sq.tiles + tile + 1) * sq.per_tile;
        int v = min(W - 1, int(float(upto) * float(W) / float(C)));
        while (begin_of(v) >= upto) --v;
        while (v + 1 < W && begin_of(v + 1) < upto) ++v;
        np = v - w + 1;
        d_np = np;
        d_q0 = sq.q0;
        d_rows = sq.rows;
        d_kvh = kvh;
        d_tile = tile;
      }
      if (tiles_max > 0 && threadIdx.x == 0) {
        int32_t* d = ws_desc + kDesc * ((int64_t(b) * KVH + kvh) * tiles_max + tile);
        d[0] = np;
        d[1] = w;
      }
    }
    left -= took;
    if (left > 0) next_tile();
  }
  if (err_count && any_bad && lane == 0) atomicAdd(err_count, 1);  // once per wave
  if (!whole && tiles_max == 0 && threadIdx.x == 0) {
    int32_t* d = ws_desc + kDesc * w;
    d[0] = d_np;
    d[1] = d_q0;
    d[2] = d_rows;
    d[3] = d_kvh;
    d[4] = d_tile;
  }
}

// The merge of the tiles that runs cut.  One workgroup per (item, R rows); an item is a tile of the
// batch (tiles_max > 0: of the grid of tiles_max for each sequence and KV head) or, where there
// are fewer runs than tiles, the tile that a run began.  One thread per (row, 4 dims, every kSplit-th
// piece), its pieces loaded 8 at a time; the kSplit threads' results meet in LDS.  Neighbours in
// the grid are the row groups of one item; the runs that begin a tile often lie a multiple of 8
// apart, so the groups of every next 8 items start one XCD further (all of one XCD's: 47 us instead
// of 15 at 32 tiles of 256 rows in 8 pieces).  256 tiles of 128 rows in 2 to 3 pieces, 45 MB: 11.8 us.
constexpr int tree_merge_rows(int D, int split) { return 1024 / D / split; }

template <typename Tag, int D, int kSplit>
__global__ __launch_bounds__(256) void tree_merge_kernel(
    const float* __restrict__ ws_acc, const float* __restrict__ ws_ml,
    const int32_t* __restrict__ ws_desc, const int32_t* __restrict__ cu_q,
    const int32_t* __restrict__ ctx_lens, int32_t items, int32_t groups, int32_t KVH, int32_t G,
    int32_t max_q_len, int32_t max_ctx, int32_t tiles_max, int32_t tile_rows,
    uint16_t* __restrict__ out, int64_t ost, int64_t osh, int32_t vec_out) {
  constexpr int TPR = D / 4, R = tree_merge_rows(D, kSplit), kBatch = 8;
  __shared__ float s_acc[kSplit][R][D];
  __shared__ float s_ml[kSplit][R][2];
  const Div by_groups(groups);
  const int turn = blockIdx.x / 8;
  const int idx = 8 * turn + ((int(blockIdx.x % 8) - by_groups(turn)) & 7);
  const int item = by_groups(idx), group = idx - item * groups;
  if (item >= items) return;
  const int32_t* desc = ws_desc + int64_t(kDesc) * item;
  int np = desc[0], q0, rows, kvh, tile;
  int64_t w;
  if (tiles_max > 0) {
    const Div by_tiles(tiles_max), by_heads(KVH);
    const int head = by_tiles(item), b = by_heads(head);
    tile = item - head * tiles_max;
    kvh = head - b * KVH;
    w = desc[1];
    q0 = cu_q[b];
    const int n = cu_q[b + 1] - q0;
    // (a tile that the sequence does not have has no description)
    rows = n <= 0 || tree_bad(n, ctx_lens[b], max_ctx) ? 0 : min(n, max_q_len) * G;
  } else {
    w = item;
    q0 = desc[1];
    rows = desc[2];
    kvh = desc[3];
    tile = desc[4];
    if (np <= 0) return;
  }
  const int lr = group * R + threadIdx.x / TPR % R, d = 4 * (threadIdx.x % TPR);
  const int split = kSplit == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / (TPR * R));
  static_assert(kSplit == 1 || TPR * R == 64, "a wave's pieces");
  const int r = tile * tile_rows + lr;
  if (tile * tile_rows + group * R >= rows || np <= 0) return;  // (uniform)
  const bool live = lr < tile_rows && r < rows;
  float M = -INFINITY, L = 0.f;
  f32x4 A = f32x4{0.f, 0.f, 0.f, 0.f};
  if (live)
    for (int p0 = split; p0 < np; p0 += kSplit * kBatch) {
      f32x4 va[kBatch];
      f32x2 ml[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int p = p0 + kSplit * i;
        va[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        ml[i] = f32x2{-INFINITY, 0.f};
        if (p < np) {  // (uniform: no load for nothing)
          const int64_t row = (p == 0 ? 2 * w + 1 : 2 * (w + p)) * tile_rows + lr;
          va[i] = *reinterpret_cast<const f32x4*>(ws_acc + row * D + d);
          ml[i] = *reinterpret_cast<const f32x2*>(ws_ml + 2 * row);
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
  if constexpr (kSplit > 1) {
    const int at = lr - group * R;
    *reinterpret_cast<f32x4*>(&s_acc[split][at][d]) = A;
    if (d == 0) {
      s_ml[split][at][0] = M;
      s_ml[split][at][1] = L;
    }
    __syncthreads();
    if (split > 0) return;
    float bm = M;
#pragma unroll
    for (int i = 1; i < kSplit; ++i) bm = fmaxf(bm, s_ml[i][at][0]);
    const float Mu = bm == -INFINITY ? 0.f : bm, keep = dsp_weight(M - Mu);
    L *= keep;
    A *= keep;
#pragma unroll
    for (int i = 1; i < kSplit; ++i) {
      const float x = dsp_weight(s_ml[i][at][0] - Mu);
      const f32x4 o = *reinterpret_cast<const f32x4*>(&s_acc[i][at][d]);
      L = fmaf(s_ml[i][at][1], x, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = fmaf(o[e], x, A[e]);
    }
  }
  if (!live) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int qi = r / G;
  uint16_t* o = out + int64_t(q0 + qi) * ost + int64_t(kvh * G + r - qi * G) * osh + d;
  const uint32_t lo = narrow2<Tag>(A[0] * inv, A[1] * inv);
  const uint32_t hi = narrow2<Tag>(A[2] * inv, A[3] * inv);
  if (vec_out) {
    *reinterpret_cast<dsp_u32x2*>(o) = dsp_u32x2{lo, hi};
  } else {
    o[0] = uint16_t(lo);
    o[1] = uint16_t(lo >> 16);
    o[2] = uint16_t(hi);
    o[3] = uint16_t(hi >> 16);
  }
}

// ---- which launch a shape takes
struct TreePlan {
  bool tile;        // the tile kernel (else generic)
  bool whole;       // its tiles stay whole: no second launch
  int rows;         // of a tile
  int workers;      // workgroups, each with a run of the list
  int least;        // units that a run has at least
  int tiles_max;    // tiles of a sequence and KV head, where the merge goes by them (else 0: by runs)
  int items;        // of the merge
};

TreePlan tree_plan(int32_t B, int32_t KVH, int32_t G, int32_t D, int32_t max_q_len,
                   int32_t max_ctx) {
  TreePlan p{};
  if (!(D == 64 || D == 128 || D == 256) || B < 1 || max_q_len < 1 || max_ctx < 1) return p;
  const int64_t rows = int64_t(max_q_len) * G;
  // 256 rows take one workgroup of 8 waves to a CU, 128 rows two of 4 (D 256: one, for the buffers).
  // 32 sequences of 500 to 4000 tokens, 8 KV heads, D 128, bf16: 128 rows a head 110 us with two of
  // 4 (124 with one of 8); 192, 256 and 512 rows 160, 175 and 300 us with one of 8 (169, 186 and 311
  // with two of 4, which load a chunk for 128 rows each).
  p.rows = D > 128 || rows <= 128 ? 128 : 256;
  const int64_t per_head = (rows + p.rows - 1) / p.rows, tiles = per_head * B * KVH;
  const int64_t chunks = (int64_t(max_ctx) + kChunk - 1) / kChunk, units = chunks + kStart;
  // (numbers that Div divides: a sequence's units; 32 bits: all)
  p.tile = max_ctx < (1 << 24) && rows < (1 << 24) && per_head * units * KVH < (1 << 24) &&
           tiles * units < (int64_t(1) << 31);
  if (!p.tile) return p;
  // workgroups that fit the chip at once (LDS)
  const int64_t slots = int64_t(dsp_detail::device_cus()) * (p.rows == 128 && D <= 128 ? 2 : 1);
  // Short contexts: tiles stay whole where that costs less, in chunks, than equal runs, a start each
  // and the merge (its launch 3, its partial results 2 where there are as many as fit; half of all
  // that at D 256, whose chunks take two to four times as long).  The lengths are bounds here: only
  // up to 16 chunks.  Whole against cut, heads of 128: 512 tiles of 200 to 500 tokens 26.9 us
  // (36.0), of 300 to 1000 42.7 (46.5), 128 tiles 19.3 (20.4) and 28.8 (24.3); heads of 64, 2 tiles
  // of 300 tokens 12.2 (12.3), of 500 16.1 (13.1), of 1000 24.7 (13.2); of 256, captured in a graph,
  // 64 tiles of 200 to 500 36.6 (28.9), 256 tiles 51.6 (55.9).
  const int64_t runs = std::min((tiles * units + kMinChunks - 1) / kMinChunks, slots);
  const int64_t share = std::max((tiles * units + slots - 1) / slots, int64_t(kMinChunks));
  p.whole = chunks <= 16 &&
            (tiles + slots - 1) / slots * units <=
                share + (kStart + 3 + 2 * runs / slots) / (D > 128 ? 2 : 1);
  p.least = p.whole ? 1 : kMinChunks;
  p.workers = int(p.whole ? std::min(tiles, slots) : runs);
  p.tiles_max = tiles <= p.workers ? int(per_head) : 0;
  p.items = tiles <= p.workers ? int(tiles) : p.workers;
  return p;
}

size_t tree_tile_bytes(const TreePlan& p, int32_t D) {
  return p.whole ? 0 : size_t(p.workers) * (size_t(2) * p.rows * (D + 2) + kDesc) * sizeof(float);
}

template <typename Tag, int D>
int launch_tree(const TreePlan& p, const uint16_t* q, int64_t qst, int64_t qsh, const uint16_t* kc,
                const uint16_t* vc, int64_t num_slots, int64_t kvs_slot, int64_t kvs_head,
                const int32_t* bt, int64_t bt_stride, int32_t log2_bs, const int32_t* cu_q,
                const int32_t* ctx_lens, const uint32_t* mask, int32_t words, int32_t B,
                int32_t KVH, int32_t G, int32_t max_q_len, int32_t max_ctx, float scale_log2,
                float* ws, uint16_t* out, int64_t ost, int64_t osh, int32_t* err_count,
                hipStream_t s) {
  float* ws_ml = ws + int64_t(2) * p.workers * p.rows * D;
  int32_t* ws_desc = reinterpret_cast<int32_t*>(ws_ml + int64_t(4) * p.workers * p.rows);
  // (all tiles of a sequence and KV head read the same chunks)
  const int stream_units = int(std::min(
      kStream / (4 * kChunk * D) * ((int64_t(max_q_len) * G + p.rows - 1) / p.rows),
      (int64_t(1) << 31) - 1));
  const int vec_out = ost % 4 == 0 && osh % 4 == 0 && dsp_aligned(out, 8);
  auto launch = [&](auto shape) {
    using S = decltype(shape);
    tree_tile_kernel<Tag, D, S><<<p.workers, 64 * S::NW, 0, s>>>(
        q, qst, qsh, kc, vc, uint32_t(num_slots >> log2_bs), int32_t(kvs_slot), kvs_head, bt,
        bt_stride, log2_bs, cu_q, ctx_lens, mask, words, B, KVH, G, max_q_len, max_ctx, scale_log2,
        p.whole, p.least, stream_units, p.tiles_max, ws, ws_ml, ws_desc, out, ost, osh, vec_out,
        err_count);
  };
  if constexpr (D <= 128) {
    if (p.rows == 256) launch(Shape<8, 1>{});
    else launch(Shape<4, 2>{});
  } else {
    launch(Shape<4, 1>{});
  }
  const int st = dsp_launch_status();
  if (st != DSP_OK || p.whole) return st;
  const int64_t rows = std::min(int64_t(max_q_len) * G, int64_t(p.rows));
  auto merge = [&](auto split) {
    constexpr int kSplit = decltype(split)::value;
    constexpr int R = tree_merge_rows(D, kSplit);
    const int groups = int((rows + R - 1) / R);
    tree_merge_kernel<Tag, D, kSplit>
        <<<unsigned((int64_t(p.items) * groups + 7) / 8 * 8), 256, 0, s>>>(
            ws, ws_ml, ws_desc, cu_q, ctx_lens, p.items, groups, KVH, G, max_q_len, max_ctx,
            p.tiles_max, p.rows, out, ost, osh, vec_out);
  };
  // an item's pieces shared by four threads where there are many: 32 pieces 28.9 us a call (33.9 by
  // one thread), 5 pieces 38.5 (34.1)
  if (p.workers > 16 * p.items) merge(std::integral_constant<int, 4>{});
  else merge(std::integral_constant<int, 1>{});
  return dsp_launch_status();
}

size_t generic_bytes(int32_t B, int32_t Hq, int32_t KVH, int32_t D, int32_t max_q_len,
                     int32_t max_ctx) {
  return dsp_detail::generic_workspace_bytes(
      B, Hq, D, max_q_len, max_ctx,
      dsp_paged_mq_partition_tokens(B, Hq, KVH, D, max_q_len, max_ctx));
}

}  // namespace

extern "C" int dsp_tree_mask(const int32_t* parents, const int32_t* cu_q, int64_t num_rows,
                             int32_t B, int32_t max_q_len, int32_t mask_words, int32_t* mask,
                             dsp_stream_t stream) {
  DSP_HOST_CHECK(cu_q && mask, DSP_EINVAL);
  DSP_HOST_CHECK(B >= 0 && B <= 65535 && max_q_len >= 0 && num_rows >= 0 &&
                     int64_t(mask_words) * 32 >= max_q_len,
                 DSP_EINVAL);
  if (B == 0 || max_q_len == 0) return DSP_OK;
  const dim3 grid(unsigned((max_q_len + kMaskThreads - 1) / kMaskThreads), unsigned(B));
  tree_mask_kernel<<<grid, kMaskThreads, 0, static_cast<hipStream_t>(stream)>>>(
      parents, cu_q, num_rows, max_q_len, mask_words, reinterpret_cast<uint32_t*>(mask));
  return dsp_launch_status();
}

// (either launch's: which one a call takes goes by its strides too)
extern "C" size_t dsp_paged_tree_workspace_bytes(int32_t B, int32_t Hq, int32_t KVH, int32_t D,
                                                 int32_t max_q_len, int32_t max_ctx) {
  if (B <= 0 || KVH <= 0 || Hq <= 0 || Hq % KVH != 0 || max_q_len <= 0 || max_ctx <= 0) return 0;
  const size_t generic = generic_bytes(B, Hq, KVH, D, max_q_len, max_ctx);
  const TreePlan p = tree_plan(B, KVH, Hq / KVH, D, max_q_len, max_ctx);
  return p.tile ? std::max(generic, tree_tile_bytes(p, D)) : generic;
}

extern "C" int dsp_paged_tree_attention(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
    const void* v_cache, int64_t num_slots, int64_t kv_stride_slot, int64_t kv_stride_head,
    const int32_t* block_table, int64_t bt_stride, int32_t block_size, const int32_t* cu_q,
    const int32_t* ctx_lens, const int32_t* tree_mask, int32_t mask_words, int32_t B, int32_t Hq,
    int32_t KVH, int32_t D, float scale, int32_t max_q_len, int32_t max_ctx, void* workspace,
    size_t workspace_bytes, void* out, int64_t o_stride_t, int64_t o_stride_h, int32_t dtype,
    int32_t* err_count, dsp_stream_t stream) {
  DSP_HOST_CHECK(q && k_cache && v_cache && block_table && cu_q && ctx_lens && tree_mask && out,
                 DSP_EINVAL);
  DSP_HOST_CHECK(B >= 0 && B <= 65535 && Hq > 0 && KVH > 0 && KVH <= 65535 && Hq % KVH == 0 &&
                     max_q_len >= 0 && max_ctx >= 0 && num_slots >= 0 &&
                     int64_t(mask_words) * 32 >= max_q_len,
                 DSP_EINVAL);
  DSP_HOST_CHECK(dtype == DSP_BF16 || dtype == DSP_F16 || dtype == DSP_F32, DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(dsp_detail::generic_head_dim(D), DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(dsp_is_pow2(block_size) && bt_stride * block_size >= max_ctx, DSP_EINVAL);
  if (B == 0 || max_q_len == 0) return DSP_OK;
  const int64_t es = dtype == DSP_F32 ? 4 : 2;
  DSP_HOST_CHECK(dsp_aligned(q, es) && dsp_aligned(k_cache, es) && dsp_aligned(v_cache, es) &&
                     dsp_aligned(out, es),
                 DSP_EALIGN);
  const int G = Hq / KVH;
  const TreePlan p = tree_plan(B, KVH, G, D, max_q_len, max_ctx);
  const uint32_t* mask = reinterpret_cast<const uint32_t*>(tree_mask);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool tile = p.tile && dtype != DSP_F32 && block_size >= 16 && num_slots >= 16 &&
                    num_slots % block_size == 0 && num_slots / block_size < (int64_t(1) << 31) &&
                    kv_stride_slot >= 0 && kv_stride_slot < (int64_t(1) << 25) &&
                    kv_stride_slot * block_size < (int64_t(1) << 31) &&
                    scale > 0.f && scale < FLT_MAX && q_stride_t % 8 == 0 && q_stride_h % 8 == 0 &&
                    kv_stride_slot % 8 == 0 && kv_stride_head % 8 == 0 && dsp_aligned(q, 16) &&
                    dsp_aligned(k_cache, 16) && dsp_aligned(v_cache, 16);
  const size_t need = tile ? tree_tile_bytes(p, D)
                           : generic_bytes(B, Hq, KVH, D, max_q_len, max_ctx);
  DSP_HOST_CHECK(workspace_bytes >= need && (need == 0 || workspace != nullptr), DSP_EWORKSPACE);
  DSP_HOST_CHECK(need == 0 || dsp_aligned(workspace, 16), DSP_EALIGN);
  if (!tile)
    return dsp_detail::generic_attention(
        q, q_stride_t, q_stride_h, k_cache, v_cache, num_slots, kv_stride_slot, kv_stride_head,
        block_table, bt_stride, dsp_log2i(block_size), cu_q, ctx_lens, B, Hq, KVH, D, scale,
        max_q_len, max_ctx, dsp_paged_mq_partition_tokens(B, Hq, KVH, D, max_q_len, max_ctx),
        workspace, out, o_stride_t, o_stride_h, dtype, err_count, s, mask, mask_words);
  auto launch = [&](auto fn) {
    return fn(p, static_cast<const uint16_t*>(q), q_stride_t, q_stride_h,
              static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache),
              num_slots, kv_stride_slot, kv_stride_head, block_table, bt_stride,
              dsp_log2i(block_size), cu_q, ctx_lens, mask, mask_words, B, KVH, G, max_q_len,
              max_ctx, scale * 1.4426950408889634f, static_cast<float*>(workspace),
              static_cast<uint16_t*>(out), o_stride_t, o_stride_h, err_count, s);
  };
#define DSP_TREE(DD)                                                             \
  return dtype == DSP_F16 ? launch([](auto... a) { return launch_tree<F16Tag, DD>(a...); }) \
                          : launch([](auto... a) { return launch_tree<Bf16Tag, DD>(a...); })
  if (D == 64) DSP_TREE(64);
  if (D == 128) DSP_TREE(128);
  DSP_TREE(256);
#undef DSP_TREE
}
