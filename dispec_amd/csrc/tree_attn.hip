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
// share 64-key chunks of K and V that the LDS DMA brings in, double-buffered; S^T = K Q^T and O^T =
// V^T P^T on v_mfma_f32_32x32x16, with P in registers (dsp_tile32.h), a running maximum that moves
// when it is exceeded by 2^8, sums and accumulators in fp32.  The probabilities enter P V as one
// 16-bit operand (rounded to nearest; the sum takes the unrounded ones): half a step of the type,
// as much as the output's own rounding.
//  * 4 waves (128 rows) for up to 128 rows a KV head, 8 waves (256 rows, a chunk loaded once for
//    twice the rows) above.
//  * The list of (sequence, KV head, tile, chunk) units is cut into as many equal runs as there are
//    workgroups resident on the chip, computed on the device from the lengths.  A run's end within
//    kSnap chunks of a tile's end moves onto it.  A tile inside a run is written; a tile that runs
//    cut leaves its rows' maximum, sum and accumulator per piece, and the second launch merges them.
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
constexpr int kMinChunks = 2;  // a workgroup gets at least this many chunks
constexpr int kSnap = 2;
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

// One sequence: `tiles` of TR packed rows (its first max_q_len nodes'), each of `chunks` units (one
// unit a tile where the tiles stay whole).
struct TreeSeq {
  int q0, n, ctx, rows, tiles, chunks, units;
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
  s.units = whole ? s.tiles : s.tiles * s.chunks;
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

template <typename Tag, int D, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(
    D > 128 ? 1 : D > 64 ? 2 : NW > 4 ? 4 : 3))) void tree_tile_kernel(
    const uint16_t* __restrict__ q, int64_t qst, int64_t qsh, const uint16_t* __restrict__ kc,
    const uint16_t* __restrict__ vc, int64_t num_slots, int64_t kvs_slot, int64_t kvs_head,
    const int32_t* __restrict__ bt, int64_t bt_stride, int32_t log2_bs,
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ ctx_lens,
    const uint32_t* __restrict__ mask, int32_t words, int32_t B, int32_t KVH, int32_t G,
    int32_t max_q_len, int32_t max_ctx, float scale_log2, int32_t whole,
    float* __restrict__ ws_acc, float* __restrict__ ws_ml, int32_t* __restrict__ ws_desc,
    uint16_t* __restrict__ out, int64_t ost, int64_t osh, int32_t vec_out,
    int32_t* __restrict__ err_count) {
  constexpr int TR = 32 * NW;                    // packed rows per tile
  constexpr int NKS = D / 16, NDT = D / 32;      // 16-dim steps of K Q^T, 32-dim tiles of V^T P^T
  constexpr int CPR = D / 8, ROWB = 2 * D;       // 16-byte pieces and bytes of a K or V row
  constexpr int SLAB = kChunk * ROWB;            // a chunk of K (or V)
  constexpr int RPI = 1024 / ROWB;               // rows per 1-KiB DMA load
  constexpr int LPW = SLAB / 1024 / NW;          // loads per wave and slab
  constexpr int RPW = kChunk / NW;               // rows per wave: one block's
  static_assert(LPW >= 1 && LPW * RPI == RPW && RPW <= 16, "a wave's rows lie in one block");
  __shared__ __attribute__((aligned(1024))) char lds[2][2][SLAB];  // [buffer][K | V]
  __shared__ int32_t s_flag[2][NW];              // of each wave's rows: 1 bad block, 2 odd values

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
    // bad lengths: counted once, the rows written as zeros, one sequence per workgroup
    for (int b = lin; b < B; b += gridDim.x) {
      if (b < f || b >= f + 64) continue;
      const TreeSeq s = lane_seq(mine, b - f);
      if (!tree_bad(s.n, s.ctx, max_ctx)) continue;
      if (threadIdx.x == 0 && err_count) atomicAdd(err_count, 1);
      const int row = KVH * G * D, n = min(s.n, max_q_len);
      for (int i = 0; i < n; ++i)
        for (int e = threadIdx.x; e < row; e += 64 * NW)
          out[int64_t(s.q0 + i) * ost + int64_t(e / D) * osh + e % D] = 0;
    }
  }
  const int C = total * KVH;
  const int least = whole ? 1 : kMinChunks;
  const int W = min((C + least - 1) / least, int(gridDim.x));
  if (lin >= W) {
    if (!whole && threadIdx.x == 0) ws_desc[4 * lin + 3] = 0;
    return;
  }
  // workgroup lin runs on XCD lin % 8: each XCD takes a contiguous part of the list, so that the
  // tiles and pieces of one (sequence, KV head) share an L2
  const int q8 = W / 8, r8 = W % 8, xcd = lin % 8, pos = lin / 8;
  const int w = xcd < r8 ? xcd * (q8 + 1) + pos : r8 * (q8 + 1) + (xcd - r8) * q8 + pos;
  const int share = C / W, extra = C - share * W;
  int b = 0, kvh = 0, tile = 0, c0 = 0;  // where the run stands
  int base = 0;                          // units (of all KV heads) before sequence b
  TreeSeq sq;
  // unit u -> (b, kvh, tile, c0); u < C
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
    kvh = rest / sq.units;
    rest -= kvh * sq.units;
    if (whole) {
      tile = rest;
      c0 = 0;
    } else {
      tile = rest / sq.chunks;
      c0 = rest - tile * sq.chunks;
    }
  };
  // the tile after this one (there is one)
  auto next_tile = [&]() {
    c0 = 0;
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
  // Run w begins at unit floor(w C / W), moved onto a tile's end where that is within kSnap chunks
  // (in the same way by both its neighbours).
  auto begin_of = [&](int v) { return v * share + int(int64_t(v) * extra / W); };
  int end = C;
  if (w + 1 < W) {
    end = begin_of(w + 1);
    if (!whole) {
      locate(end);
      if (c0 <= kSnap) end -= c0;
      else if (sq.chunks - c0 <= kSnap) end += sq.chunks - c0;
    }
  }
  int u = begin_of(w);
  locate(u);
  int left;
  if (whole || c0 <= kSnap) {
    left = end - (u - c0);
    c0 = 0;
  } else if (sq.chunks - c0 <= kSnap) {
    left = end - (u + sq.chunks - c0);
    if (left > 0) next_tile();
  } else {
    left = end - u;
  }

  // ---- its pieces: chunks c0 .. c1 of a tile
  auto kswz = [](int row) { return row & (CPR - 1); };
  auto vswz = [](int row) { return D >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); };
  const int bmask = (1 << log2_bs) - 1;
  uint32_t koff[LPW], voff[LPW];
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    const int rw = j * RPI + lane / CPR, row = RPW * wave + rw, sl = lane % CPR;
    koff[j] = uint32_t(rw * kvs_slot * 2 + 16 * (sl ^ kswz(row)));
    voff[j] = uint32_t(rw * kvs_slot * 2 + 16 * (sl ^ vswz(row)));
  }
  const uint32_t lds_base = uint32_t(reinterpret_cast<uintptr_t>((lds_void_t*)&lds[0][0][0]));
  int32_t d_b = 0, d_kvh = 0, d_tile = 0, d_np = 0;
  bool any_bad = false;
  for (bool again = false; left > 0; again = true) {
    const int nch = sq.chunks, c1 = whole ? nch : min(nch, c0 + left);
    const int kbeg = c0 * kChunk, kfin = min(c1 * kChunk, sq.ctx), tree0 = sq.ctx - sq.n;
    const int r0 = tile * TR;
    const int64_t bt_row = int64_t(b) * bt_stride;
    auto load_blk = [&](int t0) {
      return bt[bt_row + (min(t0 + RPW * wave, kfin - 1) >> log2_bs)];
    };
    int32_t blk = load_blk(kbeg);
    const int32_t blk_second = load_blk(kbeg + kChunk);
    const int r = r0 + 32 * wave + col;
    const bool row_ok = r < sq.rows;
    const bool wave_has_rows = r0 + 32 * wave < sq.rows;
    const int qi = row_ok ? r / G : 0;
    const int h = kvh * G + (row_ok ? r - qi * G : 0);
    const uint32_t* const mrow = mask + int64_t(sq.q0 + qi) * words;
    dsp_u32x4 qop[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
      qop[ks] = row_ok ? *reinterpret_cast<const dsp_u32x4*>(q + int64_t(sq.q0 + qi) * qst +
                                                             int64_t(h) * qsh + 16 * ks + 8 * hl)
                       : dsp_u32x4{0u, 0u, 0u, 0u};
    float m = -INFINITY, lpart = 0.f;
    f32x16 acc[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[dt][j] = 0.f;
    const int64_t head_off = int64_t(kvh) * kvs_head;
    bool bad_rows = false;  // the rows this wave loaded last are those of a bad block id (uniform)
    // K and V of the chunk at t0 into buffer buf: this wave's RPW rows, those past kfin as the last
    // key's (a stale row may hold anything), of a bad block slots 0 ..
    auto issue = [&](int buf, int t0, int32_t blk_v) {
      const int32_t id = __builtin_amdgcn_readfirstlane(blk_v);
      const int from = min(t0 + RPW * wave, kfin - 1);
      int64_t slot0 = int64_t(id) * (bmask + 1) + (from & bmask);
      bad_rows = id < 0 || (int64_t(id) + 1) * (bmask + 1) > num_slots;
      if (bad_rows) {
        slot0 = 0;
        any_bad |= t0 + RPW * wave < kfin;
      }
      const int64_t e = slot0 * kvs_slot + head_off;
      const char* kb = reinterpret_cast<const char*>(kc + e);
      const char* vb = reinterpret_cast<const char*>(vc + e);
      const uint32_t m0 = lds_base + uint32_t(buf * 2 * SLAB + wave * LPW * 1024);
      if (t0 + kChunk > kfin) {
#pragma unroll
        for (int j = 0; j < LPW; ++j) {
          const int rw = j * RPI + lane / CPR, row = RPW * wave + rw, sl = lane % CPR;
          const uint32_t ro = uint32_t(min(rw, kfin - 1 - from) * kvs_slot * 2);
          dma16<false>(kb, ro + 16 * (sl ^ kswz(row)), m0 + j * 1024);
          dma16<false>(vb, ro + 16 * (sl ^ vswz(row)), m0 + SLAB + j * 1024);
        }
        return;
      }
#pragma unroll
      for (int j = 0; j < LPW; ++j) {
        dma16<false>(kb, koff[j], m0 + j * 1024);
        dma16<false>(vb, voff[j], m0 + SLAB + j * 1024);
      }
    };
    if (again) __syncthreads();  // every wave is done with the previous piece's buffers
    issue(0, kbeg, blk);
    blk = blk_second;
    const int nc = c1 - c0;
    for (int c = 0; c < nc; ++c) {
      const int t0 = kbeg + c * kChunk, buf = c & 1;
      // this wave's DMAs of chunk c (and the block ids of chunk c + 1) are in; after the barrier
      // every wave's are, and every wave is done with chunk c - 1, whose buffer the next overwrites
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<0>());
      char* const my_v = &lds[buf][1][wave * LPW * 1024];  // the V rows this wave loaded
      const bool edge = t0 + kChunk > tree0;               // (uniform) some row may not see all of it
      if (bad_rows) zero_rows<CPR, LPW>(my_v, 0);
      int flag = bad_rows ? 1 : 0;
      if (edge) {
        __builtin_amdgcn_sched_barrier(0);
        flag |= any_nonfinite<Tag, LPW>(my_v) ? 2 : 0;
      }
      s_flag[buf][wave] = flag;
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      int flags = 0;
#pragma unroll
      for (int x = 0; x < NW; ++x) flags |= s_flag[buf][x];
      flags = __builtin_amdgcn_readfirstlane(flags);
      const bool odd = (flags & 2) != 0;
      auto clear_odd = [&] {
        __syncthreads();  // every wave has taken the chunk's infinities and NaN
        clear_nonfinite<Tag, LPW>(my_v);
        __syncthreads();
      };
      if (c + 1 < nc) {
        issue(buf ^ 1, t0 + kChunk, blk);
        if (c + 2 < nc) blk = load_blk(t0 + 2 * kChunk);
      }
      if (!wave_has_rows) {  // it only loads
        if (odd) clear_odd();
        continue;
      }
      const char* ks_lds = &lds[buf][0][0];
      const char* vs_lds = &lds[buf][1][0];
      // ---- scores S^T (keys x rows): two 32-key halves.  sc[mt][j] is key 32*mt + 8*(j/4) + 4*hl
      // + j%4 of this lane's row.
      f32x16 sc[2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int j = 0; j < 16; ++j) sc[mt][j] = 0.f;
        const int krow = 32 * mt + col;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          const dsp_u32x4 kop = *reinterpret_cast<const dsp_u32x4*>(
              ks_lds + krow * ROWB + 16 * ((2 * ks + hl) ^ kswz(krow)));
          sc[mt] = mfma32x32<Tag>(kop, qop[ks], sc[mt]);
        }
      }
      // ---- which keys the row sees, in the chunks that hold nodes (bit i: key t0 + 32 mt + 4 hl + i)
      uint32_t seen[2] = {~0u, ~0u};
      if (edge) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          seen[mt] = dsp_tree_window(mrow, words, sq.n, t0 + 32 * mt - tree0) >> (4 * hl);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            sc[mt][j] = (seen[mt] >> (8 * (j >> 2) + (j & 3))) & 1u ? sc[mt][j] : -INFINITY;
        }
      }
      if (flags & 1) {
        // sc[mt][j] lies in the chunk's 16-key group 2*mt + j/8
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (__builtin_amdgcn_readfirstlane(s_flag[buf][g * (NW / 4)]) & 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) sc[g >> 1][8 * (g & 1) + j] = -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, sc[mt][j]);
      mx = fmaxf(mx, dsp_shfl_xor(mx, 32)) * scale_log2;  // base 2; -inf stays -inf
      // the maximum moves when some row's exceeds it by 8 (p <= 2^8): the sum and the accumulators
      // share it, so the result is the same
      if (__builtin_amdgcn_ballot_w64(mx > m + 8.f) != 0) {
        const float m_new = fmaxf(m, mx);
        const float alpha = m_new == -INFINITY ? 1.f : dsp_exp2(m - m_new);
        m = m_new;
        lpart *= alpha;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) acc[dt] *= alpha;
      }
      const float neg_m = m == -INFINITY ? 0.f : -m;
      // P^T operands of the four 16-key steps: step ps = 2*mt + half takes registers j = 8*half ..
      // 8*half + 7, i.e. keys 16*ps + 4*hl + {0..3, 8..11}
      dsp_u32x4 pop[4];
#pragma unroll
      for (int ps = 0; ps < 4; ++ps) {
        float p8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p8[i] = dsp_exp2(fmaf(sc[ps >> 1][8 * (ps & 1) + i], scale_log2, neg_m));
          lpart += p8[i];
        }
        pop[ps] = dsp_u32x4{pack2(narrow<Tag>(p8[0]), narrow<Tag>(p8[1])),
                            pack2(narrow<Tag>(p8[2]), narrow<Tag>(p8[3])),
                            pack2(narrow<Tag>(p8[4]), narrow<Tag>(p8[5])),
                            pack2(narrow<Tag>(p8[6]), narrow<Tag>(p8[7]))};
      }
      // (rare) infinities and NaN of V to the rows that see them
      if (odd) {
#pragma unroll 1
        for (int ps = 0; ps < 4; ++ps) {
          const uint32_t bits = (ps < 2 ? seen[0] : seen[1]) >> (16 * (ps & 1));
          dsp_u32x4 huge;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t two = bits >> (8 * (i >> 1) + 2 * (i & 1));
            huge[i] = (two & 1u ? kHuge : 0u) | (two & 2u ? kHuge << 16 : 0u);
          }
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            __builtin_amdgcn_sched_barrier(0);  // one tile's operands at a time: registers
            const dsp_u32x4 v = load_vt<D>(vs_lds, ps, dt);
            acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, false), huge, acc[dt]);
            acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, true), huge, acc[dt]);
          }
        }
        clear_odd();
      }
      // ---- O^T += V^T . P^T
#pragma unroll
      for (int ps = 0; ps < 4; ++ps)
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          v4i16 vh[2];
#pragma unroll
          for (int inst = 0; inst < 2; ++inst) {  // (load_vt written out: paged_prefill.hip)
            const int kr = 16 * ps + 8 * inst + 4 * hl + ((lane & 15) >> 2);
            const int dim0 = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            vh[inst] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(
                vs_lds + kr * ROWB + 16 * ((dim0 >> 3) ^ vswz(kr)) + 2 * (dim0 & 7)));
          }
          acc[dt] = mfma32x32<Tag>(__builtin_bit_cast(dsp_u32x4, vh), pop[ps], acc[dt]);
        }
    }
    // ---- the piece's rows: acc[dt][j] = O[row col][dim 32*dt + 8*(j/4) + 4*hl + j%4]
    lpart += dsp_shfl_xor(lpart, 32);
    if (c0 == 0 && c1 == nch) {
      const float inv = lpart == 0.f ? 0.f : 1.f / lpart;  // (0: the row sees no key; NaN stays)
      if (row_ok) {
        uint16_t* o = out + int64_t(sq.q0 + qi) * ost + int64_t(h) * osh;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int j4 = 0; j4 < 4; ++j4) {
            uint16_t x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = narrow<Tag>(acc[dt][4 * j4 + j] * inv);
            uint16_t* const at = o + 32 * dt + 8 * j4 + 4 * hl;
            if (vec_out) {
              *reinterpret_cast<dsp_u32x2*>(at) = dsp_u32x2{pack2(x[0], x[1]), pack2(x[2], x[3])};
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) at[j] = x[j];
            }
          }
      }
    } else {
      const int64_t wrow = int64_t(2 * w + (c0 == 0 ? 1 : 0)) * TR + 32 * wave + col;
      if (row_ok) {
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
      if (c0 == 0) {  // this run began the tile: its merge is described here
        const int tile_end = base + (kvh * sq.tiles + tile + 1) * nch;
        d_b = b;
        d_kvh = kvh;
        d_tile = tile;
        // up to the last run that begins before the tile's end (those within kSnap moved onto it)
        d_np = int32_t((int64_t(tile_end - kSnap) * W - 1) / C) - w + 1;
      }
    }
    left -= whole ? 1 : c1 - c0;
    if (left > 0) next_tile();
  }
  if (err_count && any_bad && lane == 0) atomicAdd(err_count, 1);  // once per wave
  if (!whole && threadIdx.x == 0) {
    int32_t* d = ws_desc + 4 * w;
    d[0] = d_b;
    d[1] = d_kvh;
    d[2] = d_tile;
    d[3] = d_np;
  }
}

// Grid (workgroups of the first launch, row groups): R rows of the tile that run x began and did
// not finish, one thread per (row, 4 dims); its pieces are loaded 16 at a time before they are
// folded.
constexpr int tree_merge_rows(int D) { return 1024 / D; }

template <typename Tag, int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(
    const float* __restrict__ ws_acc, const float* __restrict__ ws_ml,
    const int32_t* __restrict__ ws_desc, const int32_t* __restrict__ cu_q, int32_t G,
    int32_t max_q_len, int32_t tile_rows, uint16_t* __restrict__ out, int64_t ost, int64_t osh) {
  constexpr int TPR = D / 4, R = tree_merge_rows(D), kBatch = 16;
  const int64_t w = blockIdx.x;
  const int32_t* desc = ws_desc + 4 * w;
  const int b = desc[0], kvh = desc[1], tile = desc[2], np = desc[3];
  if (np <= 0) return;
  const int q0 = cu_q[b], rows = min(cu_q[b + 1] - q0, max_q_len) * G;
  const int lr = blockIdx.y * R + threadIdx.x / TPR, d = 4 * (threadIdx.x % TPR);
  const int r = tile * tile_rows + lr;
  if (lr >= tile_rows || r >= rows) return;
  float M = -INFINITY, L = 0.f;
  f32x4 A = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < np; p0 += kBatch) {
    const int n = min(np - p0, kBatch);
    f32x4 va[kBatch];
    float vm[kBatch], vl[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (i < n) {
        const int p = p0 + i;
        const int64_t row = (p == 0 ? 2 * w + 1 : 2 * (w + p)) * tile_rows + lr;
        va[i] = *reinterpret_cast<const f32x4*>(ws_acc + row * D + d);
        vm[i] = ws_ml[2 * row];
        vl[i] = ws_ml[2 * row + 1];
      }
    float bm = M;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) bm = i < n ? fmaxf(bm, vm[i]) : bm;
    const float Mu = bm == -INFINITY ? 0.f : bm;
    const float keep = dsp_exp2(M - Mu);
    L *= keep;
    A *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float x = i < n ? dsp_exp2(vm[i] - Mu) : 0.f;
      L = fmaf(i < n ? vl[i] : 0.f, x, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) A[e] = fmaf(i < n ? va[i][e] : 0.f, x, A[e]);
    }
    M = bm;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint16_t* o = out + int64_t(q0 + r / G) * ost + int64_t(kvh * G + r % G) * osh + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = narrow<Tag>(A[e] * inv);
}

// ---- which launch a shape takes
struct TreePlan {
  bool tile;       // the tile kernel (else generic)
  bool whole;      // its tiles stay whole: no second launch
  int waves;       // of a workgroup
  int workers;     // workgroups
};

bool tree_tile_shape(int32_t D) { return D == 64 || D == 128 || D == 256; }

int tree_waves(int32_t D, int64_t rows) { return rows > 128 && D <= 128 ? 8 : 4; }

TreePlan tree_plan(int32_t B, int32_t KVH, int32_t G, int32_t D, int32_t max_q_len,
                   int32_t max_ctx) {
  TreePlan p{};
  if (!tree_tile_shape(D) || B < 1 || max_q_len < 1 || max_ctx < 1) return p;
  const int64_t rows = int64_t(max_q_len) * G;
  p.waves = tree_waves(D, rows);
  const int64_t tiles = (rows + 32 * p.waves - 1) / (32 * p.waves) * B * KVH;
  const int64_t chunks = (int64_t(max_ctx) + kChunk - 1) / kChunk;
  p.tile = rows < (int64_t(1) << 30) && tiles * chunks < (int64_t(1) << 31) &&
           max_ctx < (1 << 30);
  p.whole = chunks <= 8;
  // workgroups that fit the chip at once (LDS and registers)
  const int per_cu = D > 128 ? 1 : D > 64 ? (p.waves > 4 ? 1 : 2) : (p.waves > 4 ? 2 : 3);
  const int64_t slots = int64_t(per_cu) * dsp_detail::device_cus();
  p.workers = int(p.whole ? std::min(tiles, slots)
                          : std::min((tiles * chunks + kMinChunks - 1) / kMinChunks, slots));
  return p;
}

size_t tree_tile_bytes(const TreePlan& p, int32_t D) {
  return p.whole ? 0 : size_t(p.workers) * (size_t(2) * 32 * p.waves * (D + 2) + 4) * sizeof(float);
}

template <typename Tag, int D>
int launch_tree(const TreePlan& p, const uint16_t* q, int64_t qst, int64_t qsh, const uint16_t* kc,
                const uint16_t* vc, int64_t num_slots, int64_t kvs_slot, int64_t kvs_head,
                const int32_t* bt, int64_t bt_stride, int32_t log2_bs, const int32_t* cu_q,
                const int32_t* ctx_lens, const uint32_t* mask, int32_t words, int32_t B,
                int32_t KVH, int32_t G, int32_t max_q_len, int32_t max_ctx, float scale_log2,
                float* ws, uint16_t* out, int64_t ost, int64_t osh, int32_t* err_count,
                hipStream_t s) {
  const int tr = 32 * p.waves;
  float* ws_ml = ws + int64_t(2) * p.workers * tr * D;
  int32_t* ws_desc = reinterpret_cast<int32_t*>(ws_ml + int64_t(4) * p.workers * tr);
  const int vec_out = ost % 4 == 0 && osh % 4 == 0 && dsp_aligned(out, 8);
  auto launch = [&](auto kernel) {
    kernel<<<p.workers, 64 * p.waves, 0, s>>>(
        q, qst, qsh, kc, vc, num_slots, kvs_slot, kvs_head, bt, bt_stride, log2_bs, cu_q, ctx_lens,
        mask, words, B, KVH, G, max_q_len, max_ctx, scale_log2, p.whole, ws, ws_ml, ws_desc, out,
        ost, osh, vec_out, err_count);
  };
  if constexpr (D <= 128) {
    if (p.waves == 8) launch(tree_tile_kernel<Tag, D, 8>);
    else launch(tree_tile_kernel<Tag, D, 4>);
  } else {
    launch(tree_tile_kernel<Tag, D, 4>);
  }
  const int st = dsp_launch_status();
  if (st != DSP_OK || p.whole) return st;
  const int64_t rows = std::min(int64_t(max_q_len) * G, int64_t(tr));
  const dim3 grid(unsigned(p.workers), unsigned((rows + tree_merge_rows(D) - 1) / tree_merge_rows(D)));
  tree_merge_kernel<Tag, D><<<grid, 256, 0, s>>>(ws, ws_ml, ws_desc, cu_q, G, max_q_len, tr, out,
                                                 ost, osh);
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
                    num_slots % block_size == 0 && kv_stride_slot < (int64_t(1) << 25) &&
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
