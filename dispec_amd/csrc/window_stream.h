// Windowed attention of few rows a KV head (decode, verify): a kernel that streams the keys through
// registers.
//
// A wave holds kRG groups of 16 packed rows and takes 32-key chunks on its own, without a barrier: S^T =
// K Q^T on v_mfma_f32_16x16x32 with K rows straight from memory (the dims of an operand dealt so that
// a lane's elements are one load), V through a per-wave slab in LDS for the transposing reads.  The
// waves of a workgroup are `heads` neighbouring KV heads times key splits, chunk c of a piece going to
// split c % splits; the splits meet in LDS.
//
// kWhole: a workgroup takes a tile.  kRuns: the list of (sequence, head group, tile, chunk) units is cut
// into as many equal runs as the chip has CUs, computed on the device from the lengths; a tile's start
// counts as `start` chunks.  A tile that runs cut leaves a piece of each, which the second launch merges.
//
// Bound by HBM where there is much to read: 16 contexts of 32768 fp8 tokens (1.1 GB) 196 us, 5.8 TB/s, of
// which the merge is 4.7; 32 tokens under a window of 1024, 131 MB, 28 us; small calls by the chain of
// lengths, block ids and first keys, 4 us, and 1.6 us a chunk: 48 over up to 2048 fp4 tokens 17 us, 24
// verifies of 1 to 9 under a window of 512 14.  16-bit q: probabilities as in the tile kernel, one operand at
// 64 and 128 dims, three at 256 (32 tokens under a window of 2048, 8 KV heads of 256: 96 us, 95 with one).
// Slower: two chunks ahead in registers (37, 214 and 19 us for 29, 194 and 18), four waves a workgroup and
// three a SIMD (33, 204, 19).
#pragma once

#include "window_attn.h"

namespace dsp_window {
namespace {

enum Mode { kWhole, kRuns, kRunsOnce };  // (kRunsOnce: K and V by non-temporal loads)

template <typename Tag, int D, int kFmt, bool kF32, int kRG, int kMode>
__global__ __launch_bounds__(64 * stream_block(D)) __attribute__((
    amdgpu_waves_per_eu(stream_block(D) / 4))) void
window_stream_kernel(const WinArgs a) {
  constexpr int NW = stream_block(D), TR = 16 * kRG;
  constexpr int NKK = D / 32, NT = D / 16, ROWB = 2 * D, SLAB = kStreamChunk * ROWB;
  constexpr int kTerms = kF32 ? 3 : 1;                 // operands of q
  constexpr int kPTerms = kF32 ? 3 : prob_terms<D>();  // ... of a probability (as in the tile kernel)
  constexpr bool kF16 = std::is_same<Tag, F16Tag>::value;
  // K: of a key's row a lane takes the pieces grp + 4 i; V: 64 pieces at a time
  constexpr int kKB = kFmt == kNone ? D / 2 : dsp_quant::bytes<kFmt>(D / 4);  // bytes of a lane's dims
  constexpr int PB = kKB < 16 ? kKB : 16, NP = kKB / PB, PW = PB / 4;
  constexpr int PE = kFmt == kNone ? PB / 2 : kFmt == kFp8 ? PB : 2 * PB;     // elements of a piece
  constexpr int VE = kFmt == kNone ? 8 : kFmt == kFp8 ? 16 : 32;              // of a piece of V, 16 bytes
  constexpr int LR = D / VE, RL = 64 / LR, NV = kStreamChunk / RL;            // lanes a row, rows a load
  constexpr int SB = D / dsp_quant::kGroup;                                   // bytes of a row's scales
  static_assert(NP * (PE / 8) == NKK, "a lane's operands");
  // where the splits meet: [wave][row group][4 dims][row], 17 rows apart so that a row's dims, read side
  // by side, lie in different banks
  constexpr int kPitch = 17, kMeet = NT * 4 * kPitch;
  constexpr int kLds = NW * std::max(SLAB, kRG * kMeet * 16);
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  __shared__ float s_ml[NW][TR][2], s_sum[NW][TR][2];  // of waves; of heads

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, grp = lane >> 4;

  // ---- this workgroup's (sequence, group of KV heads, tile), placed as in the tile kernel, or its run
  const int splits = NW / a.heads, hw = wave % a.heads, split = wave / a.heads;
  const int groups = a.KVH / a.heads;
  auto zero_rows_of = [&](const Seq& sq, int group, int from, int upto) {
    const int kvh = group * a.heads + hw;
    for (int i = split * 64 + lane; i < (upto - from) * D; i += 64 * splits) {
      const int r = from + i / D;
      const int64_t o = int64_t(sq.q0 + r / a.G) * a.ost + int64_t(kvh * a.G + r % a.G) * a.osh + i % D;
      if constexpr (kF32) static_cast<float*>(a.out)[o] = 0.f;
      else static_cast<uint16_t*>(a.out)[o] = 0;
    }
  };
  int b = 0, group = 0, tile = 0;
  Seq sq;
  // (runs) sequences first .. first + 63, one a lane: their units of one head group
  int first = 0, units = 0, incl = 0;
  int begun = 0;                 // units before (b, group, tile)
  int seq_units = 0;             // of (b, group)
  int total = 0, W = 1, w = 0, left = 1, x = 0, share = 0, extra = 0;
  auto look = [&](int f) {
    first = f;
    const int i = min(f + lane, a.B - 1);
    const int ctx = a.ctx_lens[i], q0 = a.cu_q ? a.cu_q[i] : i, q1 = a.cu_q ? a.cu_q[i + 1] : i + 1;
    const int n = q1 - q0, bad = n > 0 && (ctx < n || ctx > a.max_ctx);
    const int queries = f + lane >= a.B || bad ? 0 : min(n, a.max_q_len), rows = queries * a.G;
    units = 0;
    for (int t = 0; t < a.tiles; ++t)
      if (t * TR < rows) {
        const int pl = rows <= (t + 1) * TR ? queries - 1 : ((t + 1) * TR - 1) * a.inv_g >> 16;
        units += a.start + span_of<kStreamChunk>(ctx - n + (t * TR * a.inv_g >> 16), ctx - n + pl, a.window,
                                               a.sinks).n;
      }
    incl = wave_incl_scan(units);
  };
  auto begin_of = [&](int v) { return v * share + v * extra / W; };
  // the positions of a tile's first and last query
  auto first_pos = [&](int t) { return sq.ctx - sq.n + (t * TR * a.inv_g >> 16); };
  auto last_pos = [&](int t) {
    return sq.ctx - sq.n + (sq.rows <= (t + 1) * TR ? sq.queries - 1 : ((t + 1) * TR - 1) * a.inv_g >> 16);
  };
  auto tile_units = [&](int t) {
    return a.start + span_of<kStreamChunk>(first_pos(t), last_pos(t), a.window, a.sinks).n;
  };
  // unit u -> (b, group, tile, x); u < total * groups
  auto locate = [&](int u) {
    for (int f = 0, before = 0; f < a.B; f += 64) {
      if (f != first || a.B > 64) look(f);
      const uint64_t hit = __ballot(groups * (before + incl) > u);
      if (hit) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
        b = f + l;
        seq_units = __builtin_amdgcn_readlane(units, l);
        begun = groups * (before + __builtin_amdgcn_readlane(incl, l) - seq_units);
        break;
      }
      before += __builtin_amdgcn_readlane(incl, 63);
    }
    sq = sequence(a, b);
    group = __builtin_amdgcn_readfirstlane((u - begun) / seq_units);
    begun += group * seq_units;
    x = u - begun;
    for (tile = 0; tile + 1 < a.tiles && x >= tile_units(tile); ++tile) {
      begun += tile_units(tile);
      x -= tile_units(tile);
    }
  };
  if constexpr (kMode == kWhole) {
    const int pairs = a.B * groups;
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
    const int item = pairs >= 8 ? at / a.tiles * 8 + xcd : 0;
    const int flat = xcd * ((pairs * a.tiles + 7) / 8) + at;
    const int pair = pairs >= 8 ? item : flat / a.tiles;
    tile = pairs >= 8 ? at % a.tiles : flat % a.tiles;
    if (pair >= pairs) return;
    b = pair / groups;
    group = pair % groups;
    sq = sequence(a, b);
    if (tile * TR >= sq.rows) return;
    if (sq.bad) {
      if (tile == 0 && group == 0 && threadIdx.x == 0 && a.err && (a.cu_q || sq.ctx != 0))
        atomicAdd(a.err, 1);
      zero_rows_of(sq, group, tile * TR, min(sq.rows, (tile + 1) * TR));
      return;
    }
  } else {
    for (int f = 0; f < a.B; f += 64) {
      look(f);
      total += __builtin_amdgcn_readlane(incl, 63);
      // bad lengths (rare): counted once, the rows written as zeros, one sequence a workgroup
      const int i = min(f + lane, a.B - 1);
      const int ctx = a.ctx_lens[i], n = a.cu_q ? a.cu_q[i + 1] - a.cu_q[i] : 1;
      uint64_t bad = __ballot(f + lane < a.B && n > 0 && (ctx < n || ctx > a.max_ctx));
      for (; bad; bad &= bad - 1) {
        const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(bad)) - 1);
        if ((f + l) % int(gridDim.x) != int(blockIdx.x)) continue;
        const Seq s = sequence(a, f + l);
        if (threadIdx.x == 0 && a.err && (a.cu_q || s.ctx != 0)) atomicAdd(a.err, 1);
        for (int g = 0; g < groups; ++g) zero_rows_of(s, g, 0, s.rows);
      }
    }
    const int C = total * groups;
    W = min(C / a.least + (C % a.least != 0), a.runs);
    const int lin = blockIdx.x;
    if (lin >= W) {
      if (threadIdx.x == 0) a.desc[kDesc * lin] = 0;
      return;
    }
    // workgroup lin runs on XCD lin % 8: each XCD takes a contiguous part of the list
    const int q8 = W / 8, r8 = W % 8, xcd = lin % 8, at = lin / 8;
    w = xcd < r8 ? xcd * (q8 + 1) + at : r8 * (q8 + 1) + (xcd - r8) * q8 + at;
    share = C / W;
    extra = C - share * W;
    // run v begins at unit floor(v C / W), or at the tile's first where that is one of its start
    int end = C;
    if (w + 1 < W) {
      end = begin_of(w + 1);
      locate(end);
      if (x <= a.start) end -= x;
    }
    left = end - begin_of(w);
    locate(begin_of(w));
    if (x <= a.start) {
      left += x;
      x = 0;
    }
  }
  int32_t d_np = 0, d_q0 = 0, d_rows = 0, d_row = 0, d_head = 0;
  bool any_bad = false;
  while (left > 0) {
    // ---- a piece: chunks c0 .. c1 of a tile
    const int kvh = group * a.heads + hw, t0 = tile * TR;
    const int base = sq.ctx - sq.n, pf = first_pos(tile), pl = last_pos(tile);
    const Span span = span_of<kStreamChunk>(pf, pl, a.window, a.sinks);
    int c0 = 0, c1 = span.n, took = 1;
    if constexpr (kMode != kWhole) {
      took = min(a.start + span.n - x, left);
      c0 = x == 0 ? 0 : x - a.start;
      c1 = x + took - a.start;
    }
    const bool whole = c0 == 0 && c1 == span.n;
    auto key_of = [&](int c) {
      return kStreamChunk * (c + ((span.first - span.sink) & ~((c - span.sink) >> 31)));
    };

    // ---- rows: lane n holds row t0 + 16 g + n of each group g (or the sequence's first, for nothing)
    bool row_ok[kRG];
    int tok[kRG], head[kRG], pos[kRG];
    dsp_u32x4 qop[kRG][kTerms][NKK];
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
      const int r = t0 + 16 * g + n;
      row_ok[g] = r < sq.rows;
      const int qi = row_ok[g] ? r * a.inv_g >> 16 : 0;
      tok[g] = sq.q0 + qi;
      head[g] = kvh * a.G + (row_ok[g] ? r - qi * a.G : 0);
      pos[g] = base + qi;
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int o = 0; o < PE / 8; ++o) {
          const int kk = i * (PE / 8) + o;
          const int64_t e = int64_t(tok[g]) * a.qst + int64_t(head[g]) * a.qsh + PE * (grp + 4 * i) + 8 * o;
          if constexpr (kF32) {
            const float* p = static_cast<const float*>(a.q) + e;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x0 = p[2 * j], x1 = p[2 * j + 1];
#pragma unroll
              for (int k = 0; k < 3; ++k) {
                const uint32_t w = k < 2 ? (__float_as_uint(x0) >> 16) | (__float_as_uint(x1) & 0xffff0000u)
                                         : narrow2<Tag>(x0, x1);
                qop[g][k][kk][j] = w;
                x0 -= dsp_bf16lo(w);
                x1 -= dsp_bf16hi(w);
              }
            }
          } else {
            qop[g][0][kk] = *reinterpret_cast<const dsp_u32x4*>(static_cast<const uint16_t*>(a.q) + e);
          }
        }
    }

    // ---- a chunk's rows: two halves of 16 keys, each in one block.  As in the tile kernel a half none of
    // whose keys is seen, and rows past the last key, repeat the last key.
    const int bmask = (1 << a.log2_bs) - 1;
    const int32_t* const bt_row = a.bt + int64_t(b) * a.bt_stride;
    auto first_key = [&](int t, int h) {
      const int k = t + 16 * h;
      // (sign bits: all ones where the half is seen)
      const int seen = ((k - span.hi) & ((span.lo - k - 16) | (k - a.sinks))) >> 31;
      return (k & seen) | ((span.hi - 1) & ~seen);
    };
    struct Raw {
      uint32_t k[2][NP][PW], v[NV][4], scale_k[2][SB > 4 ? 2 : 1], scale_v[NV];
      uint32_t bad;    // halves whose block id is bad
      int32_t ids[2];  // block ids of the chunk that comes next
    };
    Raw raw;
    auto load_ids = [&](int c) {
      const int t = key_of(min(c, c1 - 1));
#pragma unroll
      for (int h = 0; h < 2; ++h) raw.ids[h] = scalar_load(bt_row + (first_key(t, h) >> a.log2_bs));
    };
    auto fetch = [](auto* p) {
      if constexpr (kMode == kRunsOnce) return __builtin_nontemporal_load(p);
      else return *p;
    };
    auto load = [&](int c) {
      const int t = key_of(c);
      int64_t slot[2];
      int room[2];
      raw.bad = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = first_key(t, h);
        const uint32_t id = uint32_t(raw.ids[h]);
        // (of a bad id slot 0 alone is read)
        const uint32_t good = id < a.num_blocks ? ~0u : 0u;
        raw.bad |= (good & 1 ^ 1) << h;
        slot[h] = (int64_t(id & good) << a.log2_bs) + (k & bmask & good);
        room[h] = min(span.hi - 1 - k, 15) & good;
      }
      any_bad |= raw.bad != 0;
      load_ids(c + splits);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char* const rows = a.kc + slot[h] * a.slot_bytes + kvh * a.head_bytes;
        const uint32_t row = uint32_t(min(n, room[h]));
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const char* p = rows + (row * uint32_t(a.slot_bytes) + uint32_t(PB * (grp + 4 * i)));
          if constexpr (PW == 4) {
            const dsp_u32x4 w = fetch(reinterpret_cast<const dsp_u32x4*>(p));
#pragma unroll
            for (int j = 0; j < 4; ++j) raw.k[h][i][j] = w[j];
          } else {
            const dsp_u32x2 w = fetch(reinterpret_cast<const dsp_u32x2*>(p));
            raw.k[h][i][0] = w[0];
            raw.k[h][i][1] = w[1];
          }
        }
        if constexpr (kFmt != kNone) {
          const uint8_t* p = a.ks + slot[h] * a.scale_slot + kvh * a.scale_head +
                             row * uint32_t(a.scale_slot);
          if constexpr (SB == 2) {
            raw.scale_k[h][0] = *reinterpret_cast<const uint16_t*>(p);
          } else if constexpr (SB == 4) {
            raw.scale_k[h][0] = *reinterpret_cast<const uint32_t*>(p);
          } else {
            const dsp_u32x2 w = *reinterpret_cast<const dsp_u32x2*>(p);
            raw.scale_k[h][0] = w[0];
            raw.scale_k[h][1] = w[1];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int r = j * RL + lane / LR;
        const int h = RL > 16 ? r >> 4 : j * RL / 16;
        const int64_t s = RL > 16 ? (h ? slot[1] : slot[0]) : slot[h];
        const uint32_t row = uint32_t(min(r & 15, RL > 16 ? (h ? room[1] : room[0]) : room[h]));
        const uint32_t el = uint32_t(lane % LR * VE);
        const char* p = a.vc + s * a.slot_bytes + kvh * a.head_bytes +
                        (row * uint32_t(a.slot_bytes) + (kFmt == kFp8 ? el : kFmt == kFp4 ? el / 2 : 2 * el));
        const dsp_u32x4 w = fetch(reinterpret_cast<const dsp_u32x4*>(p));
#pragma unroll
        for (int i = 0; i < 4; ++i) raw.v[j][i] = w[i];
        if constexpr (kFmt != kNone)
          raw.scale_v[j] = a.vs[s * a.scale_slot + kvh * a.scale_head +
                            (row * uint32_t(a.scale_slot) + el / dsp_quant::kGroup)];
      }
    };


    // ---- the slab: 16-byte piece p of row r lies at p ^ vx(r), so that the 8 rows x 32 bytes of half a
    // transposing read fall on all banks
    char* const slab = lds + wave * SLAB;
    auto vx = [](int r) { return D >= 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); };
    auto store_v = [&] {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int r = j * RL + lane / LR, p0 = lane % LR * (VE / 8);
        uint32_t w[VE / 2];
        if constexpr (kFmt == kNone) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = raw.v[j][i];
        } else {
          dsp_quant::widen<kFmt, kF16, VE>(raw.v[j], dsp_quant::scale_of(raw.scale_v[j]), w);
        }
#pragma unroll
        for (int i = 0; i < VE / 8; ++i)
          *reinterpret_cast<dsp_u32x4*>(slab + r * ROWB + 16 * ((p0 + i) ^ vx(r))) =
              dsp_u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      }
    };
    // V^T operand of 16-dim tile nt: dim 16 nt + n, keys 4 grp + {0..3} and 16 + 4 grp + {0..3}
    auto read_v = [&](int nt) {
      v4i16 vh[2];
#pragma unroll
      for (int inst = 0; inst < 2; ++inst) {
        const int r = 16 * inst + 4 * grp + (n >> 2);
        vh[inst] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(
            slab + r * ROWB + 16 * ((2 * nt + ((n >> 1) & 1)) ^ vx(r)) + 8 * (n & 1)));
      }
      return __builtin_bit_cast(dsp_u32x4, vh);
    };

    float m[kRG], lpart[kRG];
    f32x4 acc[kRG][NT];
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
      m[g] = -INFINITY;
      lpart[g] = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[g][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr float kLag = lag<Tag, kPTerms>(), kRef = kF16 ? 15.f - kLag : 0.f;  // (as in the tile kernel)
    constexpr uint32_t kLeast = kF16 ? 0x00010001u : 0x00800080u;
    constexpr float kLeastP = kF16 ? 0x1p-24f : 0x1p-126f;
    // which keys of half h of the chunk at key t row group g's row sees (bit j: key t + 16 h + 4 grp + j)
    auto window_bits = [&](int g, int t, int h) {
      const int k = t + 16 * h + 4 * grp;
      return low_bits(pos[g] - k + 1) & (~low_bits(pos[g] - a.window - k + 1) | low_bits(a.sinks - k));
    };

    int c = c0 + split;
    if (c < c1) {
      load_ids(c);
      load(c);
    }
    for (; c < c1; c += splits) {
      const int t = key_of(c);
      const uint32_t bad_now = raw.bad;
      const bool edge = !(t + kStreamChunk - 1 <= pf &&
                          (t > pl - a.window || t + kStreamChunk <= a.sinks));
      wave_lds_fence();  // the slab's reads are done
      store_v();
      if (bad_now) {  // (rare)
        wave_lds_fence();
        zero_rows<D / 8, SLAB / 1024>(slab, (bad_now & 1u ? 0u : 0xffffu) | (bad_now & 2u ? 0u : 0xffff0000u));
      }
      // scores: sc[g][h][j] is key t + 16 h + 4 grp + j of row n
      f32x4 sc[kRG][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int g = 0; g < kRG; ++g) sc[g][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          uint32_t w[PE / 2];
          if constexpr (kFmt == kNone) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = raw.k[h][i][j];
          } else {
            const uint32_t byte = uint32_t(PE * (grp + 4 * i)) / dsp_quant::kGroup;
            const uint32_t word = SB > 4 ? (byte & 4 ? raw.scale_k[h][SB > 4 ? 1 : 0] : raw.scale_k[h][0])
                                         : raw.scale_k[h][0];
            dsp_quant::widen<kFmt, kF16, PE>(
                raw.k[h][i], dsp_quant::scale_of((word >> (8 * (byte & 3))) & 255u), w);
          }
#pragma unroll
          for (int o = 0; o < PE / 8; ++o) {
            const dsp_u32x4 k = dsp_u32x4{w[4 * o], w[4 * o + 1], w[4 * o + 2], w[4 * o + 3]};
#pragma unroll
            for (int g = 0; g < kRG; ++g)
#pragma unroll
              for (int x = kTerms - 1; x >= 0; --x)
                sc[g][h] = mfma32<Tag>(k, qop[g][x][i * (PE / 8) + o], sc[g][h]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (c + splits < c1) load(c + splits);
      __builtin_amdgcn_sched_barrier(0);
      if (edge) {
#pragma unroll
        for (int g = 0; g < kRG; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t seen = window_bits(g, t, h);
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[g][h][j] = (seen >> j) & 1u ? sc[g][h][j] : -INFINITY;
          }
      }
      if (bad_now) {
#pragma unroll
        for (int g = 0; g < kRG; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if ((bad_now >> h) & 1u) sc[g][h] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      }
      wave_lds_fence();  // V is in the slab
      if (edge) {
        if (any_nonfinite<Tag, SLAB / 1024>(slab)) {
          // (rare) infinities and NaN of V to the rows that see their keys; then they are cleared
#pragma unroll 1
          for (int nt = 0; nt < NT; ++nt) {
            const dsp_u32x4 v = read_v(nt);
#pragma unroll
            for (int g = 0; g < kRG; ++g) {
              dsp_u32x4 huge;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t two = window_bits(g, t, i >> 1) >> (2 * (i & 1));
                huge[i] = (two & 1u ? kHuge : 0u) | (two & 2u ? kHuge << 16 : 0u);
              }
              f32x4 add = f32x4{0.f, 0.f, 0.f, 0.f};
              add = mfma32<Bf16Tag>(odd_operand<Tag>(v, false), huge, add);
              add = mfma32<Bf16Tag>(odd_operand<Tag>(v, true), huge, add);
#pragma unroll
              for (int x = 0; x < NT; ++x)
                if (x == nt) acc[g][x] += add;
            }
          }
          wave_lds_fence();
          clear_nonfinite<Tag, SLAB / 1024>(slab);
          wave_lds_fence();
        }
      }
      dsp_u32x4 pop[kRG][kPTerms];
#pragma unroll
      for (int g = 0; g < kRG; ++g) {
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) top = fmaxf(top, sc[g][h][j]);
        top = fmaxf(top, dsp_shfl_xor(top, 16));
        top = fmaxf(top, dsp_shfl_xor(top, 32));
        const bool moves = fmaf(top, a.scale_log2, -m[g]) > kRef + kLag;  // (-inf, -inf: no)
        if (__builtin_amdgcn_ballot_w64(moves)) {
          float m_new = moves ? fmaf(top, a.scale_log2, -kRef) : m[g];
          if (moves && fmaf(top, a.scale_log2, -m_new) > 15.f)
            m_new = __uint_as_float(__float_as_uint(m_new) + (m_new > 0.f ? 1 : -1));
          const float alpha = moves ? fmaxf(dsp_exp2(m[g] - m_new), 0x1p-126f) : 1.f;
          m[g] = m_new;
          lpart[g] *= alpha;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[g][nt] *= alpha;
        }
        const float neg_m = m[g] == -INFINITY ? 0.f : -m[g];
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = dsp_exp2(fmaf(sc[g][i >> 2][i & 3], a.scale_log2, neg_m));
          lpart[g] += p[i];
        }
        if constexpr (kPTerms == 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            pop[g][0][i] = not_below(narrow2<Tag>(p[2 * i], p[2 * i + 1]), edge || bad_now ? 0u : kLeast);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] = fmaxf(p[i], edge || bad_now ? 0.f : kLeastP);
          pack8<Tag, kPTerms>(p, pop[g]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const dsp_u32x4 v = read_v(nt);
#pragma unroll
        for (int g = 0; g < kRG; ++g)
#pragma unroll
          for (int x = kPTerms - 1; x >= 0; --x) acc[g][nt] = mfma32<Tag>(v, pop[g][x], acc[g][nt]);
      }
    }
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
      lpart[g] += dsp_shfl_xor(lpart[g], 16);
      lpart[g] += dsp_shfl_xor(lpart[g], 32);
    }

    // ---- the splits meet in LDS: their maxima and sums, then their accumulators by the common maximum
#pragma unroll
    for (int g = 0; g < kRG; ++g)
      if (grp == 0) {
        s_ml[wave][16 * g + n][0] = m[g];
        s_ml[wave][16 * g + n][1] = lpart[g];
      }
    __syncthreads();  // (and every wave is done with the slabs)
    f32x4* const meet = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int g = 0; g < kRG; ++g) {
      float top = -INFINITY, sum = 0.f;
      for (int i = 0; i < splits; ++i) top = fmaxf(top, s_ml[i * a.heads + hw][16 * g + n][0]);
      const float to = top == -INFINITY ? 0.f : top;
      if (split == 0) {
        for (int i = 0; i < splits; ++i)
          sum = fmaf(s_ml[i * a.heads + hw][16 * g + n][1],
                     dsp_weight(s_ml[i * a.heads + hw][16 * g + n][0] - to), sum);
        if (grp == 0) {
          s_sum[hw][16 * g + n][0] = top;
          s_sum[hw][16 * g + n][1] = sum;
        }
      }
      const float weight = dsp_weight(m[g] - to);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        meet[(wave * kRG + g) * kMeet + (4 * nt + grp) * kPitch + n] = acc[g][nt] * weight;
    }
    __syncthreads();
    // ---- rows of the workgroup's heads, 4 dims a thread
    const int live = min(TR, sq.rows - t0);
    constexpr int kStep = 64 * NW / (D / 4);
    const int d = 4 * (threadIdx.x % (D / 4));
    for (int h = 0, lr = threadIdx.x / (D / 4);; lr += kStep) {
      while (lr >= live && h < a.heads) {
        lr -= live;
        ++h;
      }
      if (h >= a.heads) break;
      const f32x4* const at = meet + (lr >> 4) * kMeet + d / 4 * kPitch + (lr & 15);
      f32x4 v = at[h * kRG * kMeet];
      for (int k = 1; k < splits; ++k) v += at[(k * a.heads + h) * kRG * kMeet];
      const int r = t0 + lr, qi = r * a.inv_g >> 16;
      const float sum = s_sum[h][lr][1];
      if (whole) {
        v *= sum == 0.f ? 0.f : 1.f / sum;  // (0: no key counted; NaN stays)
        store4<Tag, kF32>(a, int64_t(sq.q0 + qi) * a.ost +
                                 int64_t((group * a.heads + h) * a.G + r - qi * a.G) * a.osh + d, v);
      } else {
        const int64_t row = (int64_t(2 * w + (c0 == 0 ? 1 : 0)) * a.heads + h) * TR + lr;
        *reinterpret_cast<f32x4*>(a.ws_acc + row * D + d) = v;
        if (d == 0) {
          a.ws_ml[2 * row] = s_sum[h][lr][0];
          a.ws_ml[2 * row + 1] = sum;
        }
      }
    }
    if constexpr (kMode == kWhole) break;
    if (c0 == 0 && !whole) {
      // this run began the tile: its merge.  Pieces: up to the last run that begins before the tile's end.
      const int upto = begun + took + span.n - c1;
      int v = min(W - 1, int(float(upto) * float(W) / float(total * groups)));
      while (begin_of(v) >= upto) --v;
      while (v + 1 < W && begin_of(v + 1) < upto) ++v;
      d_np = v - w + 1;
      d_q0 = sq.q0;
      d_rows = live;
      d_row = t0;
      d_head = group * a.heads;
    }
    left -= took;
    if (left <= 0) break;
    // the next tile (there is one)
    begun += a.start + span.n;
    x = 0;
    if ((++tile) * TR >= sq.rows) {
      tile = 0;
      if (++group == groups) {
        group = 0;
        do sq = sequence(a, ++b);
        while (sq.bad || sq.rows <= 0);
      }
    }
    __syncthreads();  // (the meeting place is free)
  }
  if (a.err && any_bad && lane == 0) atomicAdd(a.err, 1);  // once per wave
  if constexpr (kMode != kWhole)
    if (threadIdx.x == 0) {
      int32_t* d = a.desc + kDesc * w;
      d[0] = d_np;
      d[1] = d_q0;
      d[2] = d_rows;
      d[3] = d_row;
      d[4] = d_head;
    }
}

// The merge of the tiles that runs cut: workgroups (run that began a tile, some of its rows of all its
// heads), one thread per (row, 4 dims).  The first piece is the second of its run's two rows of tiles,
// those of the runs behind it their first.
template <typename Tag, int D, bool kF32, int TR>
__global__ __launch_bounds__(256) void window_runs_merge_kernel(const WinArgs a, int32_t blocks) {
  const int w = blockIdx.x / blocks, block = blockIdx.x % blocks;
  const int32_t* const d = a.desc + kDesc * w;
  const int np = scalar_load(d), q0 = scalar_load(d + 1), live = scalar_load(d + 2);
  const int first = scalar_load(d + 3), head = scalar_load(d + 4);
  if (np <= 0) return;
  const int i = (block * 256 + threadIdx.x) / (D / 4), h = i / live, lr = i - h * live;
  if (h >= a.heads) return;
  merge_row<Tag, D, kF32>(a, q0, (int64_t(2 * w + 1) * a.heads + h) * TR + lr,
                          (int64_t(2 * (w + 1)) * a.heads + h) * TR + lr, 2 * a.heads * TR, np,
                          first + lr, head + h, 4 * (threadIdx.x % (D / 4)));
}

template <typename Tag, int D, int kFmt, bool kF32, int kRG>
int launch_groups(const WinPlan& p, const WinArgs& a, hipStream_t s) {
  const int64_t pairs = int64_t(a.B) * a.KVH / p.heads;
  const unsigned whole =
      unsigned(pairs >= 8 ? (pairs + 7) / 8 * 8 * p.tiles : (pairs * p.tiles + 7) / 8 * 8);
  constexpr int kThreads = 64 * stream_block(D);
  if (!p.runs) {
    window_stream_kernel<Tag, D, kFmt, kF32, kRG, kWhole><<<whole, kThreads, 0, s>>>(a);
    return dsp_launch_status();
  }
  if (p.once)
    window_stream_kernel<Tag, D, kFmt, kF32, kRG, kRunsOnce><<<unsigned(p.runs), kThreads, 0, s>>>(a);
  else
    window_stream_kernel<Tag, D, kFmt, kF32, kRG, kRuns><<<unsigned(p.runs), kThreads, 0, s>>>(a);
  const int st = dsp_launch_status();
  if (st != DSP_OK) return st;
  const int64_t rows = std::min<int64_t>(int64_t(a.max_q_len) * a.G, p.rows) * p.heads;
  const int blocks = int((rows * (D / 4) + 255) / 256);
  window_runs_merge_kernel<Tag, D, kF32, 16 * kRG><<<unsigned(p.runs * blocks), 256, 0, s>>>(a, blocks);
  return dsp_launch_status();
}

template <typename Tag, int D, int kFmt, bool kF32>
int launch_stream(const WinPlan& p, const WinArgs& a, hipStream_t s) {
  // (wider or in fp32, two groups of rows do not fit the registers)
  if constexpr (D <= 128 && !kF32)
    if (p.rows == 32) return launch_groups<Tag, D, kFmt, kF32, 2>(p, a, s);
  return launch_groups<Tag, D, kFmt, kF32, 1>(p, a, s);
}

template <int D, int kFmt>
int stream_type(int32_t dtype, const WinPlan& p, const WinArgs& a, hipStream_t s) {
  if (dtype == DSP_F16) return launch_stream<F16Tag, D, kFmt, false>(p, a, s);
  if (dtype == DSP_BF16) return launch_stream<Bf16Tag, D, kFmt, false>(p, a, s);
  if constexpr (kFmt != kNone) return launch_stream<Bf16Tag, D, kFmt, true>(p, a, s);
  return DSP_EUNSUPPORTED;
}

template <int kFmt>
int stream_format(int32_t D, int32_t dtype, const WinPlan& p, const WinArgs& a, hipStream_t s) {
  if (D == 64) return stream_type<64, kFmt>(dtype, p, a, s);
  if (D == 128) return stream_type<128, kFmt>(dtype, p, a, s);
  return stream_type<256, kFmt>(dtype, p, a, s);
}

}  // namespace
}  // namespace dsp_window
