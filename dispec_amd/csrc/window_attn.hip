// Attention over the paged cache with a sliding window and sinks, and over quantised caches (the
// reference attends the whole context of a pool in the model's type:
// dispec/engine/model_runner.py:160-185).
//
//     o[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_ih . k_j),
//     j <= pos_i and (j > pos_i - window or j < sinks),   pos_i = ctx - q_len + i.
//
// Tile: NW waves of 32 packed rows each (row r: query r / G of head kvh G + r % G) share 64-key chunks
// of K and V in LDS; S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16 (dsp_tile32.h), P in registers.
// The chunks of a tile are those that hold a key that one of its rows sees: the sinks', then those of
// the window; of a block none of whose keys is seen neither id nor rows are read.  Two workgroups a CU at
// 64 and 128 dims: a chunk is loaded while the one before it is used, and one workgroup multiplies while
// another is at its barrier.  24 x 32 queries of 16 heads over 4 KV heads, 4000 tokens: under a window of
// 2048 29 us (64 dims), 39 (128), 101 (256); the whole context in fp8 42, 55, 180: bound by the chain of
// chunks that a workgroup has (a load, a barrier, products and exponentials one after the other).
#include "window_attn.h"

using namespace dsp_window;

namespace {

constexpr int NW = 4, TR = 32 * NW;  // waves and rows of a tile
constexpr int NB = 2;                // chunks in LDS

// kF32: q and out in fp32 over a quantised cache.  An element times its scale is exact in bf16, and
// q and the probabilities enter the products as three bf16 operands each, all 24 bits.
// 16-bit q: a probability is three operands (pack8), all 24 bits, where heads have 256 dims, as in all
// other attention of theirs (the two batches above 101 and 180 us, 77 and 135 with one operand); one,
// rounded once, at 64 and 128 dims, as in the multi-query tiles there: half the products.
template <typename Tag, int D, int kFmt, bool kF32>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(kF32 || D == 256 ? 1 : 2)))
void window_tile_kernel(const WinArgs a) {
  constexpr int NKS = D / 16, NDT = D / 32;   // 16-dim steps of K Q^T, 32-dim tiles of V^T P^T
  constexpr int CPR = D / 8, ROWB = 2 * D;    // 16-byte pieces and bytes of a row in LDS
  constexpr int SLAB = kChunk * ROWB;
  constexpr int RPW = kChunk / NW;            // rows a wave loads of a chunk, in one block
  constexpr int LPW = SLAB / 1024 / NW;       // KiB a wave loads of a slab
  constexpr int RPI = 1024 / ROWB;            // rows per LDS DMA
  constexpr int kTerms = kF32 ? 3 : 1;                        // operands of q
  constexpr int kPTerms = kF32 ? 3 : prob_terms<D>();         // ... of a probability
  // fp32 of 256 dims: q alone is 192 registers, and operands that the compiler reads ahead push more of
  // them into memory (24 x 32 rows of 4 KV heads over 4000 fp8 tokens: 398 us, 792 with them)
  constexpr bool kCrowded = kF32 && D == 256;
  static_assert(RPW <= 16 && LPW >= 1 && LPW * RPI == RPW, "a wave's rows lie in one block");
  static_assert(!kF32 || (kFmt != kNone && std::is_same<Tag, Bf16Tag>::value), "exact in bf16");
  __shared__ __attribute__((aligned(1024))) char lds[NB][2][SLAB];
  __shared__ int32_t s_bad[NB][NW];           // a wave's rows of a stage have a bad block id
  __shared__ int32_t s_odd[2][NW];            // ... hold infinities or NaN in V

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, col = lane & 31;

  // ---- this workgroup's (sequence, KV head, tile, part).  Workgroup i runs on XCD i % 8: all tiles
  // and parts of a (sequence, KV head) go to one XCD, whose L2 they share, where there are 8 such
  // pairs or more; the longest tiles come first.
  const int pairs = a.B * a.KVH, per = a.tiles * a.parts;
  const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3;
  int pair, inner;
  if (pairs >= 8) {
    pair = (at / per) * 8 + xcd;
    inner = at % per;
  } else {
    const int item = xcd * ((pairs * per + 7) / 8) + at;
    pair = item / per;
    inner = item % per;
  }
  if (pair >= pairs) return;
  const int b = pair / a.KVH, kvh = pair % a.KVH;
  const int tile = a.tiles - 1 - inner / a.parts, part = inner % a.parts;
  const Seq sq = sequence(a, b);
  const int t0 = tile * TR;
  if (t0 >= sq.rows) return;
  if (sq.bad) {
    if (part != 0) return;
    if (tile == 0 && kvh == 0 && threadIdx.x == 0 && a.err && (a.cu_q || sq.ctx != 0))
      atomicAdd(a.err, 1);
    for (int i = threadIdx.x; i < min(TR, sq.rows - t0) * D; i += 64 * NW) {
      const int r = t0 + i / D;
      const int64_t o = int64_t(sq.q0 + r / a.G) * a.ost + int64_t(kvh * a.G + r % a.G) * a.osh + i % D;
      if constexpr (kF32) static_cast<float*>(a.out)[o] = 0.f;
      else static_cast<uint16_t*>(a.out)[o] = 0;
    }
    return;
  }
  const int base = sq.ctx - sq.n;
  const int tile_pf = base + t0 / a.G, tile_pl = base + (min(sq.rows, t0 + TR) - 1) / a.G;
  const Span span = span_of<kChunk>(tile_pf, tile_pl, a.window, a.sinks);
  const int c0 = part * a.part_chunks, c1 = min(span.n, c0 + a.part_chunks);
  if (c0 >= c1) return;
  const int nc = c1 - c0;
  const bool whole = c0 == 0 && c1 == span.n;
  auto key_of = [&](int c) {  // the first key of the piece's chunk c
    const int x = c0 + c;
    return kChunk * (x < span.sink ? x : x - span.sink + span.first);
  };

  // ---- this wave's rows
  const int r0 = t0 + 32 * wave;
  const bool has_rows = r0 < sq.rows;
  const int pf = base + r0 / a.G, pl = base + (min(sq.rows, r0 + 32) - 1) / a.G;
  const int r = r0 + col;
  const bool row_ok = r < sq.rows;
  const int qi = row_ok ? r / a.G : 0, tok = sq.q0 + qi;
  const int head = kvh * a.G + (row_ok ? r - qi * a.G : 0);
  const int pos = base + qi;
  dsp_u32x4 qop[kTerms][NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int64_t e = int64_t(tok) * a.qst + int64_t(head) * a.qsh + 16 * ks + 8 * hl;
    if constexpr (kF32) {
      // the leading 8 bits, the next 8, the rest: exact
      const float* p = static_cast<const float*>(a.q) + e;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x0 = row_ok ? p[2 * i] : 0.f, x1 = row_ok ? p[2 * i + 1] : 0.f;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const uint32_t w = k < 2 ? (__float_as_uint(x0) >> 16) | (__float_as_uint(x1) & 0xffff0000u)
                                   : narrow2<Tag>(x0, x1);
          qop[k][ks][i] = w;
          x0 -= dsp_bf16lo(w);
          x1 -= dsp_bf16hi(w);
        }
      }
    } else {
      qop[0][ks] = row_ok ? *reinterpret_cast<const dsp_u32x4*>(
                                static_cast<const uint16_t*>(a.q) + e)
                          : dsp_u32x4{0u, 0u, 0u, 0u};
    }
  }

  // ---- stages.  This wave loads rows RPW * wave .. of every chunk; they lie in one block.
  auto kswz = [](int row) { return row & (CPR - 1); };
  auto vswz = [](int row) { return D >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); };
  const int bmask = (1 << a.log2_bs) - 1;
  const int32_t* const bt_row = a.bt + int64_t(b) * a.bt_stride;
  bool any_bad = false;
  // The rows of a chunk at key t: the first key read, how many follow it (a key that no row of the
  // tile sees may have no block any more: the rows of such a block repeat the tile's last key, and
  // those past the last key repeat it).
  auto first_key = [&](int t) {
    const int k = t + RPW * wave;
    const bool seen = k < span.hi && (k + RPW > span.lo || k < a.sinks);
    return seen ? k : span.hi - 1;
  };
  auto load_id = [&](int c) { return scalar_load(bt_row + (first_key(key_of(min(c, nc - 1))) >> a.log2_bs)); };
  const uint32_t lds_base = uint32_t(reinterpret_cast<uintptr_t>((lds_void_t*)&lds[0][0][0]));
  int32_t id_next = load_id(0);
  // where chunk c's rows of this wave begin in kc and vc (bytes, of the slot)
  struct Rows { int64_t slot; int room; bool bad; };
  auto rows_of = [&](int c) {
    const int k = first_key(key_of(c));
    const uint32_t id = uint32_t(id_next);
    Rows w;
    w.bad = id >= a.num_blocks;
    any_bad |= w.bad;
    w.slot = w.bad ? 0 : (int64_t(id) << a.log2_bs) + (k & bmask);
    w.room = w.bad ? 0 : min(span.hi - 1 - k, RPW - 1);
    id_next = load_id(c + 1);
    return w;
  };
  // 16-bit caches: the LDS DMA
  uint32_t koff[LPW], voff[LPW];
  if constexpr (kFmt == kNone) {
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
      const int rw = j * RPI + lane / CPR, row = RPW * wave + rw, sl = lane % CPR;
      koff[j] = uint32_t(rw) * uint32_t(a.slot_bytes) + 16 * (sl ^ kswz(row));
      voff[j] = uint32_t(rw) * uint32_t(a.slot_bytes) + 16 * (sl ^ vswz(row));
    }
  }
  auto send = [&](int c) {
    const int buf = c % NB;
    const Rows w = rows_of(c);
    if (lane == 0) s_bad[buf][wave] = w.bad;
    const char* const kb = a.kc + w.slot * a.slot_bytes + kvh * a.head_bytes;
    const char* const vb = a.vc + w.slot * a.slot_bytes + kvh * a.head_bytes;
    const uint32_t m0 = lds_base + uint32_t(2 * buf * SLAB + wave * LPW * 1024);
    if (w.room < RPW - 1) {
#pragma unroll
      for (int j = 0; j < LPW; ++j) {
        const int rw = j * RPI + lane / CPR, row = RPW * wave + rw, sl = lane % CPR;
        const uint32_t ro = uint32_t(min(rw, w.room)) * uint32_t(a.slot_bytes);
        dma16<false>(kb, ro + 16 * (sl ^ kswz(row)), m0 + j * 1024);
        dma16<false>(vb, ro + 16 * (sl ^ vswz(row)), m0 + SLAB + j * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < LPW; ++j) {
        dma16<false>(kb, koff[j], m0 + j * 1024);
        dma16<false>(vb, voff[j], m0 + SLAB + j * 1024);
      }
    }
  };
  // Quantised caches: through registers, widened on the way to LDS.  A lane takes EL elements of a row
  // at a time, NLD times; they share a scale.
  constexpr int kPerLane = RPW * D / 64, EL = kPerLane < 16 ? kPerLane : 16, NLD = kPerLane / EL;
  constexpr int EPR = D / EL, RPL = 64 / EPR;  // lanes a row, rows a load
  constexpr int WL = (kFmt == kFp8 ? EL : EL / 2) / 4;  // words a load
  constexpr int kRaw = kFmt == kNone ? 1 : NLD, kWords = kFmt == kNone ? 1 : WL;
  uint32_t raw[2][kRaw][kWords], raw_scale[2][kRaw];
  bool raw_bad = false;
  auto load_raw = [&](int c) {
    const Rows w = rows_of(c);
    raw_bad = w.bad;
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int rw = j * RPL + lane / EPR, el = lane % EPR * EL;
      const int64_t slot = w.slot + min(rw, w.room);
      const int64_t at = slot * a.slot_bytes + kvh * a.head_bytes + dsp_quant::bytes<kFmt>(el);
      const int64_t sat = slot * a.scale_slot + kvh * a.scale_head + el / dsp_quant::kGroup;
      typedef uint32_t words_t __attribute__((ext_vector_type(WL < 2 ? 2 : WL)));
      if constexpr (WL == 1) {
        raw[0][j][0] = *reinterpret_cast<const uint32_t*>(a.kc + at);
        raw[1][j][0] = *reinterpret_cast<const uint32_t*>(a.vc + at);
      } else {
        const words_t k = *reinterpret_cast<const words_t*>(a.kc + at);
        const words_t v = *reinterpret_cast<const words_t*>(a.vc + at);
#pragma unroll
        for (int i = 0; i < WL; ++i) {
          raw[0][j][i] = k[i];
          raw[1][j][i] = v[i];
        }
      }
      raw_scale[0][j] = a.ks[sat];
      raw_scale[1][j] = a.vs[sat];
    }
  };
  auto store_raw = [&](int c) {
    const int buf = c % NB;
    if (lane == 0) s_bad[buf][wave] = raw_bad;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < NLD; ++j) {
        const int rw = j * RPL + lane / EPR, row = RPW * wave + rw, sl = lane % EPR * EL / 8;
        uint32_t w[EL / 2];
        dsp_quant::widen<kFmt, std::is_same<Tag, F16Tag>::value, EL>(
            raw[p][j], dsp_quant::scale_of(raw_scale[p][j]), w);
#pragma unroll
        for (int i = 0; i < EL / 8; ++i)
          *reinterpret_cast<dsp_u32x4*>(&lds[buf][p][row * ROWB +
                                                     16 * ((sl + i) ^ (p ? vswz(row) : kswz(row)))]) =
              dsp_u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      }
  };

  // ---- operands from LDS (the layouts of the tree kernel's: K rows of 16-byte pieces XORed by kswz;
  // V^T by load_vt)
  auto read_k = [&](int buf, int x, int ks) {
    const int row = 32 * x + col;
    return *reinterpret_cast<const dsp_u32x4*>(
        &lds[buf][0][row * ROWB + 16 * ((2 * ks + hl) ^ kswz(row))]);
  };
  auto read_v = [&](int buf, int ps, int dt) { return load_vt<D>(&lds[buf][1][0], ps, dt); };

  float m = -INFINITY, lpart = 0.f;
  f32x16 acc[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[dt][j] = 0.f;
  // What m holds is the running maximum (base 2) less kRef: fp16 probabilities go up to 2^15 and end
  // at 2^-31 of a row's largest (three operands: 2^-36).  It moves when a score exceeds it by kLag more.
  constexpr bool kF16 = std::is_same<Tag, F16Tag>::value;
  constexpr float kLag = lag<Tag, kPTerms>(), kRef = kF16 ? 15.f - kLag : 0.f;
  // In a chunk that every row sees whole a probability is kept above 0, so that an infinity in V
  // meets a positive factor (three operands: pack8 keeps those of what is not below kLeastP).
  constexpr uint32_t kLeast = kF16 ? 0x00010001u : 0x00800080u;
  constexpr float kLeastP = kF16 ? 0x1p-24f : 0x1p-126f;

  // which keys of half x of the chunk at key t this lane's row sees (bit i: key t + 32 x + 4 hl + i)
  auto window_bits = [&](int t, int x) {
    const int k = t + 32 * x + 4 * hl;
    return low_bits(pos - k + 1) & (~low_bits(pos - a.window - k + 1) | low_bits(a.sinks - k));
  };
  // whether rows at positions f .. l see all keys of the chunk at key t
  auto sees_all = [&](int t, int f, int l) {
    return t + kChunk - 1 <= f && (t > l - a.window || t + kChunk <= a.sinks);
  };

  if constexpr (kFmt == kNone) {
    for (int c = 0; c < min(nc, NB - 1); ++c) send(c);
  } else {
    load_raw(0);
    store_raw(0);
    if (nc > 1) load_raw(1);
  }
  for (int c = 0; c < nc; ++c) {
    const int buf = c % NB, t = key_of(c);
    if constexpr (kFmt == kNone) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<0>());
    }
    const bool tile_edge = !sees_all(t, tile_pf, tile_pl);
    char* const my_v = &lds[buf][1][wave * LPW * 1024];  // the V rows this wave loaded
    if (tile_edge) {  // (uniform)
      __builtin_amdgcn_sched_barrier(0);
      const bool odd = any_nonfinite<Tag, LPW>(my_v);
      if (lane == 0) s_odd[c & 1][wave] = odd;
    }
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    uint32_t bad = 0, odd = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      bad |= uint32_t(s_bad[buf][w] != 0) << w;
      if (tile_edge) odd |= uint32_t(s_odd[c & 1][w] != 0);
    }
    bad = __builtin_amdgcn_readfirstlane(bad);
    odd = __builtin_amdgcn_readfirstlane(odd);
    if constexpr (kFmt == kNone) {
      if (c + NB - 1 < nc) send(c + NB - 1);
    } else {
      if (c + 1 < nc) store_raw(c + 1);
      if (c + 2 < nc) load_raw(c + 2);
    }
    if (bad) {
      // (rare) keys of bad block ids count for nothing: their rows hold slot 0's
      if ((bad >> wave) & 1u) zero_rows<CPR, LPW>(my_v, 0);
      __syncthreads();
    }
    if (odd) {
      // (rare) infinities and NaN of V to the rows that see their keys; then they are cleared
      if (has_rows)
#pragma unroll 1
        for (int ps = 0; ps < 4; ++ps) {
          const uint32_t seen = window_bits(t, ps >> 1) >> (16 * (ps & 1));
          dsp_u32x4 huge;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t two = seen >> (8 * (i >> 1) + 2 * (i & 1));
            huge[i] = (two & 1u ? kHuge : 0u) | (two & 2u ? kHuge << 16 : 0u);
          }
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            __builtin_amdgcn_sched_barrier(0);
            const dsp_u32x4 v = read_v(buf, ps, dt);
            acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, false), huge, acc[dt]);
            acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, true), huge, acc[dt]);
          }
        }
      __syncthreads();
      clear_nonfinite<Tag, LPW>(my_v);
      __syncthreads();
    }
    if (!has_rows) continue;
    // ---- scores S^T (keys x rows): sc[x][j] is key t + 32 x + 8 (j / 4) + 4 hl + j % 4 of row col
    f32x16 sc[2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[x][j] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if constexpr (kCrowded) __builtin_amdgcn_sched_barrier(0);
        const dsp_u32x4 k = read_k(buf, x, ks);
#pragma unroll
        for (int i = kTerms - 1; i >= 0; --i) sc[x] = mfma32x32<Tag>(k, qop[i][ks], sc[x]);
      }
    const bool edge = !sees_all(t, pf, pl);
    if (edge) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t seen = window_bits(t, x);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          sc[x][j] = (seen >> (8 * (j >> 2) + (j & 3))) & 1u ? sc[x][j] : -INFINITY;
      }
    }
    if (bad) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j4 = 0; j4 < 4; ++j4)
          if ((bad >> ((32 * x + 8 * j4) / RPW)) & 1u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[x][4 * j4 + j] = -INFINITY;
          }
    }
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, sc[x][j]);
    top = fmaxf(top, dsp_shfl_xor(top, 32));
    const bool moves = fmaf(top, a.scale_log2, -m) > kRef + kLag;  // (-inf, -inf: no)
    if (__builtin_amdgcn_ballot_w64(moves)) {
      float m_new = moves ? fmaf(top, a.scale_log2, -kRef) : m;
      if (moves && fmaf(top, a.scale_log2, -m_new) > 15.f)  // (steps of 16 and more: the next one up)
        m_new = __uint_as_float(__float_as_uint(m_new) + (m_new > 0.f ? 1 : -1));
      const float alpha = moves ? fmaxf(dsp_exp2(m - m_new), 0x1p-126f) : 1.f;
      m = m_new;
      lpart *= alpha;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) acc[dt] *= alpha;
    }
    const float neg_m = m == -INFINITY ? 0.f : -m;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float p = dsp_exp2(fmaf(sc[x][j], a.scale_log2, neg_m));
        lpart += p;
        sc[x][j] = p;
      }
    // ---- O^T += V^T P^T, 16 keys a step: step ps takes registers 8 (ps % 2) .. of half ps / 2
#pragma unroll
    for (int ps = 0; ps < 4; ++ps) {
      dsp_u32x4 pop[kPTerms];
      if constexpr (kPTerms == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pop[0][i] = not_below(narrow2<Tag>(sc[ps >> 1][8 * (ps & 1) + 2 * i],
                                             sc[ps >> 1][8 * (ps & 1) + 2 * i + 1]),
                                edge || bad ? 0u : kLeast);
      } else {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          p[i] = fmaxf(sc[ps >> 1][8 * (ps & 1) + i], edge || bad ? 0.f : kLeastP);
        pack8<Tag, kPTerms>(p, pop);
      }
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        if constexpr (kCrowded) __builtin_amdgcn_sched_barrier(0);
        const dsp_u32x4 v = read_v(buf, ps, dt);
#pragma unroll
        for (int i = kPTerms - 1; i >= 0; --i) acc[dt] = mfma32x32<Tag>(v, pop[i], acc[dt]);
      }
    }
  }
  if (a.err && any_bad && lane == 0) atomicAdd(a.err, 1);  // once per wave
  if (!has_rows) return;
  // ---- the piece's rows: acc[dt][j] = O[row col][dim 32 dt + 8 (j / 4) + 4 hl + j % 4]
  lpart += dsp_shfl_xor(lpart, 32);
  if (!row_ok) return;
  if (whole) {
    const float inv = lpart == 0.f ? 0.f : 1.f / lpart;  // (0: no key counted; NaN stays)
    const int64_t o = int64_t(tok) * a.ost + int64_t(head) * a.osh + 4 * hl;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int j4 = 0; j4 < 4; ++j4) {
        const f32x4 v = f32x4{acc[dt][4 * j4], acc[dt][4 * j4 + 1], acc[dt][4 * j4 + 2],
                              acc[dt][4 * j4 + 3]} * inv;
        const int64_t e = o + 32 * dt + 8 * j4;
        if constexpr (kF32) {
          float* p = static_cast<float*>(a.out) + e;
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = v[j];
        } else {
          uint16_t* p = static_cast<uint16_t*>(a.out) + e;
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
  } else {
    const int64_t row = ((int64_t(pair) * a.tiles + tile) * a.parts + part) * TR + 32 * wave + col;
    float* dst = a.ws_acc + row * D + 4 * hl;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int j4 = 0; j4 < 4; ++j4)
        *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * j4) =
            f32x4{acc[dt][4 * j4], acc[dt][4 * j4 + 1], acc[dt][4 * j4 + 2], acc[dt][4 * j4 + 3]};
    if (hl == 0) {
      a.ws_ml[2 * row] = m;
      a.ws_ml[2 * row + 1] = lpart;
    }
  }
}

// The merge of the tile kernel's tiles in several parts: one thread per (row, 4 dims).
template <int D>
constexpr int merge_rows() { return 1024 / D; }

template <typename Tag, int D, bool kF32>
__global__ __launch_bounds__(256) void window_merge_kernel(const WinArgs a, int32_t groups,
                                                           int32_t tile_rows) {
  constexpr int TPR = D / 4;
  const int item = blockIdx.x / groups, group = blockIdx.x % groups;
  const int pair = item / a.tiles, tile = item % a.tiles;
  const int b = pair / a.KVH, kvh = pair % a.KVH;
  const Seq sq = sequence(a, b);
  const int t0 = tile * tile_rows, lr = group * merge_rows<D>() + threadIdx.x / TPR;
  const int r = t0 + lr, d = 4 * (threadIdx.x % TPR);
  if (sq.bad || t0 >= sq.rows) return;
  const int base = sq.ctx - sq.n;
  const Span span = span_of<kChunk>(base + t0 / a.G, base + (min(sq.rows, t0 + tile_rows) - 1) / a.G,
                                    a.window, a.sinks);
  const int np = (span.n + a.part_chunks - 1) / a.part_chunks;
  if (np <= 1 || lr >= tile_rows || r >= sq.rows) return;
  const int64_t row = int64_t(item) * a.parts * tile_rows + lr;
  merge_row<Tag, D, kF32>(a, sq.q0, row, row + tile_rows, tile_rows, np, r, kvh, d);
}

// ---- which launch a shape takes
bool quantised(int32_t format) { return format == DSP_KV_FP8 || format == DSP_KV_FP4; }

WinPlan win_plan(int32_t B, int32_t KVH, int32_t G, int32_t D, int32_t max_q_len, int32_t max_ctx,
                 int32_t window, int32_t sinks, int32_t format, int32_t dtype, bool may_stream) {
  WinPlan p{};
  if (!(D == 64 || D == 128 || D == 256) || (dtype == DSP_F32 && !quantised(format))) return p;
  const int64_t rows = int64_t(max_q_len) * G;
  p.stream = may_stream && rows <= 64;
  // Tiles of 256 rows where a sequence has more than half of one and its registers suffice
  // (window_prefill.hip); of 128 they pass K and V through LDS twice as often.
  p.rows = p.stream ? (rows <= 16 || D > 128 || dtype == DSP_F32 ? 16 : 32)
                    : D > 128 || rows <= 128 || dtype == DSP_F32 ? 128 : 256;
  const int size = p.stream ? kStreamChunk : kChunk;
  const int64_t tiles = (rows + p.rows - 1) / p.rows;
  // chunks that a tile can have: its queries' windows side by side, anywhere in a chunk; the sinks'
  int64_t chunks = (int64_t(max_ctx) + size - 1) / size;
  if (window > 0) {
    const int64_t queries = std::min<int64_t>(max_q_len, p.rows / G + 2);
    chunks = std::min(chunks, (int64_t(window) + queries) / size + 2 + (int64_t(sinks) + size - 1) / size);
  }
  const int64_t cus = dsp_detail::device_cus(), all = int64_t(B) * KVH;
  int64_t workgroups;
  if (p.stream) {
    // In steps of 1.6 us, a wave's chunk of 128 dims for 16 rows: a round of whole tiles takes its start,
    // 2.5, and the chunks of a split; equal runs their start, the scan and the merge, 10, and the
    // chip's share.
    const int waves = stream_block(D), most = dsp_detail::balanced_head_group(KVH);
    const double step = (D > 128 ? 2.0 : D > 64 ? 1.0 : 0.7) * (p.rows > 16 ? 1.5 : 1.0);
    double best = 10.0 + step * double(tiles * all * chunks) / double(cus * waves);
    bool whole = false;
    p.heads = most;
    for (int h = 1; h <= std::min(most, waves); h *= 2) {
      const int64_t rounds = (tiles * (all / h) + cus - 1) / cus, splits = waves / h;
      const double cost = double(rounds) * (2.5 + step * double((chunks + splits - 1) / splits));
      if (cost < best) {
        best = cost;
        whole = true;
        p.heads = h;
      }
    }
    const int splits = waves / p.heads;
    p.start = splits;
    p.least = 2 * splits + p.start;
    const int64_t total = tiles * (all / p.heads), units = total * (chunks + p.start);
    p.runs = whole ? 0 : int(std::min(cus, (units + p.least - 1) / p.least));
    // 128 MiB of K and V, half of the last-level cache, behind which the next call finds little of its
    // own: 1.1 GB of fp8 195 us (204 by ordinary loads), 134 MB 29.6 (30.5); 102 MB 35 (30).
    const int64_t row = format == DSP_KV_FP8 ? D : format == DSP_KV_FP4 ? D / 2 : 2 * D;
    p.once = double(all) * double(chunks * size * 2 * row) >= double(128 << 20);
    workgroups = whole ? total + 8 * tiles : p.runs;
    p.tile = units < (int64_t(1) << 31) && rows < (int64_t(1) << 30);
  } else {
    const int64_t slots = cus * (p.rows == 128 && D <= 128 ? 2 : 1);
    const int64_t total = std::max<int64_t>(tiles * all, 1);
    int64_t parts = total >= slots ? 1 : slots / total;
    parts = std::max<int64_t>(1, std::min(parts, chunks / 2));
    p.part_chunks = int((chunks + parts - 1) / parts);
    p.parts = int((chunks + p.part_chunks - 1) / p.part_chunks);
    workgroups = (all + 8) * tiles * p.parts;
    p.tile = rows < (int64_t(1) << 30);
  }
  p.tiles = int(tiles);
  p.tile = p.tile && workgroups < (int64_t(1) << 31);  // (32 bits number the workgroups)
  if (p.stream && !p.tile)
    return win_plan(B, KVH, G, D, max_q_len, max_ctx, window, sinks, format, dtype, false);
  return p;
}

size_t win_bytes(const WinPlan& p, int64_t pairs, int32_t D) {
  if (!p.tile) return 0;
  if (p.stream)
    return size_t(p.runs) * (size_t(2) * p.heads * p.rows * (D + 2) + kDesc) * sizeof(float);
  return p.parts <= 1 ? 0 : size_t(pairs) * p.tiles * p.parts * p.rows * (size_t(D) + 2) * sizeof(float);
}

template <typename Tag, int D, int kFmt, bool kF32>
int launch_window(const WinPlan& p, const WinArgs& a, hipStream_t s) {
  const int64_t pairs = int64_t(a.B) * a.KVH, per = int64_t(p.tiles) * p.parts;
  const unsigned grid = unsigned(pairs >= 8 ? (pairs + 7) / 8 * 8 * per : (pairs * per + 7) / 8 * 8);
  int st;
  if (p.rows == 256) {
    st = wide_tiles(D, kFmt, std::is_same<Tag, F16Tag>::value, grid, a, s);
  } else {
    window_tile_kernel<Tag, D, kFmt, kF32><<<grid, 64 * NW, 0, s>>>(a);
    st = dsp_launch_status();
  }
  if (st != DSP_OK || p.parts <= 1) return st;
  const int64_t most = std::min<int64_t>(int64_t(a.max_q_len) * a.G, p.rows);
  const int groups = int((most + merge_rows<D>() - 1) / merge_rows<D>());
  window_merge_kernel<Tag, D, kF32><<<unsigned(pairs * p.tiles * groups), 256, 0, s>>>(a, groups, p.rows);
  return dsp_launch_status();
}

template <int D, int kFmt>
int launch_type(int32_t dtype, const WinPlan& p, const WinArgs& a, hipStream_t s) {
  if (dtype == DSP_F16) return launch_window<F16Tag, D, kFmt, false>(p, a, s);
  if (dtype == DSP_BF16) return launch_window<Bf16Tag, D, kFmt, false>(p, a, s);
  if constexpr (kFmt != kNone) return launch_window<Bf16Tag, D, kFmt, true>(p, a, s);
  return DSP_EUNSUPPORTED;
}

template <int D>
int launch_format(int32_t format, int32_t dtype, const WinPlan& p, const WinArgs& a,
                  hipStream_t s) {
  if (format == DSP_KV_FP8) return launch_type<D, kFp8>(dtype, p, a, s);
  if (format == DSP_KV_FP4) return launch_type<D, kFp4>(dtype, p, a, s);
  return launch_type<D, kNone>(dtype, p, a, s);
}

// The general kernel's partition, of the keys that a sequence's queries see.
int32_t general_span(int32_t max_q_len, int32_t max_ctx, int32_t window, int32_t sinks) {
  return int32_t(dsp_detail::generic_window_keys(max_q_len, max_ctx, window, sinks));
}
int32_t general_partition(int32_t B, int32_t Hq, int32_t KVH, int32_t D, int32_t max_q_len,
                          int32_t max_ctx, int32_t window, int32_t sinks) {
  return dsp_paged_mq_partition_tokens(B, Hq, KVH, D, max_q_len,
                                       general_span(max_q_len, max_ctx, window, sinks));
}

}  // namespace

extern "C" size_t dsp_paged_window_workspace_bytes(int32_t B, int32_t Hq, int32_t KVH, int32_t D,
                                                   int32_t max_q_len, int32_t max_ctx,
                                                   int32_t window, int32_t sinks, int32_t format,
                                                   int32_t dtype) {
  if (B <= 0 || KVH <= 0 || Hq <= 0 || Hq % KVH != 0 || max_q_len <= 0 || max_ctx < 0 ||
      window < 0 || sinks < 0)
    return 0;
  max_ctx = std::max(max_ctx, 1);  // (as the launch is planned)
  size_t tile = 0;
  for (bool stream : {false, true})
    tile = std::max(tile, win_bytes(win_plan(B, KVH, Hq / KVH, D, max_q_len, max_ctx, window, sinks,
                                             format, dtype, stream),
                                    int64_t(B) * KVH, D));
  if (quantised(format)) return tile;
  // (any launch's: which one a call takes goes by its strides too)
  return std::max(tile, dsp_detail::generic_workspace_bytes(
                            B, Hq, D, max_q_len, general_span(max_q_len, max_ctx, window, sinks),
                            general_partition(B, Hq, KVH, D, max_q_len, max_ctx, window, sinks)));
}

extern "C" int dsp_paged_window_attention(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
    const void* v_cache, int64_t num_slots, int64_t kv_stride_slot_bytes,
    int64_t kv_stride_head_bytes, const uint8_t* k_scale, const uint8_t* v_scale,
    int64_t scale_stride_slot, int64_t scale_stride_head, int32_t format,
    const int32_t* block_table, int64_t bt_stride, int32_t block_size, const int32_t* cu_q,
    const int32_t* ctx_lens, int32_t B, int32_t Hq, int32_t KVH, int32_t D, float scale,
    int32_t window, int32_t sinks, int32_t max_q_len, int32_t max_ctx, void* workspace,
    size_t workspace_bytes, void* out, int64_t o_stride_t, int64_t o_stride_h, int32_t dtype,
    int32_t* err_count, dsp_stream_t stream) {
  DSP_HOST_CHECK(q && k_cache && v_cache && block_table && ctx_lens && out, DSP_EINVAL);
  DSP_HOST_CHECK(B >= 0 && B <= 65535 && Hq > 0 && KVH > 0 && KVH <= 65535 && Hq % KVH == 0 &&
                     max_q_len >= 0 && max_ctx >= 0 && max_ctx <= kWholeWindow && num_slots >= 0 &&
                     window >= 0 && sinks >= 0 && (window > 0 || sinks == 0) &&
                     (cu_q || max_q_len <= 1),
                 DSP_EINVAL);
  DSP_HOST_CHECK(dtype == DSP_BF16 || dtype == DSP_F16 || dtype == DSP_F32, DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(dsp_is_pow2(block_size) && bt_stride * block_size >= max_ctx, DSP_EINVAL);
  const bool quant = quantised(format);
  DSP_HOST_CHECK(quant || format == DSP_KV_PLAIN, DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(!quant || (k_scale && v_scale), DSP_EINVAL);
  if (B == 0 || max_q_len == 0) return DSP_OK;
  const int64_t es = dtype == DSP_F32 ? 4 : 2;
  DSP_HOST_CHECK(dsp_aligned(q, es) && dsp_aligned(out, es), DSP_EALIGN);
  const int G = Hq / KVH;
  const int32_t plan_ctx = std::max(max_ctx, 1);  // (no context at all: as for one token)
  // (a window that reaches past every context is none)
  const bool all = window == 0 || window >= max_ctx;
  const int32_t win = all ? kWholeWindow : window, sink = all ? 0 : std::min(sinks, max_ctx);
  DSP_HOST_CHECK(!quant || D == 64 || D == 128 || D == 256, DSP_EUNSUPPORTED);
  const int64_t scale_bytes = D / dsp_quant::kGroup;  // (of a quantised cache: of a head's scales)
  // (the kernels address the rows of a block in 32 bits, as those of codes)
  DSP_HOST_CHECK(!quant || (scale_stride_slot >= 0 && scale_stride_slot < (int64_t(1) << 26)),
                 DSP_EUNSUPPORTED);
  const bool scales_ok =
      !quant || (scale_stride_slot % scale_bytes == 0 && scale_stride_head % scale_bytes == 0 &&
                 dsp_aligned(k_scale, scale_bytes) && dsp_aligned(v_scale, scale_bytes));
  const bool rows16 = kv_stride_slot_bytes % 16 == 0 && kv_stride_head_bytes % 16 == 0 &&
                      dsp_aligned(k_cache, 16) && dsp_aligned(v_cache, 16);
  const WinPlan p = win_plan(B, KVH, G, D, max_q_len, plan_ctx, window, sinks, format, dtype,
                             rows16 && scales_ok);
  const int32_t row_align = quant ? (format == DSP_KV_FP8 ? 16 : 8) : 16;
  const int64_t q_align = dtype == DSP_F32 ? 1 : 8;
  const bool tile =
      p.tile && block_size >= 16 && num_slots >= block_size && num_slots % block_size == 0 &&
      num_slots / block_size < (int64_t(1) << 31) && kv_stride_slot_bytes >= 0 &&
      kv_stride_slot_bytes < (int64_t(1) << 26) && scale > 0.f && scale < FLT_MAX &&
      q_stride_t % q_align == 0 && q_stride_h % q_align == 0 &&
      kv_stride_slot_bytes % row_align == 0 && kv_stride_head_bytes % row_align == 0 &&
      dsp_aligned(q, dtype == DSP_F32 ? 4 : 16) && dsp_aligned(k_cache, row_align) &&
      dsp_aligned(v_cache, row_align);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!tile) {
    DSP_HOST_CHECK(!quant, DSP_EUNSUPPORTED);
    DSP_HOST_CHECK(dsp_detail::generic_head_dim(D), DSP_EUNSUPPORTED);
    DSP_HOST_CHECK(dsp_aligned(k_cache, es) && dsp_aligned(v_cache, es) &&
                       kv_stride_slot_bytes % es == 0 && kv_stride_head_bytes % es == 0,
                   DSP_EALIGN);
    const int32_t P = general_partition(B, Hq, KVH, D, max_q_len, plan_ctx, window, sinks);
    const size_t need = dsp_detail::generic_workspace_bytes(
        B, Hq, D, max_q_len, general_span(max_q_len, plan_ctx, window, sinks), P);
    DSP_HOST_CHECK(workspace_bytes >= need && (need == 0 || workspace != nullptr), DSP_EWORKSPACE);
    DSP_HOST_CHECK(need == 0 || dsp_aligned(workspace, 16), DSP_EALIGN);
    return dsp_detail::generic_window_attention(
        q, q_stride_t, q_stride_h, k_cache, v_cache, num_slots, kv_stride_slot_bytes / es,
        kv_stride_head_bytes / es, block_table, bt_stride, dsp_log2i(block_size), cu_q, ctx_lens, B,
        Hq, KVH, D, scale, win, sink, max_q_len, max_ctx,
        general_span(max_q_len, plan_ctx, window, sinks), P, workspace, out, o_stride_t, o_stride_h,
        dtype, err_count, s);
  }
  const size_t need = win_bytes(p, int64_t(B) * KVH, D);
  DSP_HOST_CHECK(workspace_bytes >= need && (need == 0 || workspace != nullptr), DSP_EWORKSPACE);
  DSP_HOST_CHECK(need == 0 || dsp_aligned(workspace, 16), DSP_EALIGN);
  float* ws = static_cast<float*>(workspace);
  const int64_t part_rows = p.stream ? int64_t(2) * p.runs * p.heads * p.rows
                                     : int64_t(B) * KVH * p.tiles * p.parts * p.rows;
  float* const ws_ml = ws + part_rows * D;
  const WinArgs a{q, q_stride_t, q_stride_h, static_cast<const char*>(k_cache),
                  static_cast<const char*>(v_cache), k_scale, v_scale,
                  uint32_t(num_slots / block_size), kv_stride_slot_bytes, kv_stride_head_bytes,
                  scale_stride_slot, scale_stride_head, block_table, bt_stride,
                  dsp_log2i(block_size), cu_q, ctx_lens, B, KVH, G, max_q_len, max_ctx, win, sink,
                  scale * 1.4426950408889634f, p.tiles, p.parts, p.part_chunks, p.heads, p.runs,
                  p.least, p.start, (65536 + G - 1) / G,
                  reinterpret_cast<int32_t*>(ws_ml + 2 * part_rows), ws, ws_ml, out, o_stride_t, o_stride_h,
                  o_stride_t % 4 == 0 && o_stride_h % 4 == 0 && dsp_aligned(out, 8), err_count};
  if (p.stream)
    return format == DSP_KV_FP8   ? stream_fp8(D, dtype, p, a, s)
           : format == DSP_KV_FP4 ? stream_fp4(D, dtype, p, a, s)
                                  : stream_plain(D, dtype, p, a, s);
  if (D == 64) return launch_format<64>(format, dtype, p, a, s);
  if (D == 128) return launch_format<128>(format, dtype, p, a, s);
  return launch_format<256>(format, dtype, p, a, s);
}
