// Windowed attention of many rows a KV head (prompt chunks): tiles of 256 rows whose two groups of waves
// take turns at the matrix cores.
//
// Eight waves of 32 packed rows share 64-key chunks of K and V in LDS, as on the tile kernel of
// window_attn.hip.  There both waves of a SIMD wait for the chunk's barrier and then multiply and take
// exponentials at the same time, and the matrix cores idle while they do the latter.  Here a chunk has two
// phases with a barrier behind each -- products: S = K Q^T of the next chunk, O += V^T P^T of this one;
// vector work: mask, maximum, exponentials of the next -- and waves 4 to 7, the second wave of each SIMD,
// run one phase behind waves 0 to 3: one group's products beside the other's vector work.
//
// Stage c is V of chunk c and K of chunk c + 1, what a product phase needs; four stages lie in LDS, sent
// for two to three chunks ahead.  A stage's rows are waited for by the wave that loaded them, before the
// barrier that ends the last phase before its use.
//
// Four prompts' chunks of 2048 tokens over 8192, 32 query heads over 8 of 128 dims, a window of 4096
// (5.5e11 operations): 645 us a call in a tight loop, 738 by the tile kernel on the same card; 545 to 575,
// 1010 to 957 TFLOP/s, among other work (8192^3 products through the library: 1064 and 1152 on two cards).
// Four chunks of 512 over 3247 to 4608 fp8 tokens: 190 us, over 3766 each, as many keys, 148: a workgroup
// takes one tile, and the longest context decides; over bf16 154 and 133, so that widening is a tenth.
// A probability is one 16-bit operand, rounded once (at these head dims the multi-query tiles hold it so;
// a second one is half as many products again): 2.3e-3 from 64 bits in bf16, 1.7e-3 of it the output's own
// rounding.  In the tight loop a chunk takes 4300 cycles, of which the products of both groups are 2050: a
// product phase is 1250 (its 128 KB of operands pass LDS in 1020), the vector work beside it 1500 (512 of
// them the exponentials), and a wave's four loads hold it for 400.
#include "window_attn.h"

namespace dsp_window {
namespace {

typedef __attribute__((address_space(3))) dsp_u32x4 lds_u32x4_t;

constexpr int kWaves = 8, kRows = 32 * kWaves, kStages = 4;

// All but the newest `n` stages' loads (kLoads each) of this wave are done, n <= 2.
template <int kLoads>
__device__ __forceinline__ void wait_stages(int n) {
  if (n >= 2) __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<2 * kLoads>());
  else if (n == 1) __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<kLoads>());
  else __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<0>());
}

template <typename Tag, int D, int kFmt>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void
window_wide_kernel(const WinArgs a) {
  constexpr int NKS = D / 16, NDT = D / 32;   // 16-dim steps of K Q^T, 32-dim tiles of V^T P^T
  constexpr int CPR = D / 8, ROWB = 2 * D;    // 16-byte pieces and bytes of a row in LDS
  constexpr int SLAB = kChunk * ROWB;
  constexpr int RPW = kChunk / kWaves;        // rows a wave loads of a chunk, in one block
  constexpr int LPW = SLAB / 1024 / kWaves;   // KiB a wave loads of a slab
  constexpr int RPI = 1024 / ROWB;            // rows per LDS DMA
  constexpr bool kF16 = std::is_same<Tag, F16Tag>::value;
  static_assert(LPW >= 1 && LPW * RPI == RPW, "a wave's rows lie in one block");
  // K of chunk c in ring place c % 4, V likewise: stage c is V of chunk c, K of chunk c + 1
  __shared__ __attribute__((aligned(1024))) char lds[2][kStages][SLAB];
  // of stage c: which waves' rows of K have a bad block id; whether rows of V hold infinities or NaN
  constexpr uint32_t kOddValues = 1u << kWaves;
  __shared__ uint32_t s_flag[kStages];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hl = lane >> 5, col = lane & 31;
  const bool second = wave >= kWaves / 2;     // the group that runs a phase behind

  // ---- this workgroup's (sequence, KV head, tile, part), placed as in the tile kernel
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
  const int t0 = tile * kRows;
  if (t0 >= sq.rows) return;
  if (sq.bad) {
    if (part != 0) return;
    if (tile == 0 && kvh == 0 && threadIdx.x == 0 && a.err && (a.cu_q || sq.ctx != 0))
      atomicAdd(a.err, 1);
    for (int i = threadIdx.x; i < min(kRows, sq.rows - t0) * D; i += 64 * kWaves) {
      const int r = t0 + i / D;
      static_cast<uint16_t*>(a.out)[int64_t(sq.q0 + r / a.G) * a.ost +
                                    int64_t(kvh * a.G + r % a.G) * a.osh + i % D] = 0;
    }
    return;
  }
  const int base = sq.ctx - sq.n;
  const int tile_pf = base + t0 / a.G, tile_pl = base + (min(sq.rows, t0 + kRows) - 1) / a.G;
  const Span span = span_of<kChunk>(tile_pf, tile_pl, a.window, a.sinks);
  const int c0 = part * a.part_chunks, c1 = min(span.n, c0 + a.part_chunks);
  if (c0 >= c1) return;
  const int nc = c1 - c0;
  const bool whole = c0 == 0 && c1 == span.n;
  auto key_of = [&](int c) {  // the first key of the piece's chunk c
    const int x = c0 + c;
    return kChunk * (x + ((span.first - span.sink) & ~((x - span.sink) >> 31)));
  };

  // ---- this wave's rows (those past the last: the sequence's first, for nothing)
  const int r0 = t0 + 32 * wave;
  const bool has_rows = r0 < sq.rows;
  const int pf = base + r0 / a.G, pl = base + (min(sq.rows, r0 + 32) - 1) / a.G;
  const int r = r0 + col;
  const bool row_ok = r < sq.rows;
  const int qi = row_ok ? r / a.G : 0, tok = sq.q0 + qi;
  const int head = kvh * a.G + (row_ok ? r - qi * a.G : 0);
  const int pos = base + qi;
  dsp_u32x4 qop[NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks)
    qop[ks] = *reinterpret_cast<const dsp_u32x4*>(static_cast<const uint16_t*>(a.q) +
                                                  int64_t(tok) * a.qst + int64_t(head) * a.qsh +
                                                  16 * ks + 8 * hl);

  // ---- rows of a chunk: RPW * wave .., in one block.  (Rows of which none is seen, and those past the
  // last key, repeat the last key: as in the tile kernel.)
  auto kswz = [](int row) { return row & (CPR - 1); };
  auto vswz = [](int row) { return D >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); };
  const int bmask = (1 << a.log2_bs) - 1;
  const int32_t* const bt_row = a.bt + int64_t(b) * a.bt_stride;
  // Where they lie, for 64 chunks at a time, one in each lane: bytes from the cache's start, and the rows
  // after the first that may be read (-1: the block id is bad).
  bool any_bad = false;
  uint32_t at_lo = 0, at_hi = 0, scale_lo = 0, scale_hi = 0, room = 0;
  struct Rows {
    int64_t at, scale;
    int room;
  };
  auto next_rows = [&](int c) {  // chunk c's; called for 0, 1, 2, ...
    if ((c & 63) == 0) {
      const int k0 = key_of(min(c + lane, nc - 1)) + RPW * wave;
      const int seen = ((k0 - span.hi) & ((span.lo - k0 - RPW) | (k0 - a.sinks))) >> 31;
      const int k = (k0 & seen) | ((span.hi - 1) & ~seen);
      const uint32_t id = uint32_t(bt_row[k >> a.log2_bs]);
      const bool bad = id >= a.num_blocks;
      const int64_t slot = bad ? 0 : (int64_t(id) << a.log2_bs) + (k & bmask);
      const int64_t at = slot * a.slot_bytes, scale = slot * a.scale_slot;
      at_lo = uint32_t(at);
      at_hi = uint32_t(at >> 32);
      scale_lo = uint32_t(scale);
      scale_hi = uint32_t(scale >> 32);
      room = uint32_t(bad ? -1 : min(span.hi - 1 - k, RPW - 1));
      any_bad |= __builtin_amdgcn_ballot_w64(bad && c + lane < nc) != 0;
    }
    auto lane_of = [&](uint32_t x) { return uint32_t(__builtin_amdgcn_readlane(x, c & 63)); };
    Rows w;
    w.at = int64_t(uint64_t(lane_of(at_hi)) << 32 | lane_of(at_lo));
    w.scale = kFmt == kNone ? 0 : int64_t(uint64_t(lane_of(scale_hi)) << 32 | lane_of(scale_lo));
    w.room = int(lane_of(room));
    return w;
  };
  const char* const k_rows = a.kc + kvh * a.head_bytes;
  const char* const v_rows = a.vc + kvh * a.head_bytes;
  const uint32_t lds_base = uint32_t(reinterpret_cast<uintptr_t>((lds_void_t*)&lds[0][0][0]));
  Rows rows_k = next_rows(0), rows_v = rows_k;   // of the newest stage's K and V
  // which of the newest stages' rows are bad: bit c % 4 of K, bit 4 + c % 4 of V
  uint32_t bad_rows = 0;
  auto advance = [&](int c) {  // from stage c - 1's rows to stage c's: V of rows_v, K of rows_k
    rows_v = rows_k;
    rows_k = next_rows(c + 1);
    if (any_bad) {
      const int s = c & (kStages - 1);
      bad_rows = (bad_rows & ~(0x11u << s)) | uint32_t(rows_k.room < 0) << s |
                 uint32_t(rows_v.room < 0) << (4 + s);
    }
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
  auto send_plane = [&](const Rows& w, int plane, int place) {
    const char* const rows = (plane ? v_rows : k_rows) + w.at;
    const uint32_t m0 = lds_base + uint32_t((plane * kStages + place) * SLAB + wave * LPW * 1024);
    if (w.room < RPW - 1) {
#pragma unroll
      for (int j = 0; j < LPW; ++j) {
        const int rw = j * RPI + lane / CPR, row = RPW * wave + rw, sl = lane % CPR;
        dma16<false>(rows, uint32_t(min(rw, max(w.room, 0))) * uint32_t(a.slot_bytes) +
                               16 * (sl ^ (plane ? vswz(row) : kswz(row))), m0 + j * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < LPW; ++j) dma16<false>(rows, plane ? voff[j] : koff[j], m0 + j * 1024);
    }
  };
  // (the last stage has no next K: the last one again, so that every stage has as many loads)
  auto send = [&](int c) {
    advance(c);
    send_plane(rows_v, 1, c & (kStages - 1));
    send_plane(rows_k, 0, (c + 1) & (kStages - 1));
  };
  // Quantised caches: through registers, widened on the way to LDS.  A lane takes EL elements of a row.
  constexpr int EL = RPW * D / 64, EPR = D / EL;        // lanes a row
  constexpr int WL = (kFmt == kFp8 ? EL : EL / 2) / 4;  // words
  uint32_t raw[2][WL < 1 ? 1 : WL], raw_scale[2];
  auto load_plane = [&](const Rows& w, int plane) {
    const int rw = min(lane / EPR, max(w.room, 0)), el = lane % EPR * EL;
    const char* const p = (plane ? v_rows : k_rows) + w.at +
                          uint32_t(rw * int(a.slot_bytes) + dsp_quant::bytes<kFmt>(el));
    if constexpr (WL == 1) {
      raw[plane][0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      typedef uint32_t words_t __attribute__((ext_vector_type(WL < 2 ? 2 : WL)));
      const words_t x = *reinterpret_cast<const words_t*>(p);
#pragma unroll
      for (int i = 0; i < WL; ++i) raw[plane][i] = x[i];
    }
    raw_scale[plane] =
        ((plane ? a.vs : a.ks) + w.scale + kvh * a.scale_head)[uint32_t(
            rw * int(a.scale_slot) + el / dsp_quant::kGroup)];
  };
  auto store_plane = [&](int plane, int place) {
    const int row = RPW * wave + lane / EPR, sl = lane % EPR * EL / 8;
    uint32_t w[EL / 2];
    dsp_quant::widen<kFmt, kF16, EL>(raw[plane], dsp_quant::scale_of(raw_scale[plane]), w);
#pragma unroll
    for (int i = 0; i < EL / 8; ++i)
      *reinterpret_cast<dsp_u32x4*>(
          &lds[plane][place][row * ROWB + 16 * ((sl + i) ^ (plane ? vswz(row) : kswz(row)))]) =
          dsp_u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
  };
  auto load_stage = [&](int c) {
    advance(c);
    load_plane(rows_v, 1);
    load_plane(rows_k, 0);
  };
  auto store_stage = [&](int c) {
    store_plane(1, c & (kStages - 1));
    store_plane(0, (c + 1) & (kStages - 1));
  };

  // chunks seen0 .. seen1 - 1 of the piece: those of the window that all rows of the tile see whole
  const int seen0 =
      max(span.sink, (max(tile_pl - a.window, -1) + kChunk) / kChunk - span.first + span.sink) - c0;
  const int seen1 = (tile_pf + 1) / kChunk - span.first + span.sink - c0;
  // whether rows at positions f .. l, of the tile's, see all keys of chunk c
  auto sees_all = [&](int c, int f, int l) {
    if (c >= seen0 && c < seen1) return true;
    const int t = key_of(c);
    return t + kChunk - 1 <= f && (t > l - a.window || t + kChunk <= a.sinks);
  };
  // This wave's rows of stage c are in LDS: what the others have to know of them.
  auto arrived = [&](int c) {
    const int s = c & (kStages - 1);
    char* const my_v = &lds[1][s][wave * LPW * 1024];
    uint32_t flag = 0;
    if (any_bad) {
      flag = (bad_rows >> s & 1u) << wave;
      if (bad_rows >> (4 + s) & 1u) zero_rows<CPR, LPW>(my_v, 0);
    }
    if (!sees_all(c, tile_pf, tile_pl)) {
      __builtin_amdgcn_sched_barrier(0);
      flag |= any_nonfinite<Tag, LPW>(my_v) ? kOddValues : 0u;
    }
    if (flag && lane == 0) atomicOr(&s_flag[s], flag);
  };

  // ---- operands from LDS (V as load_vt reads it).  A slab's addresses are made from one by exclusive or,
  // anew in each phase: kept over the loop they do not fit into the registers.
  const uint32_t k_lane = lds_base + col * ROWB + 16 * (hl ^ kswz(col));
  const int v_key = 4 * hl + ((lane & 15) >> 2);
  const uint32_t v_lane = lds_base + kStages * SLAB + v_key * ROWB + 8 * (lane & 1) +
                          16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vswz(v_key));
  auto slab_at = [](uint32_t at, int c) {
    at += (c & (kStages - 1)) * SLAB;
    asm volatile("" : "+v"(at));
    return at;
  };
  auto read_k = [](uint32_t slab, int x, int ks) {
    return *reinterpret_cast<const lds_u32x4_t*>((slab ^ (32 * ks)) + 32 * x * ROWB);
  };
  auto read_v = [](uint32_t slab, int ps, int dt) {
    v4i16 vh[2];
#pragma unroll
    for (int inst = 0; inst < 2; ++inst)
      vh[inst] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_v4i16_t*>((slab ^ (64 * dt)) + (16 * ps + 8 * inst) * ROWB));
    return __builtin_bit_cast(dsp_u32x4, vh);
  };

  float m = -INFINITY, lpart = 0.f;
  f32x16 acc[NDT], sc[2];
  dsp_u32x4 pop[4];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[dt][j] = 0.f;
  // (m, kLag, kRef, kLeast: as in the tile kernel)
  constexpr float kLag = 8.f, kRef = kF16 ? 7.f : 0.f;
  constexpr uint32_t kLeast = kF16 ? 0x00010001u : 0x00800080u;
  auto window_bits = [&](int t, int x) {
    const int k = t + 32 * x + 4 * hl;
    return low_bits(pos - k + 1) & (~low_bits(pos - a.window - k + 1) | low_bits(a.sinks - k));
  };

  auto turn = [&] {  // the end of a phase
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
  };
  // S of chunk c
  auto scores = [&](int c) {
    const uint32_t slab = slab_at(k_lane, c);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[x][j] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
      for (int x = 0; x < 2; ++x) sc[x] = mfma32x32<Tag>(read_k(slab, x, ks), qop[ks], sc[x]);
  };
  // S of chunk c + 1 and O += V^T P^T of chunk c; the operands are read kAhead products ahead.
  auto products = [&](int c) {
    constexpr int kAhead = 8, kK = 2 * NKS, kV = 4 * NDT;
    const uint32_t k_slab = slab_at(k_lane, c + 1), v_slab = slab_at(v_lane, c);
    dsp_u32x4 op[kAhead];
    auto read = [&](int i) {
      if (i < kK) return read_k(k_slab, i & 1, i >> 1);
      return read_v(v_slab, (i - kK) / NDT, (i - kK) % NDT);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) op[i] = read(i);
    if constexpr (kFmt == kNone)
      if (c + 3 < nc) send(c + 3);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[x][j] = 0.f;
#pragma unroll
    for (int i = 0; i < kK + kV; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i < kK) {
        sc[i & 1] = mfma32x32<Tag>(op[i % kAhead], qop[i >> 1], sc[i & 1]);
      } else {
        const int ps = (i - kK) / NDT, dt = (i - kK) % NDT;
        acc[dt] = mfma32x32<Tag>(op[i % kAhead], pop[ps], acc[dt]);
      }
      if (i + kAhead < kK + kV) op[i % kAhead] = read(i + kAhead);
    }
  };
  // (rare) V of chunk c holds infinities or NaN and some row does not see it whole: they are added to the
  // rows that see their keys, and cleared.  By all waves at once, between the phases.
  auto odd_values = [&](int c) {
    const uint32_t slab = slab_at(v_lane, c);
    const int t = key_of(c);
#pragma unroll
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
        const dsp_u32x4 v = read_v(slab, ps, dt);
        acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, false), huge, acc[dt]);
        acc[dt] = mfma32x32<Bf16Tag>(odd_operand<Tag>(v, true), huge, acc[dt]);
      }
    }
    turn();
    clear_nonfinite<Tag, LPW>(&lds[1][c & (kStages - 1)][wave * LPW * 1024]);
    turn();
  };
  // P of chunk c from S; bad: waves whose rows of its K have a bad block id
  auto softmax = [&](int c, uint32_t bad) {
    const bool edge = !sees_all(c, pf, pl);
    if (edge) {
      const int t = key_of(c);
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
    const uint32_t least = edge || bad ? 0u : kLeast;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        const float p = dsp_exp2(fmaf(sc[x][j], a.scale_log2, neg_m));
        const float q = dsp_exp2(fmaf(sc[x][j + 1], a.scale_log2, neg_m));
        sum[0] += p;
        sum[1] += q;
        pop[2 * x + (j >> 3)][(j >> 1) & 3] = not_below(narrow2<Tag>(p, q), least);
      }
    lpart += sum[0] + sum[1];
  };

  // 16-bit caches: this wave's loads of stage c, behind which two stages more may be out
  auto arrive = [&](int c) {
    if constexpr (kFmt == kNone)
      if (c < nc) {
        __builtin_amdgcn_sched_barrier(0);
        wait_stages<2 * LPW>(min(nc - 1 - c, 2));
        arrived(c);
      }
  };

  // ---- the first chunk's S and P, by all waves
  if (threadIdx.x < kStages) s_flag[threadIdx.x] = 0;
  __syncthreads();
  const bool first_bad = rows_k.room < 0;
  if constexpr (kFmt == kNone) {
    send_plane(rows_k, 0, 0);
#pragma unroll
    for (int c = 0; c < 3; ++c)
      if (c < nc) send(c);
    __builtin_amdgcn_sched_barrier(0);
    // (of K of the first chunk; its stages' loads came behind it)
    if (nc >= 3) __builtin_amdgcn_s_waitcnt(dsp_waitcnt_vm<6 * LPW>());
    else wait_stages<2 * LPW>(nc);
  } else {
    load_plane(rows_k, 0);
    store_plane(0, 0);
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (c < nc) {
        load_stage(c);
        store_stage(c);
        arrived(c);
      }
    if (2 < nc) load_stage(2);
  }
  if (first_bad && lane == 0) atomicOr(&s_flag[kStages - 1], 1u << wave);
  // the wait for q, once: the compiler cannot count the loop's loads
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) asm volatile("" : "+v"(qop[ks]));
  turn();
  uint32_t flags = __builtin_amdgcn_readfirstlane(s_flag[kStages - 1]);
  if (has_rows) scores(0);
  arrive(0);
  if (has_rows) softmax(0, flags);
  turn();
  for (int c = 0; c < nc; ++c) {
    const uint32_t* const flag = &s_flag[c & (kStages - 1)];
    if (!(c >= seen0 && c < seen1)) {  // (in the others none looks for infinities)
      if (__builtin_amdgcn_readfirstlane(*flag) & kOddValues) odd_values(c);
    }
    if (second) turn();
    const uint32_t flag_now = *flag;
    // ---- products
    if (has_rows) {
      __builtin_amdgcn_s_setprio(1);
      products(c);  // (behind the last chunk: S of what lies there, for nothing)
      __builtin_amdgcn_s_setprio(0);
    } else if constexpr (kFmt == kNone) {
      if (c + 3 < nc) send(c + 3);
    }
    if (second) arrive(c + 1);
    turn();
    // ---- vector work
    if (flags && threadIdx.x == 0) s_flag[(c - 1) & (kStages - 1)] = 0;  // (all have read it)
    flags = __builtin_amdgcn_readfirstlane(flag_now);
    if constexpr (kFmt != kNone) {
      if (c + 2 < nc) {
        store_stage(c + 2);
        arrived(c + 2);
      }
      if (c + 3 < nc) load_stage(c + 3);
    }
    if (has_rows && c + 1 < nc) softmax(c + 1, flags & (kOddValues - 1));
    if (!second) {
      arrive(c + 1);
      turn();
    }
  }
  if (a.err && any_bad && lane == 0) atomicAdd(a.err, 1);  // once per wave
  // ---- the piece's rows: acc[dt][j] = O[row col][dim 32 dt + 8 (j / 4) + 4 hl + j % 4]
  lpart += dsp_shfl_xor(lpart, 32);
  if (!row_ok) return;
  if (whole) {
    const float inv = lpart == 0.f ? 0.f : 1.f / lpart;  // (0: no key counted; NaN stays)
    const int64_t o = int64_t(tok) * a.ost + int64_t(head) * a.osh + 4 * hl;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int j4 = 0; j4 < 4; ++j4)
        store4<Tag, false>(a, o + 32 * dt + 8 * j4,
                           f32x4{acc[dt][4 * j4], acc[dt][4 * j4 + 1], acc[dt][4 * j4 + 2],
                                 acc[dt][4 * j4 + 3]} * inv);
  } else {
    const int64_t row = ((int64_t(pair) * a.tiles + tile) * a.parts + part) * kRows + 32 * wave + col;
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

template <int D, int kFmt>
void launch_wide(bool f16, unsigned grid, const WinArgs& a, hipStream_t s) {
  if (f16) window_wide_kernel<F16Tag, D, kFmt><<<grid, 64 * kWaves, 0, s>>>(a);
  else window_wide_kernel<Bf16Tag, D, kFmt><<<grid, 64 * kWaves, 0, s>>>(a);
}

template <int D>
void launch_format(int fmt, bool f16, unsigned grid, const WinArgs& a, hipStream_t s) {
  if (fmt == kFp8) launch_wide<D, kFp8>(f16, grid, a, s);
  else if (fmt == kFp4) launch_wide<D, kFp4>(f16, grid, a, s);
  else launch_wide<D, kNone>(f16, grid, a, s);
}

}  // namespace

int wide_tiles(int D, int fmt, bool f16, unsigned grid, const WinArgs& a, hipStream_t s) {
  if (D == 64) launch_format<64>(fmt, f16, grid, a, s);
  else launch_format<128>(fmt, f16, grid, a, s);
  return dsp_launch_status();
}

}  // namespace dsp_window
