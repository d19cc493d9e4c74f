// Rows into a quantised cache, and back (the reference's pool holds the model's type only:
// dispec/kv/paged_cache.py:61-72).
//
// Written: of 32 neighbouring elements x of a head, with M the format's largest number,
//     e = the least of -100 .. 118 with max |x| <= M 2^e,   code = round(clamp(x / 2^e, -M, M)),
// to nearest, halves to the even code; read: code 2^e.  All of it is exact but the one rounding,
// so the order of the operations does not show.  fp16 rows are first clamped to the largest number
// that the format has below fp16's end (61440, 49152): what is read back is finite in fp16.
//
// A thread takes units of 8 elements; a group's maximum is that of four neighbouring lanes (two quad
// permutes).  Bound by memory: each row is read once and written once.  2050 tokens of 36 layers in and
// out 150 us in a loop (88 and 69 where a trace has the kernels one by one), in which 760 MB have to be
// moved, 5.1 TB/s, and 916 are with the codes that go out and back; 4096 out, 915 MB, 169 us, 5.4 TB/s.
// A streaming copy of 2 GiB reaches 6.4 on this card, torch's 5.1; a row here is 1 KiB of codes, in blocks
// at any place.  32 rows of one layer: 3 us a kernel, 5 with the call.
#include <algorithm>

#include "dsp_common.h"
#include "dsp_quant.h"

namespace {

using namespace dsp_quant;

constexpr int kThreads = 256;

struct QBf16 { using store = uint16_t; static constexpr int32_t code = DSP_BF16; };
struct QF16 { using store = uint16_t; static constexpr int32_t code = DSP_F16; };
struct QF32 { using store = float; static constexpr int32_t code = DSP_F32; };

// n / d for n < 2^31: ((n * mul >> 32) + n) >> shift, shift = ceil(log2 d) (the compiler's division is
// tens of instructions, and a launch does little else beside its memory traffic).
struct Div {
  uint32_t mul, shift;
  explicit Div(uint32_t d) : shift(uint32_t(dsp_log2i(d))) {
    mul = uint32_t((uint64_t((uint64_t(1) << shift) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return (__umulhi(n, mul) + n) >> shift;
  }
};

// K or V: codes and scales [layer][slot][head], rows of whole heads; values [layer][token][head][D].
struct Plane {
  uint8_t* codes;
  uint8_t* scales;
  char* rows;
  int64_t layer, token, head;  // of rows, elements
};
struct RowArgs {
  Plane plane[2];
  int64_t code_layer, code_slot, scale_layer, scale_slot;  // bytes
  int64_t num_slots;
  const int64_t* slots;
  uint32_t tokens, head_units, row_units;  // units of a head, of a row
  Div by_head, by_row;
  int32_t* err;
};

typedef dsp_u32x4 u4;

// 8 elements as they lie in memory, from element `at` on.
template <typename T, bool kVec, bool kOnce>
__device__ __forceinline__ void load8(const char* base, int64_t at, u4 (&w)[2]) {
  const typename T::store* p = reinterpret_cast<const typename T::store*>(base) + at;
  constexpr bool kF32 = std::is_same<T, QF32>::value;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < (kF32 ? 2 : 1); ++i) {
      const u4* q = reinterpret_cast<const u4*>(p) + i;
      w[i] = kOnce ? dsp_ld_stream(q) : *q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kF32) w[i / 4][i % 4] = __float_as_uint(p[i]);
      else if (i % 2 == 0) w[0][i / 2] = uint32_t(p[i]) | uint32_t(p[i + 1]) << 16;
    }
  }
}
template <typename T>
__device__ __forceinline__ void as_floats(const u4 (&w)[2], float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (std::is_same<T, QF32>::value) x[j] = __uint_as_float(w[j / 4][j % 4]);
    else if (T::code == DSP_F16) x[j] = j % 2 ? dsp_f16hi(w[0][j / 2]) : dsp_f16lo(w[0][j / 2]);
    else x[j] = j % 2 ? dsp_bf16hi(w[0][j / 2]) : dsp_bf16lo(w[0][j / 2]);
  }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), DPP_QUAD_XOR1, 0xf, 0xf, false)));
  return max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), DPP_QUAD_XOR2, 0xf, 0xf, false)));
}

// Where unit i of a plane lies: units of a row side by side, then the next token's.
struct Unit {
  uint32_t token, u;
  int64_t slot;
  bool in, ok;
};
__device__ __forceinline__ Unit unit_of(const RowArgs& a, uint32_t i) {
  Unit x;
  x.token = a.by_row(i);
  x.in = x.token < a.tokens;   // (whole groups: row_units is a multiple of 4)
  x.u = i - x.token * a.row_units;
  x.slot = a.slots[x.in ? x.token : 0];
  x.ok = x.in && x.slot >= 0 && x.slot < a.num_slots;
  // counted once, of K's first layer
  if (x.in && !x.ok && x.u == 0 && blockIdx.y == 0 && blockIdx.z == 0 && a.err) atomicAdd(a.err, 1);
  return x;
}

// Workgroups (kPer * kThreads units, layer, plane).
template <typename T, int kFmt, bool kVec, int kPer, bool kOnce>
__global__ __launch_bounds__(kThreads) void append_kernel(const RowArgs a) {
  const Plane& pl = a.plane[blockIdx.z];
  const uint32_t first = blockIdx.x * (kPer * kThreads) + threadIdx.x;
  Unit unit[kPer];
  u4 raw[kPer][2];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    unit[k] = unit_of(a, first + k * kThreads);
    if (!unit[k].in) continue;
    const uint32_t head = a.by_head(unit[k].u), part = unit[k].u - head * a.head_units;
    load8<T, kVec, kOnce>(pl.rows, blockIdx.y * pl.layer + unit[k].token * pl.token + head * pl.head +
                                       8 * part, raw[k]);
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (!unit[k].ok) continue;
    float x[8];
    as_floats<T>(raw[k], x);
    // |x| as integers rise with it: infinities and NaN are the largest
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[j]) & 0x7fffffffu);
    most = quad_max(most);
    const bool none = most >= 0x7f800000u;
    if constexpr (T::code == DSP_F16) {
      constexpr float kEnd = kFmt == kFp8 ? 61440.f : 49152.f;
      most = min(most, __float_as_uint(kEnd));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fminf(fmaxf(x[j], -kEnd), kEnd);
    }
    // M = 1.75 * 2^8 or 1.5 * 2^2
    constexpr int kTop = kFmt == kFp8 ? 8 : 2;
    constexpr uint32_t kPart = kFmt == kFp8 ? 0x600000u : 0x400000u;
    constexpr float kMost = kFmt == kFp8 ? 448.f : 6.f;
    const int e = min(max(int(most >> 23) - 127 - kTop + int((most & 0x7fffffu) > kPart), kMinExp),
                      kMaxExp);
    const float scale = scale_of(uint32_t(e + 127)), end = kMost * scale;
    if (none || e == kMaxExp) {  // (rare: elsewhere no element is beyond the end)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = none ? 0.f : fminf(fmaxf(x[j], -end), end);
    }
    uint8_t* const codes = pl.codes + blockIdx.y * a.code_layer + unit[k].slot * a.code_slot;
    if constexpr (kFmt == kFp8) {
      typedef short s16x2 __attribute__((ext_vector_type(2)));
      dsp_u32x2 w;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s16x2 c = {0, 0};
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, x[4 * h], x[4 * h + 1], scale, false);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, x[4 * h + 2], x[4 * h + 3], scale, true);
        w[h] = __builtin_bit_cast(uint32_t, c);
      }
      *reinterpret_cast<dsp_u32x2*>(codes + 8 * unit[k].u) = w;
    } else {
      uint32_t w = 0;
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
      *reinterpret_cast<uint32_t*>(codes + 4 * unit[k].u) = w;
    }
    if (unit[k].u % 4 == 0)
      pl.scales[blockIdx.y * a.scale_layer + unit[k].slot * a.scale_slot + unit[k].u / 4] =
          uint8_t(none ? kNanScale : uint32_t(e + 127));
  }
}

template <typename T, int kFmt, int kPer, bool kOnce>
__global__ __launch_bounds__(kThreads) void gather_kernel(const RowArgs a) {
  const Plane& pl = a.plane[blockIdx.z];
  const uint32_t first = blockIdx.x * (kPer * kThreads) + threadIdx.x;
  Unit unit[kPer];
  uint32_t w[kPer][2], byte[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    unit[k] = unit_of(a, first + k * kThreads);
    if (!unit[k].ok) continue;
    const uint8_t* const codes = pl.codes + blockIdx.y * a.code_layer + unit[k].slot * a.code_slot;
    byte[k] = pl.scales[blockIdx.y * a.scale_layer + unit[k].slot * a.scale_slot + unit[k].u / 4];
    if constexpr (kFmt == kFp8) {
      const dsp_u32x2* p = reinterpret_cast<const dsp_u32x2*>(codes + 8 * unit[k].u);
      const dsp_u32x2 x = kOnce ? dsp_ld_stream(p) : *p;
      w[k][0] = x[0];
      w[k][1] = x[1];
    } else {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(codes + 4 * unit[k].u);
      w[k][0] = kOnce ? dsp_ld_stream(p) : *p;
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (!unit[k].ok) continue;
    const float scale = scale_of(byte[k]);
    const int64_t at = blockIdx.y * pl.layer + unit[k].token * pl.token + 8 * int64_t(unit[k].u);
    auto put = [](u4 v, u4* p) {
      if constexpr (kOnce) dsp_st_stream(v, p);
      else *p = v;
    };
    uint32_t h[4];
    if constexpr (std::is_same<T, QF32>::value) {
      widen<kFmt, false, 8>(w[k], scale, h);  // (bf16: exact)
      u4* const p = reinterpret_cast<u4*>(reinterpret_cast<float*>(pl.rows) + at);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        put(u4{h[2 * i] << 16, h[2 * i] & 0xffff0000u, h[2 * i + 1] << 16, h[2 * i + 1] & 0xffff0000u},
            p + i);
    } else {
      widen<kFmt, T::code == DSP_F16, 8>(w[k], scale, h);
      put(u4{h[0], h[1], h[2], h[3]},
          reinterpret_cast<u4*>(reinterpret_cast<uint16_t*>(pl.rows) + at));
    }
  }
}

bool strides_ok(std::initializer_list<int64_t> strides, int64_t each) {
  for (int64_t s : strides)
    if (s < 0 || s % each != 0) return false;
  return true;
}

// The arguments that both directions check alike.
int check_rows(const RowArgs& a, int64_t layers, int64_t tokens, int32_t KVH, int32_t D,
               int32_t format, int32_t dtype) {
  for (const Plane& p : a.plane) {
    DSP_HOST_CHECK(p.codes && p.scales, DSP_EINVAL);
    DSP_HOST_CHECK(tokens == 0 || (p.rows && a.slots), DSP_EINVAL);
  }
  DSP_HOST_CHECK(layers >= 0 && layers <= 65535 && tokens >= 0 && KVH > 0 && D > 0 &&
                     a.num_slots >= 0,
                 DSP_EINVAL);
  DSP_HOST_CHECK(dtype == DSP_BF16 || dtype == DSP_F16 || dtype == DSP_F32, DSP_EUNSUPPORTED);
  DSP_HOST_CHECK((format == DSP_KV_FP8 || format == DSP_KV_FP4) && D % kGroup == 0, DSP_EUNSUPPORTED);
  DSP_HOST_CHECK(int64_t(KVH) * D <= (1 << 20), DSP_EUNSUPPORTED);
  const int64_t row = int64_t(KVH) * D / (format == DSP_KV_FP8 ? 1 : 2);
  DSP_HOST_CHECK(a.code_slot >= row && a.scale_slot >= int64_t(KVH) * D / kGroup && a.code_layer >= 0 &&
                     a.scale_layer >= 0,
                 DSP_EINVAL);
  DSP_HOST_CHECK(strides_ok({a.code_slot, a.code_layer}, 8) && dsp_aligned(a.plane[0].codes, 8) &&
                     dsp_aligned(a.plane[1].codes, 8),
                 DSP_EALIGN);
  return DSP_OK;
}

template <typename F>
int by_type(int32_t dtype, int32_t format, F f) {
  auto of = [&](auto t) {
    return format == DSP_KV_FP8 ? f(t, std::integral_constant<int, kFp8>{})
                                : f(t, std::integral_constant<int, kFp4>{});
  };
  return dtype == DSP_F32 ? of(QF32{}) : dtype == DSP_F16 ? of(QF16{}) : of(QBf16{});
}

// 4 units a thread, whose loads go together, where the chip is full with that (2050 tokens of 36 layers
// in and out 216 -> 156 us); values that no cache keeps until they are needed by non-temporal accesses.
constexpr int kUnits = 4;
constexpr int64_t kFull = int64_t(1) << 21;   // units of a launch
constexpr int64_t kOnceBytes = int64_t(128) << 20;

// f(arguments, workgroups, units a thread, non-temporal) for runs of tokens that fit a launch each (units
// are numbered in 32 bits).
template <typename F>
int in_runs(const RowArgs& a, int64_t layers, int64_t tokens, int64_t es, F f) {
  const int64_t most = (int64_t(1) << 31) / a.row_units - kUnits * kThreads;
  const int64_t units = 2 * layers * tokens * a.row_units;
  for (int64_t t = 0; t < tokens; t += most) {
    RowArgs r = a;
    r.tokens = uint32_t(std::min(most, tokens - t));
    r.slots += t;
    for (Plane& p : r.plane) p.rows += t * p.token * es;
    auto launch = [&](auto per, auto once) {
      const int64_t each = int64_t(decltype(per)::value) * kThreads;
      f(r, dim3(unsigned((int64_t(r.tokens) * r.row_units + each - 1) / each), unsigned(layers), 2u), per,
        once);
    };
    using std::integral_constant;
    if (units < kFull) launch(integral_constant<int, 1>{}, std::false_type{});
    else if (8 * es * units < kOnceBytes) launch(integral_constant<int, kUnits>{}, std::false_type{});
    else launch(integral_constant<int, kUnits>{}, std::true_type{});
    const int st = dsp_launch_status();
    if (st != DSP_OK) return st;
  }
  return DSP_OK;
}

}  // namespace

extern "C" int dsp_kv_append_quant(
    void* k_pool, void* k_scale, void* v_pool, void* v_scale, int64_t num_layers,
    int64_t pool_layer_stride_bytes, int64_t pool_slot_stride_bytes,
    int64_t scale_layer_stride_bytes, int64_t scale_slot_stride_bytes, int64_t num_slots,
    const void* k, int64_t k_stride_l, int64_t k_stride_t, int64_t k_stride_h, const void* v,
    int64_t v_stride_l, int64_t v_stride_t, int64_t v_stride_h, const int64_t* slots,
    int64_t num_tokens, int32_t KVH, int32_t D, int32_t format, int32_t dtype,
    int32_t* err_count, dsp_stream_t stream) {
  DSP_HOST_CHECK(KVH > 0 && D > 0, DSP_EINVAL);
  // (of shapes that check_rows refuses: any)
  const uint32_t head_units = uint32_t(std::max(D / 8, 1));
  const uint32_t row_units = uint32_t(std::min(int64_t(KVH) * head_units, int64_t(1) << 20));
  auto rows = [](const void* p) { return static_cast<char*>(const_cast<void*>(p)); };
  const RowArgs a{{{static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(k_scale), rows(k), k_stride_l,
                    k_stride_t, k_stride_h},
                   {static_cast<uint8_t*>(v_pool), static_cast<uint8_t*>(v_scale), rows(v), v_stride_l,
                    v_stride_t, v_stride_h}},
                  pool_layer_stride_bytes, pool_slot_stride_bytes, scale_layer_stride_bytes,
                  scale_slot_stride_bytes, num_slots, slots, 0, head_units, row_units, Div(head_units),
                  Div(row_units), err_count};
  const int st = check_rows(a, num_layers, num_tokens, KVH, D, format, dtype);
  if (st != DSP_OK) return st;
  const int64_t es = dtype == DSP_F32 ? 4 : 2;
  DSP_HOST_CHECK(dsp_aligned(k, es) && dsp_aligned(v, es), DSP_EALIGN);
  if (num_layers == 0 || num_tokens == 0) return DSP_OK;
  const bool vec = strides_ok({k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t, v_stride_h},
                              16 / es) &&
                   dsp_aligned(k, 16) && dsp_aligned(v, 16);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return by_type(dtype, format, [&](auto t, auto fmt) {
    using T = decltype(t);
    constexpr int kF = decltype(fmt)::value;
    return in_runs(a, num_layers, num_tokens, es, [&](const RowArgs& r, dim3 grid, auto per, auto once) {
      constexpr int kPer = decltype(per)::value;
      constexpr bool kOnce = decltype(once)::value;
      if (vec) append_kernel<T, kF, true, kPer, kOnce><<<grid, kThreads, 0, s>>>(r);
      else append_kernel<T, kF, false, kPer, false><<<grid, kThreads, 0, s>>>(r);
    });
  });
}

extern "C" int dsp_kv_gather_quant(
    const void* k_pool, const void* k_scale, const void* v_pool, const void* v_scale,
    int64_t num_layers, int64_t pool_layer_stride_bytes, int64_t pool_slot_stride_bytes,
    int64_t scale_layer_stride_bytes, int64_t scale_slot_stride_bytes, int64_t num_slots,
    const int64_t* slots, int64_t num_tokens, int32_t KVH, int32_t D, int32_t format, void* k_out,
    void* v_out, int32_t dtype, int32_t* err_count, dsp_stream_t stream) {
  DSP_HOST_CHECK(KVH > 0 && D > 0, DSP_EINVAL);
  // (of shapes that check_rows refuses: any)
  const uint32_t head_units = uint32_t(std::max(D / 8, 1));
  const uint32_t row_units = uint32_t(std::min(int64_t(KVH) * head_units, int64_t(1) << 20));
  const int64_t row = int64_t(KVH) * D, layer = row * num_tokens;
  auto bytes = [](const void* p) { return static_cast<uint8_t*>(const_cast<void*>(p)); };
  const RowArgs a{{{bytes(k_pool), bytes(k_scale), static_cast<char*>(k_out), layer, row, D},
                   {bytes(v_pool), bytes(v_scale), static_cast<char*>(v_out), layer, row, D}},
                  pool_layer_stride_bytes, pool_slot_stride_bytes, scale_layer_stride_bytes,
                  scale_slot_stride_bytes, num_slots, slots, 0, head_units, row_units, Div(head_units),
                  Div(row_units), err_count};
  const int st = check_rows(a, num_layers, num_tokens, KVH, D, format, dtype);
  if (st != DSP_OK) return st;
  DSP_HOST_CHECK(dsp_aligned(k_out, 16) && dsp_aligned(v_out, 16), DSP_EALIGN);
  if (num_layers == 0 || num_tokens == 0) return DSP_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return by_type(dtype, format, [&](auto t, auto fmt) {
    return in_runs(a, num_layers, num_tokens, dtype == DSP_F32 ? 4 : 2,
                   [&](const RowArgs& r, dim3 grid, auto per, auto once) {
      gather_kernel<decltype(t), decltype(fmt)::value, decltype(per)::value, decltype(once)::value>
          <<<grid, kThreads, 0, s>>>(r);
    });
  });
}
