// Rows into a quantised cache, and back (the reference's pool holds the model's type only:
// dispec/kv/paged_cache.py:61-72).
//
// Written: of 32 neighbouring elements x of a head, with M the format's largest number,
//     e = the least of -100 .. 118 with max |x| <= M 2^e,   code = round(clamp(x / 2^e, -M, M)),
// to nearest, halves to the even code; read: code 2^e.  All of it is exact but the one rounding,
// so the order of the operations does not show.  fp16 rows are first clamped to the largest number
// that the format has below fp16's end (61440, 49152): what is read back is finite in fp16.
//
// One thread takes 8 elements of K or V; a group's maximum is that of four neighbouring lanes (two
// quad permutes).  Bound by memory: each row is read once and written once.
#include "dsp_common.h"
#include "dsp_quant.h"

namespace {

using namespace dsp_quant;

constexpr int kThreads = 256;

struct QBf16 { using store = uint16_t; static constexpr int32_t code = DSP_BF16; };
struct QF16 { using store = uint16_t; static constexpr int32_t code = DSP_F16; };
struct QF32 { using store = float; static constexpr int32_t code = DSP_F32; };

struct RowArgs {
  uint8_t* kc;   // codes and scales: [layer][slot][head], rows of whole heads
  uint8_t* ks;
  uint8_t* vc;
  uint8_t* vs;
  int64_t code_layer, code_slot, scale_layer, scale_slot;  // bytes
  int64_t num_slots;
  char* k;       // rows: [layer][token][head][D]
  char* v;
  int64_t k_layer, k_token, k_head, v_layer, v_token, v_head;  // elements
  const int64_t* slots;
  uint32_t tokens, head_units, row_units;  // units (of kUnit elements) of a head, and of K's and V's row
  int32_t* err;
};

template <typename T, int kN, bool kVec>
__device__ __forceinline__ void load_row(const char* base, int64_t at, float (&x)[kN]) {
  const typename T::store* p = reinterpret_cast<const typename T::store*>(base) + at;
  if constexpr (kVec && std::is_same<T, QF32>::value) {
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      const dsp_u32x4 w = *reinterpret_cast<const dsp_u32x4*>(p + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * i + j] = __uint_as_float(w[j]);
    }
  } else if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kN / 8; ++i) {
      const dsp_u32x4 w = *reinterpret_cast<const dsp_u32x4*>(p + 8 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[8 * i + 2 * j] = T::code == DSP_F16 ? dsp_f16lo(w[j]) : dsp_bf16lo(w[j]);
        x[8 * i + 2 * j + 1] = T::code == DSP_F16 ? dsp_f16hi(w[j]) : dsp_bf16hi(w[j]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if constexpr (std::is_same<T, QF32>::value) x[i] = p[i];
      else x[i] = T::code == DSP_F16 ? dsp_f16lo(p[i]) : dsp_bf16lo(p[i]);
    }
  }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), DPP_QUAD_XOR1, 0xf, 0xf, false)));
  return max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), DPP_QUAD_XOR2, 0xf, 0xf, false)));
}

// Unit i of a launch: 8 elements; K's units of a row, then V's; a row's, then the next token's.
template <typename T, int kFmt, bool kVec>
__global__ __launch_bounds__(kThreads) void append_kernel(RowArgs a) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x, layer = blockIdx.y;
  const uint32_t token = i / (2 * a.row_units);
  if (token >= a.tokens) return;  // (whole groups: row_units is a multiple of 4)
  uint32_t u = i - token * 2 * a.row_units;
  const bool is_v = u >= a.row_units;
  if (is_v) u -= a.row_units;
  const uint32_t head = u / a.head_units, part = u - head * a.head_units;
  const int64_t slot = a.slots[token];
  float x[8];
  if (is_v)
    load_row<T, 8, kVec>(a.v, layer * a.v_layer + token * a.v_token + head * a.v_head + 8 * part, x);
  else
    load_row<T, 8, kVec>(a.k, layer * a.k_layer + token * a.k_token + head * a.k_head + 8 * part, x);
  if (slot < 0 || slot >= a.num_slots) {
    if (!is_v && u == 0 && layer == 0 && a.err) atomicAdd(a.err, 1);
    return;
  }
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
  const uint32_t byte = none ? kNanScale : uint32_t(e + 127);
  const float scale = scale_of(uint32_t(e + 127)), end = kMost * scale;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = none ? 0.f : fminf(fmaxf(x[j], -end), end);
  uint8_t* const codes = (is_v ? a.vc : a.kc) + layer * a.code_layer + slot * a.code_slot;
  uint8_t* const scales = (is_v ? a.vs : a.ks) + layer * a.scale_layer + slot * a.scale_slot;
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
    *reinterpret_cast<dsp_u32x2*>(codes + 8 * u) = w;
  } else {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    *reinterpret_cast<uint32_t*>(codes + 4 * u) = w;
  }
  if (u % 4 == 0) scales[u / 4] = uint8_t(byte);
}

template <typename T, int kFmt>
__global__ __launch_bounds__(kThreads) void gather_kernel(RowArgs a) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x, layer = blockIdx.y;
  const uint32_t token = i / (2 * a.row_units);
  if (token >= a.tokens) return;
  uint32_t u = i - token * 2 * a.row_units;
  const bool is_v = u >= a.row_units;
  if (is_v) u -= a.row_units;
  const int64_t slot = a.slots[token];
  if (slot < 0 || slot >= a.num_slots) {
    if (!is_v && u == 0 && layer == 0 && a.err) atomicAdd(a.err, 1);
    return;
  }
  const uint8_t* const codes = (is_v ? a.vc : a.kc) + layer * a.code_layer + slot * a.code_slot;
  const float scale =
      scale_of(((is_v ? a.vs : a.ks) + layer * a.scale_layer + slot * a.scale_slot)[u / 4]);
  uint32_t w[2];
  if constexpr (kFmt == kFp8) {
    const dsp_u32x2 x = *reinterpret_cast<const dsp_u32x2*>(codes + 8 * u);
    w[0] = x[0];
    w[1] = x[1];
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(codes + 4 * u);
    w[1] = 0;
  }
  char* const rows = is_v ? a.v : a.k;
  const int64_t at = layer * (is_v ? a.v_layer : a.k_layer) +
                     token * (is_v ? a.v_token : a.k_token) + 8 * int64_t(u);
  if constexpr (std::is_same<T, QF32>::value) {
    uint32_t h[4];  // bf16, exact
    widen<kFmt, false, 8>(w, scale, h);
    dsp_u32x4 o[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j / 2][2 * (j % 2)] = h[j] << 16;
      o[j / 2][2 * (j % 2) + 1] = h[j] & 0xffff0000u;
    }
    dsp_u32x4* const p = reinterpret_cast<dsp_u32x4*>(reinterpret_cast<float*>(rows) + at);
    p[0] = o[0];
    p[1] = o[1];
  } else {
    dsp_u32x4 o;
    uint32_t h[4];
    widen<kFmt, T::code == DSP_F16, 8>(w, scale, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = h[j];
    *reinterpret_cast<dsp_u32x4*>(reinterpret_cast<uint16_t*>(rows) + at) = o;
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
  DSP_HOST_CHECK(a.kc && a.ks && a.vc && a.vs, DSP_EINVAL);
  DSP_HOST_CHECK(tokens == 0 || (a.k && a.v && a.slots), DSP_EINVAL);
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
  DSP_HOST_CHECK(strides_ok({a.code_slot, a.code_layer}, 8) && dsp_aligned(a.kc, 8) &&
                     dsp_aligned(a.vc, 8),
                 DSP_EALIGN);
  return DSP_OK;
}

// Tokens of one launch: units are numbered in 32 bits.
int64_t launch_tokens(const RowArgs& a) { return (int64_t(1) << 31) / (2 * a.row_units) - kThreads; }

template <typename F>
int by_type(int32_t dtype, int32_t format, F f) {
  auto of = [&](auto t) {
    return format == DSP_KV_FP8 ? f(t, std::integral_constant<int, kFp8>{})
                                : f(t, std::integral_constant<int, kFp4>{});
  };
  return dtype == DSP_F32 ? of(QF32{}) : dtype == DSP_F16 ? of(QF16{}) : of(QBf16{});
}

// f(arguments, workgroups) for runs of tokens that fit a launch each.
template <typename F>
int in_runs(RowArgs a, int64_t tokens, int64_t es, F f) {
  const int64_t most = launch_tokens(a);
  for (int64_t t = 0; t < tokens; t += most) {
    RowArgs r = a;
    r.tokens = uint32_t(std::min(most, tokens - t));
    r.slots += t;
    r.k += t * a.k_token * es;
    r.v += t * a.v_token * es;
    f(r, unsigned((int64_t(r.tokens) * 2 * r.row_units + kThreads - 1) / kThreads));
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
  RowArgs a{static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(k_scale),
            static_cast<uint8_t*>(v_pool), static_cast<uint8_t*>(v_scale),
            pool_layer_stride_bytes, pool_slot_stride_bytes, scale_layer_stride_bytes,
            scale_slot_stride_bytes, num_slots,
            static_cast<char*>(const_cast<void*>(k)), static_cast<char*>(const_cast<void*>(v)),
            k_stride_l, k_stride_t, k_stride_h, v_stride_l, v_stride_t, v_stride_h, slots,
            0, uint32_t(D / 8), uint32_t(int64_t(KVH) * D / 8), err_count};
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
    return in_runs(a, num_tokens, es, [&](const RowArgs& r, unsigned groups) {
      const dim3 grid(groups, unsigned(num_layers));
      if (vec) append_kernel<T, kF, true><<<grid, kThreads, 0, s>>>(r);
      else append_kernel<T, kF, false><<<grid, kThreads, 0, s>>>(r);
    });
  });
}

extern "C" int dsp_kv_gather_quant(
    const void* k_pool, const void* k_scale, const void* v_pool, const void* v_scale,
    int64_t num_layers, int64_t pool_layer_stride_bytes, int64_t pool_slot_stride_bytes,
    int64_t scale_layer_stride_bytes, int64_t scale_slot_stride_bytes, int64_t num_slots,
    const int64_t* slots, int64_t num_tokens, int32_t KVH, int32_t D, int32_t format, void* k_out,
    void* v_out, int32_t dtype, int32_t* err_count, dsp_stream_t stream) {
  const int64_t row = int64_t(KVH) * D, layer = row * num_tokens;
  RowArgs a{static_cast<uint8_t*>(const_cast<void*>(k_pool)),
            static_cast<uint8_t*>(const_cast<void*>(k_scale)),
            static_cast<uint8_t*>(const_cast<void*>(v_pool)),
            static_cast<uint8_t*>(const_cast<void*>(v_scale)),
            pool_layer_stride_bytes, pool_slot_stride_bytes, scale_layer_stride_bytes,
            scale_slot_stride_bytes, num_slots, static_cast<char*>(k_out),
            static_cast<char*>(v_out), layer, row, D, layer, row, D, slots, 0, uint32_t(D / 8),
            uint32_t(row / 8), err_count};
  const int st = check_rows(a, num_layers, num_tokens, KVH, D, format, dtype);
  if (st != DSP_OK) return st;
  DSP_HOST_CHECK(dsp_aligned(k_out, 16) && dsp_aligned(v_out, 16), DSP_EALIGN);
  if (num_layers == 0 || num_tokens == 0) return DSP_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return by_type(dtype, format, [&](auto t, auto fmt) {
    return in_runs(a, num_tokens, dtype == DSP_F32 ? 4 : 2, [&](const RowArgs& r, unsigned groups) {
      gather_kernel<decltype(t), decltype(fmt)::value>
          <<<dim3(groups, unsigned(num_layers)), kThreads, 0, s>>>(r);
    });
  });
}
