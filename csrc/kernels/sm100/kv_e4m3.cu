// A paged KV cache in 8-bit floating point: rotary positions and quantisation in one pass as a token's rows are written, and the
// rows read back.
//
// A row (one token, k or v, one head: D values) is held as x = code * 2^e: D e4m3 codes and one scale byte e + 127. e is the
// smallest exponent that brings the row's largest finite value to 448 or less (448 = 1.75 * 2^8, so it is read off the float's
// bits), kept within [-40, 119]. A power of two loses nothing against a free scale, since e4m3 has the same relative step over 15
// binades, and makes the dequantised value exact in bf16 and the scale exact wherever it is folded in: into scores, exponents or
// operands. A value that is not finite is stored as NaN and takes no part in the scale.
//
// Page layout of one layer, bytes: [page][ codes [k|v][kv head][page_size][D] | scale bytes [k|v][kv head][page_size] ]. A page is
// one run of memory (2 * heads * page_size * (D + 1) bytes, a multiple of 16), a (page, k|v, head) block one page_size x D tile.
//
// Both kernels move bytes and no more: 8 values a thread, 16-byte loads, a row in D / 8 neighbouring lanes, so that norms, row
// maxima and the partners of the rotate-half pairing are shuffles.
#include <cuda_fp8.h>

#include "common.cuh"

using namespace kern;

namespace kern {

constexpr int kScaleLow = -40, kScaleHigh = 119;

KERN_DEVICE float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// the exponent of a row whose largest finite value is `top`
KERN_DEVICE int row_exponent(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleLow), kScaleHigh);
}

template <int N>
KERN_DEVICE float group_sum(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int N>
KERN_DEVICE float group_max(float v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// A double as a float that a later rounding to fewer bits takes where it would have taken the double: cut, and the last bit set
// if anything was cut off. e4m3 has few borders, but one value in a million sits near enough to one for 24 bits to pick the wrong side.
KERN_DEVICE float sticky_float(double x) {
  const float f = __double2float_rz(x);
  return __uint_as_float(__float_as_uint(f) | ((double)f != x && fabsf(f) <= 3.402823466e38f ? 1u : 0u));
}

struct AppendArgs {
  const __nv_bfloat16* qkv;
  __nv_bfloat16* q_out;
  uint8_t* pool;
  const long long* positions;
  const long long* slots;
  const float* cos_tab;
  const float* sin_tab;
  const __nv_bfloat16* q_norm;
  const __nv_bfloat16* k_norm;
  int tokens, hq, hk, rot, page_size;
  float eps;
  int norm_plus_one, interleaved;
  long long kv_slots;
  int max_pos, row_stride, q_stride;
  int* err;
};

// One block per token: its rows (q, k, v heads) are dealt to groups of D / 8 lanes; the cosines and sines that a lane needs are
// the same for every head and stay in registers.
template <int D>
KERN_DEVICE void append_body(const AppendArgs& a) {
  constexpr int kLanes = D / 8;
  pdl_wait();
  const int t = blockIdx.x;
  if (t >= a.tokens) return;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, groups = blockDim.x / kLanes;
  long long pos = a.positions[t], slot = a.slots[t];
  if (pos < 0 || pos >= a.max_pos) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BOUNDS);
    pos = 0;
  }
  if (slot >= a.kv_slots) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BOUNDS);
    slot = -1;
  }
  const int half = a.rot >> 1, i0 = lane * 8;
  const bool turns = i0 < a.rot, upper = i0 >= half;
  // the lane's pairs: 8 of the rotate-half form (its values against those of the lane half a rotation away), or 4 of its own
  float cs[8], sn[8];
  const int partner_lanes = half / 8;
  if (turns) {
    const int j0 = a.interleaved ? i0 >> 1 : (upper ? i0 - half : i0);
    const float4* cp = reinterpret_cast<const float4*>(a.cos_tab + (size_t)pos * half + j0);
    const float4* sp = reinterpret_cast<const float4*>(a.sin_tab + (size_t)pos * half + j0);
    *reinterpret_cast<float4*>(cs) = cp[0];
    *reinterpret_cast<float4*>(sn) = sp[0];
    if (!a.interleaved) {
      *reinterpret_cast<float4*>(cs + 4) = cp[1];
      *reinterpret_cast<float4*>(sn + 4) = sp[1];
    }
  }
  const long long page = slot >= 0 ? slot / a.page_size : 0;
  const int slot_off = slot >= 0 ? (int)(slot % a.page_size) : 0;
  const size_t codes = (size_t)2 * a.hk * a.page_size * D;
  uint8_t* const pg = a.pool + (size_t)page * (codes + 2 * a.hk * a.page_size);
  const int rows = a.hq + 2 * a.hk;
  const __nv_bfloat16* src = a.qkv + (size_t)t * a.row_stride;

  // every group takes the same number of turns: the shuffles below want whole warps
  for (int h0 = 0; h0 < rows; h0 += groups) {
    const int h = h0 + group;
    const bool live = h < rows && (h < a.hq || slot >= 0);
    const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.hk;
    float x[8];
    uint32_t w0[4];
    {
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (live) raw = *reinterpret_cast<const uint4*>(src + (size_t)h * D + i0);
      w0[0] = raw.x; w0[1] = raw.y; w0[2] = raw.z; w0[3] = raw.w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(w0[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
    // the partners' values, and with norms the weights of both
    float y[8], wx[8], wy[8];
    const int from = turns && !a.interleaved ? (upper ? lane - partner_lanes : lane + partner_lanes) : lane;
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(__shfl_sync(0xffffffffu, w0[i], from, kLanes));
        y[2 * i] = f.x;
        y[2 * i + 1] = f.y;
      }
    }
    const __nv_bfloat16* nw = is_q ? a.q_norm : a.k_norm;
    const bool norm = (is_q || is_k) && nw != nullptr, changed = norm || ((is_q || is_k) && turns);
    float inv = 1.f;
    if (a.q_norm != nullptr || a.k_norm != nullptr) {        // uniform
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
      ss = group_sum<kLanes>(ss);
      if (norm) {
        const float m = ss / (float)D + a.eps;
        inv = rsqrtf(m);
        inv = inv * fmaf(-0.5f * m * inv, inv, 1.5f);        // one Newton step: the hardware's estimate is two units off
        const uint4 wv = *reinterpret_cast<const uint4*>(nw + i0);
        const uint4 pv = *reinterpret_cast<const uint4*>(nw + from * 8);
        const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w}, pw[4] = {pv.x, pv.y, pv.z, pv.w};
        const float one = a.norm_plus_one ? 1.f : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack_bf16x2(ww[i]), h2 = unpack_bf16x2(pw[i]);
          wx[2 * i] = f.x + one;
          wx[2 * i + 1] = f.y + one;
          wy[2 * i] = a.interleaved ? f.y + one : h2.x + one;
          wy[2 * i + 1] = a.interleaved ? f.x + one : h2.y + one;
        }
      }
    }
    // x becomes the row's values; off: how far they may be from the exact ones (several units of the 24 bits of both partners)
    float off[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float u = x[i], v = y[i];
      if (norm) {
        u *= wx[i] * inv;
        v *= wy[i] * inv;
      }
      off[i] = changed ? (fabsf(u) + fabsf(v)) * 4.76837158e-7f : 0.f;      // 2^-21
      if (turns && (is_q || is_k)) {
        const bool minus = a.interleaved ? (i & 1) == 0 : !upper;
        u = fmaf(u, a.interleaved ? cs[i >> 1] : cs[i], (minus ? -v : v) * (a.interleaved ? sn[i >> 1] : sn[i]));
      }
      y[i] = u;
    }
    if (is_q && live)
      *reinterpret_cast<uint4*>(a.q_out + (size_t)t * a.q_stride + (size_t)h * D + i0) =
          make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
    const bool stored = live && !is_q;
    if (!__any_sync(0xffffffffu, stored)) continue;
    auto biggest = [&]() {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!(fabsf(y[i]) <= 3.402823466e38f)) y[i] = __uint_as_float(0x7fffffffu);    // not finite: NaN
        top = fmaxf(top, fabsf(y[i]));                                                // (a NaN is not taken)
      }
      return group_max<kLanes>(top);
    };
    auto encode = [&](float scale, float by, uint32_t (&c)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(fmaf(off[4 * i], by, y[4 * i]) * scale, fmaf(off[4 * i + 1], by, y[4 * i + 1]) * scale), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(fmaf(off[4 * i + 2], by, y[4 * i + 2]) * scale, fmaf(off[4 * i + 3], by, y[4 * i + 3]) * scale), __NV_SATFINITE, __NV_E4M3);
        c[i] = lo | (hi << 16);
      }
    };
    float top = biggest();
    int e = row_exponent(top);
    uint32_t c[2], c2[2];
    encode(pow2f(-e), 1.f, c);
    encode(pow2f(-e), -1.f, c2);
    const bool close = stored && changed && (c[0] != c2[0] || c[1] != c2[1] || row_exponent(top * 1.000001f) != row_exponent(top * 0.999999f));
    if (__any_sync(0xffffffffu, close)) {
      // a value, or the row's largest, sits next to a border: the warp's keys once more, in 64 bits
      double dinv = 1.0;
      if (a.k_norm != nullptr) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fma((double)x[i], (double)x[i], ss);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const double m = ss / (double)D + (double)a.eps;
        dinv = (double)rsqrtf((float)m);
        dinv = dinv * fma(-0.5 * m * dinv, dinv, 1.5);       // 22 bits, doubled twice
        dinv = dinv * fma(-0.5 * m * dinv, dinv, 1.5);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float pv;
        if (a.interleaved) pv = x[i ^ 1];
        else {
          const float2 f = unpack_bf16x2(__shfl_sync(0xffffffffu, w0[i >> 1], from, kLanes));
          pv = (i & 1) ? f.y : f.x;
        }
        if (is_k && changed) {
          double u = x[i], v = pv;
          if (norm) {
            u *= (double)wx[i] * dinv;
            v *= (double)wy[i] * dinv;
          }
          if (turns) {
            const bool minus = a.interleaved ? (i & 1) == 0 : !upper;
            u = fma(u, (double)(a.interleaved ? cs[i >> 1] : cs[i]), (minus ? -v : v) * (double)(a.interleaved ? sn[i >> 1] : sn[i]));
          }
          y[i] = sticky_float(u);
        }
      }
      top = biggest();
      e = row_exponent(top);
      encode(pow2f(-e), 0.f, c);
    }
    if (stored) {
      const size_t row = ((size_t)(is_k ? 0 : a.hk) + (h - a.hq - (is_k ? 0 : a.hk))) * a.page_size + slot_off;
      uint8_t* dst = pg + row * D + i0;
      if (KERN_CHECK(dst, 8, SITE_KV_APPEND)) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(c[0], c[1]);
        if (lane == 0) pg[codes + row] = (uint8_t)(e + 127);
      }
    }
  }
  pdl_launch_dependents();
}

// Rows back as bf16, exact: [tokens][k|v][head][D]; a slot below zero reads as zeros.
template <int D>
KERN_DEVICE void read_body(const uint8_t* pool, const long long* slots, __nv_bfloat16* out, int tokens, int hk, int page_size,
                           long long kv_slots, int* err) {
  constexpr int kLanes = D / 8;
  pdl_wait();
  const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int lane = (int)(at % kLanes);
  const long long row = at / kLanes;
  const long long t = row / (2 * hk);
  if (t >= tokens) return;
  const int h = (int)(row % (2 * hk));
  long long slot = slots[t];
  if (slot >= kv_slots) {
    set_error(err, ERR_BOUNDS);
    slot = -1;
  }
  uint4 o = make_uint4(0, 0, 0, 0);
  if (slot >= 0) {
    const size_t codes = (size_t)2 * hk * page_size * D;
    const uint8_t* pg = pool + (size_t)(slot / page_size) * (codes + 2 * hk * page_size);
    const size_t r = (size_t)h * page_size + (size_t)(slot % page_size);
    if (KERN_CHECK(pg + r * D + lane * 8, 8, SITE_KV_ROW)) {
      const uint2 c = *reinterpret_cast<const uint2*>(pg + r * D + lane * 8);
      const float s = pow2f((int)pg[codes + r] - 127);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t pair = ((i < 2 ? c.x : c.y) >> ((i & 1) * 16)) & 0xffffu;
        const __half2 hv = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3));
        const float2 f = __half22float2(hv);
        w[i] = pack_bf16x2(f.x * s, f.y * s);
      }
      o = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  *reinterpret_cast<uint4*>(out + (size_t)row * D + lane * 8) = o;
}

}  // namespace kern

#define KERN_APPEND_ENTRY(D)                                                                                                      \
  extern "C" __global__ void __launch_bounds__(256, 3) kern_rope_kv_append_e4m3_d##D(                                                \
      const __nv_bfloat16* qkv, __nv_bfloat16* q_out, uint8_t* pool, const long long* positions, const long long* slots,          \
      const float* cos_tab, const float* sin_tab, const __nv_bfloat16* q_norm, const __nv_bfloat16* k_norm, int tokens, int hq,   \
      int hk, int rot, int page_size, float eps, int norm_plus_one, int interleaved, long long kv_slots, int max_pos,             \
      int row_stride, int q_stride, int* err) {                                                                                   \
    append_body<D>(AppendArgs{qkv, q_out, pool, positions, slots, cos_tab, sin_tab, q_norm, k_norm, tokens, hq, hk, rot,          \
                              page_size, eps, norm_plus_one, interleaved, kv_slots, max_pos, row_stride, q_stride, err});         \
  }                                                                                                                               \
  extern "C" __global__ void __launch_bounds__(256) kern_kv_read_e4m3_d##D(const uint8_t* pool, const long long* slots,           \
                                                                           __nv_bfloat16* out, int tokens, int hk, int page_size, \
                                                                           long long kv_slots, int* err) {                        \
    read_body<D>(pool, slots, out, tokens, hk, page_size, kv_slots, err);                                                         \
  }
KERN_APPEND_ENTRY(64)
KERN_APPEND_ENTRY(128)
KERN_APPEND_ENTRY(256)
