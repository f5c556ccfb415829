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

#include "f32x2.cuh"

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
KERN_DEVICE uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// four f32 -> four codes
KERN_DEVICE uint32_t codes4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
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
  int hq, hk, rot, page_size;
  float eps;
  int norm_plus_one;
  long long kv_slots;
  int max_pos, row_stride, q_stride;
  int* err;
};

// One key value in 64 bits: normed (dinv the row's factor, wx and wy the weights of it and of its partner) and turned.
__device__ __noinline__ float exact_value(float x, float y, float wx, float wy, double dinv, float c, float s) {
  return sticky_float(fma((double)x * ((double)wx * dinv), (double)c, (double)y * ((double)wy * dinv) * (double)s));
}

constexpr int kAppendThreads = 128;

// One block per token: its rows (q heads, then k and v heads) are dealt to groups of D / 8 lanes, a pass of all groups at a time, the
// next pass's loads ahead; the cosines and sines that a lane needs are the same for every head and stay in registers. What bounds it
// is how many loads are under way and the number of instructions, not the bytes: 8 blocks to an SM at 64 registers (8192 tokens of
// 32 + 8 heads of 128, written and read back: 53 us; 6 blocks at 80 registers 58, 9 at 56 55; 256 threads to a token 71). The form of
// the pairs and the norms are fixed when it is compiled, pairs of values go through two-wide products, and k rows alone pay for
// exact codes.
template <int D, bool INTER, bool NORM>
KERN_DEVICE void append_body(const AppendArgs& a) {
  constexpr int kLanes = D / 8, kGroups = kAppendThreads / kLanes;
  pdl_wait();
  const int t = blockIdx.x;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, i0 = lane * 8;
  const __nv_bfloat16* q_src = a.qkv + (size_t)t * a.row_stride + group * D + i0;
  const __nv_bfloat16* kv_src = q_src + a.hq * D;
  const uint4 none = make_uint4(0, 0, 0, 0);
  auto load = [&](const __nv_bfloat16* src, int h, int heads) { return h < heads ? *reinterpret_cast<const uint4*>(src) : none; };
  uint4 q_raw = load(q_src, group, a.hq), kv_raw = load(kv_src, group, 2 * a.hk);
  const long long pos64 = a.positions[t], slot64 = a.slots[t];
  int pos = (int)pos64, slot = (int)slot64;                  // (a pool of 2^31 tokens would not fit the memory)
  if (pos64 < 0 || pos64 >= a.max_pos || slot64 >= a.kv_slots) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BOUNDS);
    if (pos64 < 0 || pos64 >= a.max_pos) pos = 0;
    slot = -1;
  }
  if (slot64 < 0) slot = -1;
  const int half = a.rot >> 1;
  const bool turns = i0 < a.rot, upper = i0 >= half;
  // the lane's pairs: 8 of the rotate-half form (its values against those of the lane half a rotation away), or 4 of its own, each
  // twice; the sine with the sign that the value's partner takes
  uint64_t cs[4], sn[4];
  const int from = !INTER && turns ? (upper ? lane - half / 8 : lane + half / 8) : lane;
  if (turns) {
    const size_t row = (size_t)pos * half + (INTER ? i0 >> 1 : (upper ? i0 - half : i0));
    const float4* cp = reinterpret_cast<const float4*>(a.cos_tab + row);
    const float4* sp = reinterpret_cast<const float4*>(a.sin_tab + row);
    const float4 c0 = cp[0], s0 = sp[0];
    if constexpr (INTER) {
      cs[0] = pair64(c0.x, c0.x); cs[1] = pair64(c0.y, c0.y); cs[2] = pair64(c0.z, c0.z); cs[3] = pair64(c0.w, c0.w);
      sn[0] = pair64(-s0.x, s0.x); sn[1] = pair64(-s0.y, s0.y); sn[2] = pair64(-s0.z, s0.z); sn[3] = pair64(-s0.w, s0.w);
    } else {
      const float4 c1 = cp[1], s1 = sp[1];
      const float sign = upper ? 1.f : -1.f;
      cs[0] = pair64(c0.x, c0.y); cs[1] = pair64(c0.z, c0.w); cs[2] = pair64(c1.x, c1.y); cs[3] = pair64(c1.z, c1.w);
      sn[0] = pair64(sign * s0.x, sign * s0.y); sn[1] = pair64(sign * s0.z, sign * s0.w);
      sn[2] = pair64(sign * s1.x, sign * s1.y); sn[3] = pair64(sign * s1.z, sign * s1.w);
    }
  }
  // a row's values, and their partners' (zeros where nothing turns)
  auto partner_word = [&](uint32_t w) -> uint32_t { return INTER ? __byte_perm(w, 0, 0x1032) : __shfl_sync(0xffffffffu, w, from, kLanes); };
  auto open = [&](const uint4& raw, uint64_t (&y)[4], uint64_t (&v)[4]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16x2(w[i]), g = unpack_bf16x2(partner_word(w[i]));
      y[i] = pair64(f.x, f.y);
      v[i] = turns ? pair64(g.x, g.y) : 0;
    }
  };
  // norm of both by the row's root mean square and the weights at nw (none: as they are); the weights, for the exact form
  auto normed = [&](const __nv_bfloat16* nw, uint64_t (&y)[4], uint64_t (&v)[4], uint64_t (&wx)[4], uint64_t (&wy)[4]) {
    uint64_t s2 = mul2(y[0], y[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) s2 = fma2(y[i], y[i], s2);
    const float2 sf = split64(s2);
    const float ss = group_sum<kLanes>(sf.x + sf.y);
    if (nw == nullptr) return;
    const float m = ss / (float)D + a.eps;
    float inv = rsqrtf(m);
    // one Newton step: the hardware's estimate is two units off (an infinite row stays at 0)
    if (m <= 3.402823466e38f) inv = inv * fmaf(-0.5f * m * inv, inv, 1.5f);
    const uint64_t inv2 = pair64(inv, inv);
    const uint4 wv = *reinterpret_cast<const uint4*>(nw + i0), pv = *reinterpret_cast<const uint4*>(nw + from * 8);
    const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w}, pw[4] = {pv.x, pv.y, pv.z, pv.w};
    const float one = a.norm_plus_one ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16x2(ww[i]), g = unpack_bf16x2(INTER ? __byte_perm(ww[i], 0, 0x1032) : pw[i]);
      wx[i] = pair64(f.x + one, f.y + one);
      wy[i] = pair64(g.x + one, g.y + one);
      y[i] = mul2(y[i], mul2(wx[i], inv2));
      if (turns) v[i] = mul2(v[i], mul2(wy[i], inv2));
    }
  };

  // ---- q heads ----
  __nv_bfloat16* q_dst = a.q_out + (size_t)t * a.q_stride + group * D + i0;
  for (int h0 = 0; h0 < a.hq; h0 += kGroups) {
    const uint4 raw = q_raw;
    q_src += kGroups * D;
    q_raw = load(q_src, h0 + kGroups + group, a.hq);
    uint64_t y[4], v[4], wx[4], wy[4];
    open(raw, y, v);
    if constexpr (NORM) normed(a.q_norm, y, v, wx, wy);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (turns) y[i] = fma2(y[i], cs[i], mul2(v[i], sn[i]));
      const float2 f = split64(y[i]);
      o[i] = pack_bf16x2(f.x, f.y);
    }
    if (h0 + group < a.hq) *reinterpret_cast<uint4*>(q_dst) = make_uint4(o[0], o[1], o[2], o[3]);
    q_dst += kGroups * D;
  }
  // ---- k and v heads ----
  if (slot < 0) return;                                      // (uniform)
  const int page = slot / a.page_size, slot_off = slot - page * a.page_size;
  const size_t codes = (size_t)2 * a.hk * a.page_size * D;
  uint8_t* const pg = a.pool + (size_t)page * (codes + 2 * a.hk * a.page_size);
  // the row's largest value; one that is not finite becomes NaN and does not count
  auto biggest = [&](float (&x)[8]) -> float {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    if (__any_sync(0xffffffffu, top >= 0x7f800000u)) {
      top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
        if (u >= 0x7f800000u) x[i] = __uint_as_float(0x7fffffffu);
        else top = max(top, u);
      }
    }
    return __uint_as_float(group_max<kLanes>(top));
  };
  for (int h0 = 0; h0 < 2 * a.hk; h0 += kGroups) {
    const uint4 raw = kv_raw;
    kv_src += kGroups * D;
    kv_raw = load(kv_src, h0 + kGroups + group, 2 * a.hk);
    const int h = h0 + group;
    const bool is_k = h < a.hk;
    float x[8];
    uint32_t c[2];
    int e;
    auto plain = [&]() {                                     // codes of x as it is
      e = row_exponent(biggest(x));
      const float s = pow2f(-e);
#pragma unroll
      for (int i = 0; i < 2; ++i) c[i] = codes4(x[4 * i] * s, x[4 * i + 1] * s, x[4 * i + 2] * s, x[4 * i + 3] * s);
    };
    if (!__any_sync(0xffffffffu, is_k)) {                    // v rows: stored as they are
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
      plain();
    } else {
      uint64_t y[4], v[4], wx[4], wy[4];
      open(raw, y, v);
      const bool k_norm = NORM && is_k && a.k_norm != nullptr;
      if constexpr (NORM) normed(k_norm ? a.k_norm : nullptr, y, v, wx, wy);
      // off: how far a key may be from the exact one, several units of the 24 bits of both partners
      const float unit = is_k && (turns || k_norm) ? 4.76837158e-7f : 0.f;      // 2^-21
      float off[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 u = split64(y[i]), q = split64(v[i]);
        // (values are as they are, and an infinite neighbour is none of theirs: no product with a unit of 0)
        off[2 * i] = unit > 0.f ? (fabsf(u.x) + fabsf(q.x)) * unit : 0.f;
        off[2 * i + 1] = unit > 0.f ? (fabsf(u.y) + fabsf(q.y)) * unit : 0.f;
        const float2 f = is_k && turns ? split64(fma2(y[i], cs[i], mul2(v[i], sn[i]))) : u;
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
      const float top = biggest(x);
      e = row_exponent(top);
      const float s = pow2f(-e);
      uint32_t c2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* u = x + 4 * i;
        const float* d = off + 4 * i;
        c[i] = codes4((u[0] + d[0]) * s, (u[1] + d[1]) * s, (u[2] + d[2]) * s, (u[3] + d[3]) * s);
        c2[i] = codes4((u[0] - d[0]) * s, (u[1] - d[1]) * s, (u[2] - d[2]) * s, (u[3] - d[3]) * s);
      }
      const bool close = unit > 0.f && (c[0] != c2[0] || c[1] != c2[1] || row_exponent(top * 1.000001f) != row_exponent(top * 0.999999f));
      if (__any_sync(0xffffffffu, close)) {
        // a value, or the row's largest, sits next to a border: the warp's keys once more, in 64 bits
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        double dinv = 1.0;
        if constexpr (NORM) {
          double ss = 0.0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_bf16x2(w[i]);
            ss = fma((double)f.x, (double)f.x, fma((double)f.y, (double)f.y, ss));
          }
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const double m = ss / (double)D + (double)a.eps;
          if (k_norm) dinv = (double)rsqrtf((float)m);
          if (k_norm && m <= 3.402823466e38) {               // 22 bits, doubled twice
            dinv = dinv * fma(-0.5 * m * dinv, dinv, 1.5);
            dinv = dinv * fma(-0.5 * m * dinv, dinv, 1.5);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 own = unpack_bf16x2(w[i]);
          float2 oth = unpack_bf16x2(partner_word(w[i]));
          if (unit > 0.f) {
            const float2 one = make_float2(1.f, 1.f), ax = k_norm ? split64(wx[i]) : one, ay = k_norm ? split64(wy[i]) : one;
            const float2 cc = turns ? split64(cs[i]) : one, ss = turns ? split64(sn[i]) : make_float2(0.f, 0.f);
            if (!turns) oth = make_float2(0.f, 0.f);
            x[2 * i] = exact_value(own.x, oth.x, ax.x, ay.x, dinv, cc.x, ss.x);
            x[2 * i + 1] = exact_value(own.y, oth.y, ax.y, ay.y, dinv, cc.y, ss.y);
          }
        }
        plain();
      }
    }
    if (h < 2 * a.hk) {
      const size_t row = (size_t)h * a.page_size + slot_off;
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
  // a block for each token and run of its rows
  const int t = blockIdx.x, lane = threadIdx.x % kLanes;
  const long long slot64 = slots[t];
  if (slot64 >= kv_slots && threadIdx.x == 0) set_error(err, ERR_BOUNDS);
  const int slot = slot64 < 0 || slot64 >= kv_slots ? -1 : (int)slot64;
  const int page = slot < 0 ? 0 : slot / page_size, off = slot < 0 ? 0 : slot - page * page_size;
  const size_t codes = (size_t)2 * hk * page_size * D;
  const uint8_t* pg = pool + (size_t)page * (codes + 2 * hk * page_size);
  __nv_bfloat16* dst = out + (size_t)t * 2 * hk * D + lane * 8;
#pragma unroll 4
  for (int h = threadIdx.x / kLanes; h < 2 * hk; h += kAppendThreads / kLanes) {
    uint4 o = make_uint4(0, 0, 0, 0);
    const size_t r = (size_t)h * page_size + off;
    if (slot >= 0 && KERN_CHECK(pg + r * D + lane * 8, 8, SITE_KV_ROW)) {
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
    *reinterpret_cast<uint4*>(dst + (size_t)h * D) = o;
  }
}

}  // namespace kern

#define KERN_APPEND_ENTRY(D, PAIRS, INTER, NAME, NORM)                                                                            \
  extern "C" __global__ void __launch_bounds__(kAppendThreads, 8) kern_rope_kv_append_e4m3_##PAIRS##NAME##_d##D(                  \
      const __nv_bfloat16* qkv, __nv_bfloat16* q_out, uint8_t* pool, const long long* positions, const long long* slots,          \
      const float* cos_tab, const float* sin_tab, const __nv_bfloat16* q_norm, const __nv_bfloat16* k_norm, int hq, int hk,       \
      int rot, int page_size, float eps, int norm_plus_one, long long kv_slots, int max_pos, int row_stride, int q_stride,        \
      int* err) {                                                                                                                 \
    append_body<D, INTER, NORM>(AppendArgs{qkv, q_out, pool, positions, slots, cos_tab, sin_tab, q_norm, k_norm, hq, hk, rot,     \
                                           page_size, eps, norm_plus_one, kv_slots, max_pos, row_stride, q_stride, err});         \
  }
#define KERN_KV_E4M3(D)                                                                                                           \
  KERN_APPEND_ENTRY(D, half, false, , false)                                                                                      \
  KERN_APPEND_ENTRY(D, half, false, _norm, true)                                                                                  \
  KERN_APPEND_ENTRY(D, interleaved, true, , false)                                                                                \
  KERN_APPEND_ENTRY(D, interleaved, true, _norm, true)                                                                            \
  extern "C" __global__ void __launch_bounds__(kAppendThreads) kern_kv_read_e4m3_d##D(const uint8_t* pool, const long long* slots,           \
                                                                           __nv_bfloat16* out, int tokens, int hk, int page_size, \
                                                                           long long kv_slots, int* err) {                        \
    read_body<D>(pool, slots, out, tokens, hk, page_size, kv_slots, err);                                                         \
  }
KERN_KV_E4M3(64)
KERN_KV_E4M3(128)
KERN_KV_E4M3(256)
