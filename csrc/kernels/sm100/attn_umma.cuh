// What the many-row kernels of attention over a cache share (attn_tile.cu: head_dim 64 and 128, attn_tile256.cu: 256): tensor-core
// instructions, which block a CTA is, what a row sees, and the ways out for values that f16 or a product does not hold.
#pragma once
#include "attn_rows.cuh"
#include "f32x2.cuh"

namespace kern {

// Shared-memory descriptors (128-byte swizzle, groups of 8 rows 1024 bytes apart) have the same upper word for K-major operands and
// for MN-major ones (rows are the contraction's, 64 columns to a row, the next 64 `block_bytes` further on); a step along the
// contraction adds to the address in the lower one. The products' warp then issues an instruction with two additions.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
KERN_DEVICE uint32_t desc_low(uint32_t smem_addr, uint32_t block_bytes) { return ((smem_addr & 0x3FFFF) >> 4) | ((block_bytes >> 4) << 16); }
// kind::f16 with f32 sums: 16-bit operands, f16 or bf16
template <bool F16>
KERN_DEVICE constexpr uint32_t tile_idesc(int m, int n, bool b_mn) {
  return (1u << 4) | ((F16 ? 0u : 1u) << 7) | ((F16 ? 0u : 1u) << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// D[tmem] (+)= A[smem] B[smem], and with A in TMEM; one thread
KERN_DEVICE void umma_ss(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
KERN_DEVICE void umma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
KERN_DEVICE bool elect_lane() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
KERN_DEVICE void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
KERN_DEVICE void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
KERN_DEVICE void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
KERN_DEVICE void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
KERN_DEVICE void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
KERN_DEVICE float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
KERN_DEVICE uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// (8-bit) What turns a row's products with a key tile into base-2 scores: the row's factor times the tile's. Kept a normal number:
// a score that is not seen is -inf and stays it (zero queries on zero keys would make the factor 2^-149, which flushes to 0, and
// -inf * 0 NaN), and a product of 0 stays 0.
KERN_DEVICE float row_scale(float row, float tile) { return fminf(fmaxf(row * tile, 1.17549435e-38f), 3.402823466e38f); }

// (8-bit) The sum of weights is of weights that hold their value tile's exponent, and is freed of it tile by tile, so tiles' exponents
// may lie this far apart: 2^-26 of the largest weight is then 2^-126 of the largest product, f32's end. Blocks past it are computed again.
constexpr int kTilesApart = 100;
// the exponent E of a value tile that holds the least scale (6 less: keys and values are multiplied by 2^6 as they become f16)
constexpr float kLeastShift = kLeastScale - 127 - 6;

// (8-bit) A share's partials (reference m, sum l, O) are left with l in [0.5, 1): m is then of scores alone, and comparable with other
// shares', whose values may be of quite another size. Returns what O is to be multiplied by, a power of two.
KERN_DEVICE float level_share(float& m, float& l) {
  const int e = (int)(__float_as_uint(l) >> 23) & 255;
  if (e == 0 || e == 255) return 1.f;                         // (nothing seen, or what is not finite)
  const int shift = min(e - 126, 126);
  const float f = pow2i(-shift);
  m += (float)shift;
  l *= f;
  return f;
}

// (8-bit) Sets wide_s if one of this lane's four rows of a half, whose scale bytes are `word`, holds anything but zeros and is lost under
// the half's largest scale (`top`; f16 has room for 2^20 below it). Asked for where there is such a scale, which in earnest is a row of
// zeros'. Rows lie as they came: BLOCKS column blocks of BYTES to a row, in whatever order its pieces are. A call that gives nothing
// back, of 14 registers: 4 prompts take 388 us with it, 392 where it gave the answer back, and 395 with its loop among the conversions.
template <int BYTES, int BLOCKS>
__device__ __noinline__ void rows_lost(uint32_t codes, uint32_t block_bytes, int lane, uint32_t word, int top, volatile int* wide_s) {
  uint32_t any = 0;
#pragma unroll 1
  for (int k = 0; k < 4; ++k) {
    const int b = (int)(word >> (8 * k)) & 255;
    if (b == 0 || b + 20 >= top) continue;                    // (0: behind the end, or never written)
#pragma unroll 1
    for (int x = 0; x < BLOCKS * (BYTES / 16); ++x) {
      uint32_t v0, v1, v2, v3;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3)
                   : "r"(codes + (x / (BYTES / 16)) * block_bytes + (4 * lane + k) * BYTES + (x % (BYTES / 16)) * 16)
                   : "memory");
      any |= v0 | v1 | v2 | v3;
    }
  }
  if ((any & 0x7f7f7f7fu) != 0) *wide_s = 1;
}

// Block y of the call: (sequence, block of its rows) to found[0] and [1]; sequence -1 past the last. Blocks are counted through the
// sequences; where more are launched than run at once these are taken by length, so that the last blocks to start are the shortest.
// Every thread of the block calls (at least 256), warp 0 writes; scratch: 512 places in shared memory.
template <bool TREE>
KERN_DEVICE void find_block(const RowsArgs& a, int seqs, int toks, int* scratch, int* found) {
  const int lane = threadIdx.x & 31;
  const bool ranked = seqs > 1 && seqs <= 256 && gridDim.z == 1 && gridDim.x * gridDim.y > sm_count();
  int* order = scratch + 256;
  if (ranked) {
    const int rank = by_length(a.seq_lens, seqs, scratch);
    if (rank >= 0) order[rank] = threadIdx.x;
    __syncthreads();
  }
  if (threadIdx.x >= 32) return;
  int base = 0, sq = -1, bk = 0;
  for (int s0 = 0; s0 < seqs && sq < 0; s0 += 32) {
    const int s = ranked && s0 + lane < seqs ? order[s0 + lane] : s0 + lane;
    int rows = 0;
    if (s < seqs) rows = a.cu_q ? a.cu_q[s + 1] - a.cu_q[s] : a.rows_per_seq;
    if (rows > a.max_rows) {                                  // (there may be no blocks for them)
      set_error(a.err, ERR_BOUNDS);
      rows = 0;
    }
    int n = rows > 0 && rows >= a.row_lo && rows <= a.row_hi ? (rows + toks - 1) / toks : 0;
    const int own = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, n, d);
      if (lane >= d) n += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, (int)blockIdx.y < base + n);
    if (hit) {
      const int l = __ffs(hit) - 1;
      sq = __shfl_sync(0xffffffffu, s, l);
      const int upto = __shfl_sync(0xffffffffu, n, l), mine = __shfl_sync(0xffffffffu, own, l);
      bk = (int)blockIdx.y - (base + upto - mine);
      if (!TREE) bk = mine - 1 - bk;                          // causal: the longest walks first
    }
    base += __shfl_sync(0xffffffffu, n, 31);
  }
  if (lane == 0) {
    found[0] = sq;
    found[1] = bk;
  }
}

// Which of tokens j .. j + 31 a row sees: of a tree those before it (`past`) and the nodes of its mask, causal those up to its own
// place `pos`; none from `to` on.
template <bool TREE>
KERN_DEVICE uint32_t seen32(const long long* mask, int words, int past, int pos, int to, int j) {
  auto below = [](int n) -> uint32_t { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
  uint32_t b;
  if constexpr (TREE) {
    b = below(past - j);
    const int n0 = j - past;                                  // the node of bit 0 (negative: the context's last tokens before it)
    for (int w = max(n0 >> 6, 0); w <= (n0 + 31) >> 6 && w < words && n0 + 31 >= 0; ++w) {
      const unsigned long long m = (unsigned long long)mask[w];
      const int sh = n0 - w * 64;
      b |= sh >= 0 ? (uint32_t)(m >> sh) : (uint32_t)((m & 0xffffffffull) << -sh);
    }
  } else {
    b = below(pos + 1 - j);
  }
  return b & below(to - j);
}

// Infinities and NaN that a row sees among tokens j0 .. to - 1, whose products went without them: from the cache itself, into 32
// columns of the row from `col` on.
template <int D, bool E4M3, bool TREE>
KERN_DEVICE void put_back(const RowsArgs& a, const long long* mask, int seq, int past, int pos, int j0, int to, int col, uint32_t (&x)[32]) {
  const int kvh = blockIdx.x;
#pragma unroll 1
  for (int j = j0; j < to; ++j) {
    if (!(seen32<TREE>(mask, a.words, past, pos, to, j) & 1u)) continue;
    const int pi = j / a.page_size, off = j - pi * a.page_size;
    int page = pi < a.max_pages ? a.block_table[(size_t)seq * a.max_pages + pi] : 0;
    if (page < 0 || page >= a.pool_pages) page = 0;
    const size_t v_row = (size_t)(a.hk + kvh) * a.page_size + off;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if constexpr (E4M3) {
        const uint8_t code = a.pool[(size_t)page * (2 * a.hk * a.page_size * (size_t)(D + 1)) + v_row * D + col + i];
        if ((code & 0x7f) == 0x7f) x[i] = 0x7fffffffu;
      } else {
        const uint16_t w = reinterpret_cast<const uint16_t*>(a.pool)[(size_t)page * (2 * a.hk * a.page_size * (size_t)D) + v_row * D + col + i];
        if ((w & 0x7f80u) == 0x7f80u) x[i] = __float_as_uint(__uint_as_float(x[i]) + __uint_as_float((uint32_t)w << 16));
      }
    }
  }
}

// A block's rows over the 8-bit cache, a row to a warp in turn and some tokens at a time, for scales that have no common exponent, in a tile
// or over the tiles. Far slower than the products are: 4 prompts of up to 2048 rows on up to 6000 with such a row in every page take 97 ms, not
// 0.4, and 16 trees of up to 64 nodes on up to 4096 19 ms, not 0.08 (176 and 69 with one token under way at a time).
template <int D, bool TREE>
__device__ __noinline__ void tile_wide(const RowsArgs& a, int seq, int row0, int tok_lo, int valid, int past, int from, int to, int shares,
                                       int warps) {
  constexpr int kCols = D / 32, kAtOnce = D == 256 ? 4 : 8;   // columns of a lane; tokens
  const int G = a.hq / a.hk, kvh = blockIdx.x, lane = threadIdx.x & 31;
  const size_t codes = (size_t)2 * a.hk * a.page_size * D, page_bytes = codes + 2 * a.hk * a.page_size;
  const size_t to_v = (size_t)a.hk * a.page_size;
  for (int r = threadIdx.x >> 5; r < valid; r += warps) {
    const int tk = tok_lo + r / G, head = kvh * G + r % G, stop = TREE ? to : min(to, past + tk + 1);
    const long long* mask = TREE ? a.masks + (size_t)(row0 + tk) * a.words : nullptr;
    float q[kCols], o[kCols], m = kUnset, l = 0.f;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      q[i] = __bfloat162float(a.q[(size_t)(row0 + tk) * a.q_stride + (size_t)head * D + lane * kCols + i]) * a.scale_log2;
      o[i] = 0.f;
    }
#pragma unroll 1
    for (int j0 = from; j0 < stop; j0 += kAtOnce) {
      // a lane to each token: whether the row sees it, where it lies, its scale bytes
      const int j = j0 + lane % kAtOnce, in = min(j, stop - 1);
      bool see = j < stop;
      if (TREE && see && j >= past) {
        const int n = j - past;
        see = n >> 6 < a.words && (mask[n >> 6] >> (n & 63) & 1);
      }
      const unsigned live = __ballot_sync(0xffffffffu, see) & ((1u << kAtOnce) - 1);
      if (live == 0) continue;
      const int pi = in / a.page_size, off = in - pi * a.page_size;
      int page = pi < a.max_pages ? a.block_table[(size_t)seq * a.max_pages + pi] : 0;
      if (page < 0 || page >= a.pool_pages) page = 0;         // (recorded by the walk before)
      const uint8_t* sizes = a.pool + (size_t)page * page_bytes + codes + (size_t)kvh * a.page_size + off;
      const int k_size = sizes[0], v_size = sizes[to_v];
      uint32_t w[kAtOnce][2][(kCols + 3) / 4];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const uint8_t* src = a.pool + (size_t)__shfl_sync(0xffffffffu, page, u) * page_bytes +
                             ((size_t)kvh * a.page_size + __shfl_sync(0xffffffffu, off, u)) * D + lane * kCols;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* at = src + h * to_v * D;
          if constexpr (kCols == 2) {
            w[u][h][0] = *reinterpret_cast<const uint16_t*>(at);
          } else {
#pragma unroll
            for (int i = 0; i < kCols / 4; ++i) w[u][h][i] = reinterpret_cast<const uint32_t*>(at)[i];
          }
        }
      }
      // the lane's values of k or v of token u
      auto open = [&](int u, int h, float (&x)[kCols]) {
#pragma unroll
        for (int i = 0; i < kCols; i += 2) {
          uint32_t two, none;
          codes_f16x4(w[u][h][i / 4] >> (8 * (i & 2)), two, none);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
          x[i] = f.x;
          x[i + 1] = f.y;
        }
      };
      float s[kAtOnce], top = m;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        float k[kCols];
        open(u, 0, k);
        s[u] = 0.f;
#pragma unroll
        for (int i = 0; i < kCols; ++i) s[u] = fmaf(q[i], k[i], s[u]);
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1)
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], x);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        s[u] *= pow2i(__shfl_sync(0xffffffffu, k_size, u) - 127);
        if (live >> u & 1) top = fmaxf(top, s[u]);
      }
      const float keep = exp2f(m - top);
      m = top;
      l *= keep;
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[i] *= keep;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const float size = pow2i(__shfl_sync(0xffffffffu, v_size, u) - 127);
        if (!(live >> u & 1)) continue;                       // (uniform; what is not seen does not reach the row, whatever it is)
        float v[kCols];
        open(u, 1, v);
        const float p = exp2f(s[u] - m);
        l += p;
#pragma unroll
        for (int i = 0; i < kCols; ++i) o[i] = fmaf(p, v[i] * size, o[i]);
      }
    }
    if (shares == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int i = 0; i < kCols; i += 2)
        *reinterpret_cast<uint32_t*>(a.out + (size_t)(row0 + tk) * a.out_stride + (size_t)head * D + lane * kCols + i) = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
    } else {
      const size_t at = (ws_row(a.ws_step, seq, row0, tk) * a.hq + head) * gridDim.z + blockIdx.z;
#pragma unroll
      for (int i = 0; i < kCols; ++i) a.ws_o[at * D + lane * kCols + i] = o[i];
      if (lane == 0) {
        a.ws_ml[at * 2] = m;
        a.ws_ml[at * 2 + 1] = l;
      }
    }
  }
}

}  // namespace kern
