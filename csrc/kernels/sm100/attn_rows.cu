// Attention of few query rows over a paged cache, bf16 or e4m3 (kv_e4m3.cu has the 8-bit layout): single tokens, short causal
// blocks, and trees of drafted tokens, in which a row sees the whole context before the tree and those nodes of it whose bit its
// mask has.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^(scale log2(e) q_i.k_j - m_i)  over the j that row i sees; no such j: zeros
//
// One CTA = (16 query rows: the G heads of 16 / G tokens, one kv head, a share of the context). A producer warp brings tiles of
// 64 tokens into a ring of shared memory by TMA; four warps take 16 tokens of each tile and keep (m, l, O) of their own; the four
// are joined at the end, and the shares of one row, written as partials, by a second kernel (kern_attn_rows_merge).
//
// The time goes to reading the cache, so the arithmetic has to stay well under the memory's rate with little shared-memory
// traffic. Operands go from shared memory to registers in 16-byte loads and are not moved again: the order of the contraction
// index and of the output columns inside an mma.sync fragment is free as long as both operands agree, so a lane takes whole
// 16-byte pieces of a key row (Q's fragment is built in the same order), and whole pieces of value rows, of which it pairs two
// tokens' bytes with PRMT. The same code then serves bf16 words and e4m3 bytes, which become f16 pairs, exactly, in one
// instruction (cvt.rn.f16x2.e4m3x2). Tokens are dealt to lanes so that the 8 lanes of a shared-memory phase hit 8 different
// 16-byte columns of the 128-byte swizzle.
//
// 8-bit: Q goes to f16 with its row's power of two taken out; the scores of a key row are multiplied by its scale in f32; a value
// row's scale goes into its weight, w_ij = p_ij 2^(e_j - c_i), where c_i follows the largest s_ij + e_j - m_i seen, so that the
// f16 weights that matter are between 2^-14 and 1 whatever the sizes of the value rows. Rounding a weight to f16 (2^-11) is four
// steps finer than the output's own rounding; bf16 caches take bf16 weights (2^-8 of each weight, as the value rows' own rounding).
//
// Values that a row does not see do not reach it, whatever they are: tokens behind the sequence's end are cleared, and in the
// tiles where rows see different tokens values that are not finite are taken out of the product and put back for the rows that
// see them (a second pass of products over 0 / 1, only when there are any).
#include <cuda_fp8.h>

#include "common.cuh"

namespace kern {

constexpr int kTile = 64;            // tokens per tile
constexpr int kRowsThreads = 160;    // four warps of products, one producer

struct RowsArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* ws_o;               // partials [row][head][splits][D] (one split: none)
  float* ws_ml;              // [row][head][splits][2]
  const uint8_t* pool;       // (8-bit) scale bytes are read from here
  const int* block_table;
  const int* seq_lens;
  const int* cu_q;
  const long long* masks;    // (tree) [row][words]
  int* err;
  int words, rows_per_seq, hq, hk, q_stride, out_stride, max_pages, page_size, splits, pool_pages;
  float scale_log2;
};

template <int D, bool E4M3>
struct RowsCfg {
  static constexpr int kRowBytes = D * (E4M3 ? 1 : 2);
  static constexpr int kHalf = kTile * kRowBytes;                    // a tile of K or of V
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kScaleBytes = E4M3 ? 2 * kTile : 0;
  // about 96 KB of ring, so that two CTAs share an SM (one at 128 KB rows)
  static constexpr int kStages = kStage >= 65536 ? 3 : (98304 / kStage > 8 ? 8 : 98304 / kStage);
  static constexpr int kQBytes = D == 256 ? (D / 16) * 32 * 16 : 0;  // Q's fragments, where registers do not hold them
  static constexpr int kSmem = 1024 + kStages * (kStage + kScaleBytes) + kQBytes + 256;
  static constexpr int kBox = kRowBytes < 128 ? kRowBytes : 128;     // bytes of a row in one box
};

// byte offset of (token, 16-byte piece) in a tile of kRowBytes rows stored as 128-byte column blocks with the TMA's swizzle
template <int RB>
KERN_DEVICE uint32_t piece_off(int tok, int piece) {
  if constexpr (RB == 64) {
    return (uint32_t)(tok * 64 + ((piece ^ ((tok >> 1) & 3)) << 4));
  } else {
    return (uint32_t)((piece >> 3) * (kTile * 128) + tok * 128 + (((piece & 7) ^ (tok & 7)) << 4));
  }
}

KERN_DEVICE uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
KERN_DEVICE uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
KERN_DEVICE uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
// two e4m3 codes (low 16 bits) -> two f16, exact
KERN_DEVICE uint32_t codes_f16x2(uint32_t pair) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(pair));
  return r;
}
KERN_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool F16>
KERN_DEVICE void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// 4 bytes global -> shared, and an arrival on `bar` once this lane's copies so far have landed (counted by the barrier's setting)
KERN_DEVICE void async_copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
KERN_DEVICE void async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// of the two 16-bit (f16 or bf16) halves of w: all ones where the half is not finite
template <bool F16>
KERN_DEVICE uint32_t not_finite(uint32_t w) {
  constexpr uint32_t lo = F16 ? 0x7c00u : 0x7f80u;
  uint32_t r = 0;
  if ((w & lo) == lo) r |= 0xffffu;
  if ((w & (lo << 16)) == (lo << 16)) r |= 0xffff0000u;
  return r;
}

KERN_DEVICE float pow2i(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }

// how many shares the context of `tiles` tiles is cut into: no share under four tiles
KERN_DEVICE int rows_shares(int tiles, int splits) { return min(splits, max(1, (tiles + 3) / 4)); }

template <int D, bool E4M3, bool TREE>
KERN_DEVICE void rows_body(const CUtensorMap* kv_map, const RowsArgs& a) {
  using Cfg = RowsCfg<D, E4M3>;
  constexpr int RB = Cfg::kRowBytes, kStages = Cfg::kStages;
  constexpr int KP = RB / 64;              // 16-byte pieces of a key row per lane
  constexpr int VB = RB / 8;               // bytes of a value row per lane: D / 8 columns
  constexpr int NC = D / 8;                // value columns per lane = n-tiles of O
  constexpr int KS = D / 16;               // k-steps of Q K^T
  constexpr bool kQShared = D == 256;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stages = smem;
  uint8_t* scales = smem + kStages * Cfg::kStage;
  uint4* q_frag = reinterpret_cast<uint4*>(scales + kStages * Cfg::kScaleBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(q_frag) + Cfg::kQBytes);
  uint64_t* empty_bar = full_bar + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty_bar + kStages);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.hq / a.hk;
  const int seq = blockIdx.y, blk = blockIdx.x / a.hk, kvh = blockIdx.x % a.hk;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], E4M3 ? 33 : 1);
      mbar_init(&empty_bar[s], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(kv_map);
  }
  __syncthreads();
  pdl_wait();

  const int L = max(a.seq_lens[seq], 0);
  const int row0 = a.cu_q ? a.cu_q[seq] : seq * a.rows_per_seq;
  const int R = a.cu_q ? a.cu_q[seq + 1] - row0 : a.rows_per_seq;
  const int toks = 16 / G > 0 ? 16 / G : 1;
  const int tok_lo = blk * toks;
  if (tok_lo >= R) return;                                   // uniform per CTA
  const int valid = min(toks, R - tok_lo) * G;
  const int past = L - R;                                    // what the sequence had before this call's rows
  // causal: the last row of the block decides how far the walk goes
  const int end = TREE ? L : max(0, past + tok_lo + min(toks, R - tok_lo));
  const int tiles_all = (end + kTile - 1) / kTile;
  const int shares = rows_shares(tiles_all, a.splits);
  const int split = blockIdx.z;
  if (split >= shares) return;
  const int per = (tiles_all + shares - 1) / shares;
  const int tile_lo = split * per, ntiles = max(0, min(tiles_all, tile_lo + per) - tile_lo);

  // ---- Q's fragments, in the order in which a lane holds the keys ----
  const int g = lane >> 2, c = lane & 3;
  const int rA = g, rB = g + 8;
  uint32_t qf[KS][4];
  float f_row[2] = {a.scale_log2, a.scale_log2};             // what turns a row's products into base-2 scores
  if (warp < 4 && (!kQShared || warp == 0)) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = hh ? rB : rA;
      const bool ok = r < valid;
      const __nv_bfloat16* src = a.q + (size_t)(row0 + tok_lo + (ok ? r / G : 0)) * a.q_stride + (size_t)(kvh * G + (ok ? r % G : 0)) * D;
      if constexpr (E4M3) {
        // 16 values to a piece: words w of the piece make k-step 4 i + w
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            const uint4 v = ok ? *reinterpret_cast<const uint4*>(src + (c + 4 * i) * 16 + h2 * 8) : make_uint4(0, 0, 0, 0);
            qf[4 * i + 2 * h2][hh] = v.x;
            qf[4 * i + 2 * h2][2 + hh] = v.y;
            qf[4 * i + 2 * h2 + 1][hh] = v.z;
            qf[4 * i + 2 * h2 + 1][2 + hh] = v.w;
          }
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const float2 u = unpack_bf16x2(qf[s][hh]), v = unpack_bf16x2(qf[s][2 + hh]);
          top = fmaxf(top, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(v.x), fabsf(v.y))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int x = min(max((int)((__float_as_uint(top) >> 23) & 255) - 127, -100), 100);
        const float inv = pow2i(-x);
        f_row[hh] = a.scale_log2 * pow2i(x);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const float2 u = unpack_bf16x2(qf[s][hh]), v = unpack_bf16x2(qf[s][2 + hh]);
          qf[s][hh] = pack_f16x2(u.x * inv, u.y * inv);
          qf[s][2 + hh] = pack_f16x2(v.x * inv, v.y * inv);
        }
      } else {
        // 8 values to a piece: its words make k-steps 2 i and 2 i + 1
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          const uint4 v = ok ? *reinterpret_cast<const uint4*>(src + (c + 4 * i) * 8) : make_uint4(0, 0, 0, 0);
          qf[2 * i][hh] = v.x;
          qf[2 * i][2 + hh] = v.y;
          qf[2 * i + 1][hh] = v.z;
          qf[2 * i + 1][2 + hh] = v.w;
        }
      }
    }
  }
  if constexpr (kQShared) {
    float* f_s = reinterpret_cast<float*>(const_cast<int*>(abort_flag) + 1);
    if (warp == 0) {
#pragma unroll
      for (int s = 0; s < KS; ++s) q_frag[s * 32 + lane] = make_uint4(qf[s][0], qf[s][1], qf[s][2], qf[s][3]);
      if (c == 0) {
        f_s[rA] = f_row[0];
        f_s[rB] = f_row[1];
      }
    }
    __syncthreads();
    f_row[0] = f_s[rA];
    f_row[1] = f_s[rB];
  }

  float o[NC][4];
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, w_run[2] = {-INFINITY, -INFINITY};
  int c_run[2] = {-1000, -1000};
#pragma unroll
  for (int i = 0; i < NC; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  if (warp == 4) {
    // ---------------- producer ----------------
    const int box = a.page_size < kTile ? a.page_size : kTile;
    const int* pages = a.block_table + (size_t)seq * a.max_pages;
    int stage = 0;
    uint32_t phase = 0;
    for (int t = 0; t < ntiles; ++t) {
      if (!mbar_wait_ns(&empty_bar[stage], phase ^ 1, abort_flag)) {
        set_error(a.err, ERR_WAIT_EMPTY);
        *abort_flag = 1;
        break;
      }
      const int tok0 = (tile_lo + t) * kTile;
      uint8_t* sk = stages + stage * Cfg::kStage;
      // (page, row in page) of a token; tokens behind the end read the pool's first page
      auto place = [&](int tok, int& page, int& off) {
        page = 0;
        off = 0;
        const int pi = tok / a.page_size;
        if (tok < L && pi < a.max_pages) {
          page = pages[pi];
          off = tok - pi * a.page_size;
        }
        if (page < 0 || page >= a.pool_pages) {
          set_error(a.err, ERR_BOUNDS);
          page = 0;
        }
      };
      if (lane == 0) mbar_expect_tx(&full_bar[stage], Cfg::kStage);
      __syncwarp();
      for (int b = lane; b < kTile / box; b += 32) {
        int page, off;
        place(tok0 + b * box, page, off);
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
          for (int cb = 0; cb < RB / Cfg::kBox; ++cb)
            tma_load_3d(sk + which * Cfg::kHalf + cb * (kTile * 128) + b * box * Cfg::kBox, kv_map, cb * (Cfg::kBox * D / RB),
                        (which * a.hk + kvh) * a.page_size + off, page, &full_bar[stage]);
      }
      if constexpr (E4M3) {
        const int which = lane >> 4, i4 = (lane & 15) * 4;
        int page, off;
        place(tok0 + i4, page, off);
        const size_t codes = (size_t)2 * a.hk * a.page_size * D;
        const uint8_t* src = a.pool + (size_t)page * (codes + 2 * a.hk * a.page_size) + codes + (size_t)(which * a.hk + kvh) * a.page_size + off;
        if (KERN_CHECK(src, 4, SITE_KV_ROW)) async_copy4(smem_u32(scales + stage * Cfg::kScaleBytes + which * kTile + i4), src);
        async_arrive(&full_bar[stage]);
      }
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
  } else {
    // ---------------- products ----------------
    const int posA = rA < valid ? past + tok_lo + rA / G : -1, posB = rB < valid ? past + tok_lo + rB / G : -1;
    const long long* maskA = TREE ? a.masks + (size_t)(row0 + tok_lo + (rA < valid ? rA / G : 0)) * a.words : nullptr;
    const long long* maskB = TREE ? a.masks + (size_t)(row0 + tok_lo + (rB < valid ? rB / G : 0)) * a.words : nullptr;
    // whether a row of this block sees token j
    auto sees = [&](int j, int pos, const long long* mask) -> bool {
      if constexpr (TREE) {
        if (j < past) return true;
        const int n = j - past;
        return j < L && n < a.words * 64 && ((mask[n >> 6] >> (n & 63)) & 1);
      } else {
        return j <= pos;
      }
    };
    // the first token that some row of the block may not see
    const int clear = TREE ? past : past + tok_lo + 1;
    const int wtok = warp * 16;
    int stage = 0;
    uint32_t phase = 0;
    for (int t = 0; t < ntiles; ++t) {
      if (!mbar_wait_ns(&full_bar[stage], phase, abort_flag)) {
        set_error(a.err, ERR_WAIT_FULL);
        *abort_flag = 1;
        break;
      }
      const uint32_t sk = smem_u32(stages + stage * Cfg::kStage), sv = sk + Cfg::kHalf;
      const int tok0 = (tile_lo + t) * kTile + wtok;          // this warp's first token
      if (tok0 < end) {
        // ---- S = Q K^T: n-tile n holds tokens n * 8 + (0, 4, 1, 5, 2, 6, 3, 7), so that neighbouring rows of a load differ in
        // the bit of the swizzle that a row's own pieces do not reach ----
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
          const int tok = wtok + n * 8 + ((g & 1) << 2 | (g >> 1));
#pragma unroll
          for (int i = 0; i < KP; ++i) {
            const uint4 kv = lds128(sk + piece_off<RB>(tok, c + 4 * i));
            const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
            if constexpr (E4M3) {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                uint4 qv;
                if constexpr (kQShared) qv = q_frag[(4 * i + x) * 32 + lane];
                else qv = make_uint4(qf[4 * i + x][0], qf[4 * i + x][1], qf[4 * i + x][2], qf[4 * i + x][3]);
                mma_16816<true>(s[n], qv.x, qv.y, qv.z, qv.w, codes_f16x2(w[x]), codes_f16x2(w[x] >> 16));
              }
            } else {
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                uint4 qv;
                if constexpr (kQShared) qv = q_frag[(2 * i + x) * 32 + lane];
                else qv = make_uint4(qf[2 * i + x][0], qf[2 * i + x][1], qf[2 * i + x][2], qf[2 * i + x][3]);
                mma_16816<false>(s[n], qv.x, qv.y, qv.z, qv.w, w[2 * x], w[2 * x + 1]);
              }
            }
          }
        }
        // ---- scores, what the rows see, running maximum ----
        const bool edge = tok0 + 16 > clear;                  // rows see different tokens, or some are behind the end
        bool see[2][4];
        float ev[2][2];                                       // (8-bit) exponents of this lane's value rows, tokens c and c + 4
        float mx[2] = {-INFINITY, -INFINITY}, wx[2] = {-INFINITY, -INFINITY};
        const uint32_t ss = smem_u32(scales + stage * Cfg::kScaleBytes) + wtok;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            const int off = n * 8 + h2 * 4 + c, j = tok0 + off;
            float kscale = 1.f;
            if constexpr (E4M3) {
              kscale = __uint_as_float(lds8(ss + off) << 23);
              ev[n][h2] = (float)((int)lds8(ss + kTile + off) - 127);
            }
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              float& x = s[n][hh * 2 + h2];
              x *= f_row[hh] * kscale;
              bool ok = true;
              if (edge) {
                ok = (hh ? rB : rA) < valid && sees(j, hh ? posB : posA, hh ? maskB : maskA);
                if (!ok) x = -INFINITY;
              }
              see[n][hh * 2 + h2] = ok;
              mx[hh] = fmaxf(mx[hh], x);
              if constexpr (E4M3) wx[hh] = fmaxf(wx[hh], x + ev[n][h2]);
            }
          }
        }
        float p[2][4];
        float corr[2];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          mx[hh] = fmaxf(mx[hh], __shfl_xor_sync(0xffffffffu, mx[hh], 1));
          mx[hh] = fmaxf(mx[hh], __shfl_xor_sync(0xffffffffu, mx[hh], 2));
          const float m = fmaxf(m_run[hh], mx[hh]), mu = m == -INFINITY ? 0.f : m;
          corr[hh] = exp2f(m_run[hh] - mu);
          l_run[hh] *= corr[hh];
          float cf = 1.f;                                     // 2^-c of the weights of this tile
          if constexpr (E4M3) {
            wx[hh] = fmaxf(wx[hh], __shfl_xor_sync(0xffffffffu, wx[hh], 1));
            wx[hh] = fmaxf(wx[hh], __shfl_xor_sync(0xffffffffu, wx[hh], 2));
            w_run[hh] = fmaxf(w_run[hh], wx[hh]);
            // both maxima are running ones, so c never lets a weight above 1
            const float cw = ceilf(w_run[hh] - mu);
            const int cn = cw > -120.f ? (int)fminf(cw, 120.f) : -120;
            if (c_run[hh] != -1000) corr[hh] *= pow2i(c_run[hh] - cn);
            c_run[hh] = cn;
            cf = pow2i(-cn);
          }
          m_run[hh] = m;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int h2 = 0; h2 < 2; ++h2) {
              const float e = exp2f(s[n][hh * 2 + h2] - mu);
              l_run[hh] += e;
              if constexpr (E4M3) p[n][hh * 2 + h2] = e * pow2i((int)ev[n][h2]) * cf;
              else p[n][hh * 2 + h2] = e;
            }
        }
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            o[i][0] *= corr[0]; o[i][1] *= corr[0]; o[i][2] *= corr[1]; o[i][3] *= corr[1];
          }
        }
        uint32_t pa[4];
        if constexpr (E4M3) {
          pa[0] = pack_f16x2(p[0][0], p[0][1]); pa[1] = pack_f16x2(p[0][2], p[0][3]);
          pa[2] = pack_f16x2(p[1][0], p[1][1]); pa[3] = pack_f16x2(p[1][2], p[1][3]);
        } else {
          pa[0] = pack_bf16x2(p[0][0], p[0][1]); pa[1] = pack_bf16x2(p[0][2], p[0][3]);
          pa[2] = pack_bf16x2(p[1][0], p[1][1]); pa[3] = pack_bf16x2(p[1][2], p[1][3]);
        }
        // ---- O += P V: the lane's k indices are tokens c, c + 4, 8 + c, 12 + c; its columns g * D / 8 onward. Which of a pair of
        // tokens is loaded first is chosen by the lane so that a phase's 8 lanes hit different columns of the swizzle. ----
        constexpr int VP = VB >= 16 ? VB / 16 : 1;            // loads per token
        const int swap = RB == 64 ? (c >> 1) & 1 : (RB == 512 ? 0 : g & 1);
#pragma unroll
        for (int h = 0; h < VP; ++h) {
          uint32_t v[2][2][4];                                // [n][first, second][words]
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int tok = wtok + n * 8 + c + 4 * (x ^ swap);
              if constexpr (VB >= 16) {
                const uint4 w = lds128(sv + piece_off<RB>(tok, g * VP + h));
                v[n][x][0] = w.x; v[n][x][1] = w.y; v[n][x][2] = w.z; v[n][x][3] = w.w;
              } else {
                const uint2 w = lds64(sv + piece_off<RB>(tok, g >> 1) + (g & 1) * 8);
                v[n][x][0] = w.x; v[n][x][1] = w.y; v[n][x][2] = 0; v[n][x][3] = 0;
              }
              if (edge && tok0 - wtok + tok >= L) v[n][x][0] = v[n][x][1] = v[n][x][2] = v[n][x][3] = 0;
            }
          constexpr int W = VB >= 16 ? 4 : 2;                 // words per load
          // columns of one word: their operand pairs (first token low)
          auto column = [&](int w, int col, uint32_t& b0, uint32_t& b1) {
            if constexpr (E4M3) {
              const uint32_t sel = col < 2 ? (swap ? 0x1504u : 0x5140u) : (swap ? 0x3726u : 0x7362u);
              b0 = codes_f16x2(__byte_perm(v[0][0][w], v[0][1][w], sel) >> ((col & 1) * 16));
              b1 = codes_f16x2(__byte_perm(v[1][0][w], v[1][1][w], sel) >> ((col & 1) * 16));
            } else {
              const uint32_t sel = col == 0 ? (swap ? 0x1054u : 0x5410u) : (swap ? 0x3276u : 0x7632u);
              b0 = __byte_perm(v[0][0][w], v[0][1][w], sel);
              b1 = __byte_perm(v[1][0][w], v[1][1][w], sel);
            }
          };
          constexpr int CW = E4M3 ? 4 : 2;                    // columns per word
          if (!edge) {
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
              for (int col = 0; col < CW; ++col) {
                uint32_t b0, b1;
                column(w, col, b0, b1);
                mma_16816<E4M3>(o[h * W * CW + w * CW + col], pa[0], pa[1], pa[2], pa[3], b0, b1);
              }
          } else {
            constexpr uint32_t one = E4M3 ? 0x3c003c00u : 0x3f803f80u;
            auto half_one = [](bool lo, bool hi) { return (lo ? (one & 0xffffu) : 0u) | (hi ? (one & 0xffff0000u) : 0u); };
            const uint32_t a0 = half_one(see[0][0], see[0][1]), a1 = half_one(see[0][2], see[0][3]);
            const uint32_t a2 = half_one(see[1][0], see[1][1]), a3 = half_one(see[1][2], see[1][3]);
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
              for (int col = 0; col < CW; ++col) {
                uint32_t b0, b1;
                column(w, col, b0, b1);
                float (&oo)[4] = o[h * W * CW + w * CW + col];
                const uint32_t n0 = not_finite<E4M3>(b0), n1 = not_finite<E4M3>(b1);
                if (__any_sync(0xffffffffu, (n0 | n1) != 0)) {
                  // rows that see an infinity or a NaN here get it back: counts of those that pull up (+inf, NaN) and down
                  constexpr uint32_t inf = E4M3 ? 0x7c00u : 0x7f80u;
                  auto pulls = [](uint32_t w16, bool bad, uint32_t towards) { return bad && (w16 == towards || (w16 & 0x7fffu) > inf); };
                  const uint32_t up0 = half_one(pulls(b0 & 0xffffu, n0 & 1u, inf), pulls(b0 >> 16, n0 >> 16, inf));
                  const uint32_t up1 = half_one(pulls(b1 & 0xffffu, n1 & 1u, inf), pulls(b1 >> 16, n1 >> 16, inf));
                  const uint32_t dn0 = half_one(pulls(b0 & 0xffffu, n0 & 1u, inf | 0x8000u), pulls(b0 >> 16, n0 >> 16, inf | 0x8000u));
                  const uint32_t dn1 = half_one(pulls(b1 & 0xffffu, n1 & 1u, inf | 0x8000u), pulls(b1 >> 16, n1 >> 16, inf | 0x8000u));
                  float up[4] = {0.f, 0.f, 0.f, 0.f}, dn[4] = {0.f, 0.f, 0.f, 0.f};
                  mma_16816<E4M3>(up, a0, a1, a2, a3, up0, up1);
                  mma_16816<E4M3>(dn, a0, a1, a2, a3, dn0, dn1);
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    if (up[x] > 0.f) oo[x] += INFINITY;
                    if (dn[x] > 0.f) oo[x] -= INFINITY;
                  }
                }
                mma_16816<E4M3>(oo, pa[0], pa[1], pa[2], pa[3], b0 & ~n0, b1 & ~n1);
              }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[stage]);
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 1);
      l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 2);
    }
    if constexpr (E4M3) {
      const float fa = c_run[0] == -1000 ? 1.f : pow2i(c_run[0]), fb = c_run[1] == -1000 ? 1.f : pow2i(c_run[1]);
#pragma unroll
      for (int i = 0; i < NC; ++i) { o[i][0] *= fa; o[i][1] *= fa; o[i][2] *= fb; o[i][3] *= fb; }
    }
  }

  // ---------------- the four warps' parts are joined: rows of floats in the ring's memory ----------------
  pdl_launch_dependents();
  __syncthreads();
  if (*abort_flag != 0) {
    const uint64_t t0 = globaltimer_ns();       // let copies in flight land before the memory is used again or goes away
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    return;
  }
  constexpr int kPad = D + 4;
  float* mo = reinterpret_cast<float*>(stages);               // [4][16][D + 4]
  float* mm = mo + 4 * 16 * kPad;                             // [4][16] maxima
  float* ml = mm + 64;                                        // [4][16] sums
  if (warp < 4) {
    if (c == 0) {
      mm[warp * 16 + rA] = m_run[0]; mm[warp * 16 + rB] = m_run[1];
      ml[warp * 16 + rA] = l_run[0]; ml[warp * 16 + rB] = l_run[1];
    }
    // the lane's columns: two runs of D / 8, from 2 c D / 8 and (2 c + 1) D / 8
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int par = 0; par < 2; ++par)
#pragma unroll
        for (int i = 0; i < NC; i += 4)
          *reinterpret_cast<float4*>(mo + (warp * 16 + (hh ? rB : rA)) * kPad + (2 * c + par) * NC + i) =
              make_float4(o[i][hh * 2 + par], o[i + 1][hh * 2 + par], o[i + 2][hh * 2 + par], o[i + 3][hh * 2 + par]);
  }
  __syncthreads();
  const bool whole = shares == 1;
  for (int i = threadIdx.x; i < valid * (D / 8); i += kRowsThreads) {
    const int r = i / (D / 8), col = (i % (D / 8)) * 8;
    const float m0 = mm[r], m1 = mm[16 + r], m2 = mm[32 + r], m3 = mm[48 + r];
    const float m = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), mu = m == -INFINITY ? 0.f : m;
    float f[4] = {exp2f(m0 - mu), exp2f(m1 - mu), exp2f(m2 - mu), exp2f(m3 - mu)};
    float l = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (mm[w * 16 + r] == -INFINITY && ml[w * 16 + r] == 0.f) continue;       // a warp that saw nothing of this row
      l += f[w] * ml[w * 16 + r];
      const float* src = mo + (w * 16 + r) * kPad + col;
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] += f[w] * src[k];
    }
    const int tk = row0 + tok_lo + r / G, head = kvh * G + r % G;
    if (whole) {
      const float inv = l == 0.f ? 0.f : 1.f / l;             // a row that sees nothing: zeros
      *reinterpret_cast<uint4*>(a.out + (size_t)tk * a.out_stride + (size_t)head * D + col) =
          make_uint4(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv), pack_bf16x2(x[4] * inv, x[5] * inv),
                     pack_bf16x2(x[6] * inv, x[7] * inv));
    } else {
      const size_t at = ((size_t)tk * a.hq + head) * a.splits + split;
      float4* dst = reinterpret_cast<float4*>(a.ws_o + at * D + col);
      dst[0] = make_float4(x[0], x[1], x[2], x[3]);
      dst[1] = make_float4(x[4], x[5], x[6], x[7]);
      if (col == 0) {
        a.ws_ml[at * 2] = m;
        a.ws_ml[at * 2 + 1] = l;
      }
    }
  }
}

// Joins the shares of every row that was cut: a warp per (row, head), D / 32 columns a lane. grid (ceil(max_rows * hq / 8), seqs).
template <int D, bool TREE>
KERN_DEVICE void rows_merge(const float* ws_o, const float* ws_ml, __nv_bfloat16* out, const int* seq_lens, const int* cu_q, int rows_per_seq,
                            int hq, int hk, int splits, int out_stride) {
  pdl_wait();
  const int lane = threadIdx.x & 31, seq = blockIdx.y;
  const int at = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int row0 = cu_q ? cu_q[seq] : seq * rows_per_seq, R = cu_q ? cu_q[seq + 1] - row0 : rows_per_seq;
  const int tok = at / hq, head = at % hq;
  if (tok >= R) return;
  const int L = max(seq_lens[seq], 0), G = hq / hk, toks = 16 / G > 0 ? 16 / G : 1;
  const int lo = tok / toks * toks;
  const int end = TREE ? L : max(0, L - R + lo + min(toks, R - lo));
  const int shares = rows_shares((end + kTile - 1) / kTile, splits);
  if (shares == 1) return;                                    // written by its one CTA
  const size_t base = ((size_t)(row0 + tok) * hq + head) * splits;
  float m = -INFINITY;
  for (int s = 0; s < shares; ++s) m = fmaxf(m, ws_ml[(base + s) * 2]);
  const float mu = m == -INFINITY ? 0.f : m;
  constexpr int N = D / 32;
  float x[N], l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < shares; ++s) {
    const float ms = ws_ml[(base + s) * 2], ls = ws_ml[(base + s) * 2 + 1];
    if (ms == -INFINITY && ls == 0.f) continue;
    const float f = exp2f(ms - mu);
    l += f * ls;
    const float* src = ws_o + (base + s) * D + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += f * src[i];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = out + (size_t)(row0 + tok) * out_stride + (size_t)head * D + lane * N;
#pragma unroll
  for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16x2(x[i] * inv, x[i + 1] * inv);
}

}  // namespace kern

using namespace kern;

#define KERN_ROWS_ENTRY(D, KIND, E4M3, FORM, TREE)                                                                                \
  extern "C" __global__ void __launch_bounds__(kRowsThreads, D == 256 ? 1 : 2) kern_attn_rows_##KIND##_##FORM##_d##D(             \
      const __grid_constant__ CUtensorMap kv_map, const __nv_bfloat16* q, __nv_bfloat16* out, float* ws_o, float* ws_ml,          \
      const uint8_t* pool, const int* block_table, const int* seq_lens, const int* cu_q, const long long* masks, int words,       \
      int rows_per_seq, int hq, int hk, int q_stride, int out_stride, int max_pages, int page_size, int splits, int pool_pages,   \
      float scale_log2, int* err) {                                                                                               \
    rows_body<D, E4M3, TREE>(&kv_map, RowsArgs{q, out, ws_o, ws_ml, pool, block_table, seq_lens, cu_q, masks, err, words,         \
                                               rows_per_seq, hq, hk, q_stride, out_stride, max_pages, page_size, splits,          \
                                               pool_pages, scale_log2});                                                          \
  }
#define KERN_ROWS_MERGE(D, FORM, TREE)                                                                                            \
  extern "C" __global__ void __launch_bounds__(256) kern_attn_rows_merge_##FORM##_d##D(                                           \
      const float* ws_o, const float* ws_ml, __nv_bfloat16* out, const int* seq_lens, const int* cu_q, int rows_per_seq, int hq,  \
      int hk, int splits, int out_stride) {                                                                                       \
    rows_merge<D, TREE>(ws_o, ws_ml, out, seq_lens, cu_q, rows_per_seq, hq, hk, splits, out_stride);                              \
  }
#define KERN_ROWS(D)                           \
  KERN_ROWS_ENTRY(D, e4m3, true, causal, false) \
  KERN_ROWS_ENTRY(D, e4m3, true, tree, true)    \
  KERN_ROWS_ENTRY(D, bf16, false, tree, true)   \
  KERN_ROWS_MERGE(D, causal, false)             \
  KERN_ROWS_MERGE(D, tree, true)
KERN_ROWS(64)
KERN_ROWS(128)
KERN_ROWS(256)
