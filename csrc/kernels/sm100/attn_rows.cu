// Attention of few query rows over a paged cache, bf16 or e4m3 (kv_e4m3.cu has the 8-bit layout): single tokens, short causal
// blocks, and trees of drafted tokens, in which a row sees the whole context before the tree and those nodes of it whose bit its
// mask has.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^(scale log2(e) q_i.k_j - m_i)  over the j that row i sees; no such j: zeros
//
// One CTA = (8 or 16 query rows: the G heads of some tokens, one kv head, a share of the context). A producer warp brings
// tiles of tokens into a ring of shared memory by TMA; four warps take 16 tokens of a tile at a time and keep (m, l, O) of
// their own. They are joined at the end, then the shares of one row: over distributed shared memory in a cluster of up to 8 CTAs, and
// where that is not enough as partials that a second kernel joins (kern_attn_rows_merge).
//
// The time goes to reading the cache, so a byte of it may cost few instructions. Products are turned around: S^T = K Q^T and
// O^T = V^T P^T on mma.sync, so that the 16-row operand is the cache and the 8-column one the query rows, of which a single token
// has 4 or 8. The order of the contraction index and of the operand rows inside a fragment is free as long as both operands agree,
// so a lane takes whole 16-byte pieces of key and value rows from shared memory and nothing is moved again: of a value row's
// pieces it pairs two tokens' bytes with PRMT, and P^T comes from S^T by movmatrix. The same code serves bf16 words and e4m3
// bytes, which become f16 pairs, exactly, in one instruction (cvt.rn.f16x2.e4m3x2). Tokens are dealt to lanes so that the 8 lanes
// of a shared-memory phase hit 8 different 16-byte columns of the swizzle. The references m (and R below) move only when a weight
// has outgrown them by 2^15: most tiles need no maximum over lanes and no pass over O.
//
// 8-bit: Q goes to f16 with its row's power of two taken out; the scores of a key row are multiplied by its scale in f32; a value
// row's scale goes into its weight, w_ij = 2^(s_ij + e_j - R_i). R follows the largest s_ij + e_j seen, less 7, so the largest weight
// of a row is between 2^6 and 2^15 whatever the sizes of the value rows, and every weight down to 2^-20 of it keeps all of f16's
// bits. Rounding a weight to f16 (2^-11) is three bits finer than the output's own rounding; bf16 caches take bf16 weights (2^-8 of
// each weight, as the value rows' own rounding), and their sum is of the rounded weights: a row that looks at a few keys then is off by
// 0.0018 in the mean where the exact sum gave 0.0024, the output's own rounding included.
//
// Values that a row does not see do not reach it, whatever they are: tokens behind the end are cleared, and in the tiles where
// rows see different tokens values that are not finite are taken out of the product and put back for the rows that see them (a
// second pass of products over 0 / 1, only when there are any).
//
// Measured (8-bit, 8 kv heads, 32 heads of 128): single tokens of 64 sequences of up to 4096 tokens 51 us, 0.88 of the measured copy
// bandwidth, of 128 sequences of up to 8000 168 us, 0.97; 2 sequences of 100,003 40 us, 0.74; one of 1001 8 us, which is launch,
// one round to DRAM and the join.
#include "attn_rows.cuh"

namespace kern {

// D, cache format, NT: columns of query rows in eights
template <int D, bool E4M3, int NT>
struct RowsCfg {
  static constexpr int kRowBytes = D * (E4M3 ? 1 : 2);
  static constexpr int kTile = kRowBytes <= 128 ? 128 : 64;          // tokens: a stage of 32 KB where rows allow it
  static constexpr int kHalf = kTile * kRowBytes;                    // a tile of K or of V
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kScaleBytes = E4M3 ? 2 * kTile : 0;
  // 96 KB of ring, so that two CTAs share an SM; one where 512-byte rows and their accumulators take the room of two
  static constexpr int kPerSm = D == 256 ? 1 : 2;
  static constexpr int kStages = kStage >= 65536 ? 3 : (kPerSm == 1 ? 196608 : 98304) / kStage;
  static constexpr int kBox = kRowBytes < 128 ? kRowBytes : 128;     // bytes of a row in one box
  // warps of products, 16 tokens of a tile at a time each (eight of them, at 96 registers, were 15 % slower: 75 us against 66 for
  // 64 sequences of up to 4096 tokens)
  static constexpr int kWarps = 4;
  static constexpr int kThreads = 32 * (kWarps + 1);                 // and a producer
  static constexpr bool kQShared = D == 256 && NT > 1;               // Q's fragments in shared memory: registers do not hold them
  static constexpr int kQBytes = kQShared ? NT * (D / 16) * 32 * 8 : 0;
};

// byte offset of (token, 16-byte piece) in a tile of RB-byte rows stored as 128-byte column blocks with the TMA's swizzle
template <int RB, int TILE>
KERN_DEVICE uint32_t piece_off(int tok, int piece) {
  if constexpr (RB == 64) {
    return (uint32_t)(tok * 64 + ((piece ^ ((tok >> 1) & 3)) << 4));
  } else {
    return (uint32_t)((piece >> 3) * (TILE * 128) + tok * 128 + (((piece & 7) ^ (tok & 7)) << 4));
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
// the 8 x 8 matrix of 16-bit values whose row lane / 4, columns 2 (lane % 4) and + 1 each lane holds, transposed
KERN_DEVICE uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// 4 bytes global -> shared, and an arrival on `bar` once this lane's copies so far have landed (counted by the barrier's setting)
KERN_DEVICE void async_copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
KERN_DEVICE void async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// clusters: the same place in another CTA's shared memory, and a barrier over the CTAs that orders what they wrote there
KERN_DEVICE uint32_t at_rank(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
KERN_DEVICE float ld_rank(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
KERN_DEVICE float4 ld_rank4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
KERN_DEVICE void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int D, bool E4M3, bool TREE, int NT>
KERN_DEVICE void rows_body(const CUtensorMap* kv_map, const RowsArgs& a) {
  using Cfg = RowsCfg<D, E4M3, NT>;
  constexpr int RB = Cfg::kRowBytes, kStages = Cfg::kStages, kTile = Cfg::kTile;
  constexpr int KP = RB / 64;              // 16-byte pieces of a key row per lane
  constexpr int VB = RB / 8;               // bytes of a value row per lane: D / 8 columns
  constexpr int MI = D / 16;               // 16-row tiles of O^T
  constexpr int KS = D / 16;               // k-steps of K Q^T
  constexpr int kRows = 8 * NT, kWarps = Cfg::kWarps, kThreads = Cfg::kThreads;
  constexpr bool kQShared = Cfg::kQShared;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stages = smem;
  uint8_t* scales = smem + kStages * Cfg::kStage;
  uint2* q_frag = reinterpret_cast<uint2*>(scales + kStages * Cfg::kScaleBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(q_frag) + Cfg::kQBytes);
  uint64_t* empty_bar = full_bar + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty_bar + kStages);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.hq / a.hk;
  const int blk = blockIdx.x / a.hk, kvh = blockIdx.x % a.hk;
  int seq = blockIdx.y;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], E4M3 ? 33 : 1);
      mbar_init(&empty_bar[s], kWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(kv_map);
  }
  pdl_wait();
  if (gridDim.z == 1 && gridDim.y <= kThreads && gridDim.x * gridDim.y > sm_count() * Cfg::kPerSm) {
    // more blocks than run at once: block y takes the sequence of rank y by length, so that the last to start are the shortest
    volatile int* found = abort_flag + 1;
    if (by_length(a.seq_lens, gridDim.y, reinterpret_cast<int*>(stages)) == seq) *found = threadIdx.x;
    fence_proxy_async();                                      // (copies come to the same place)
    __syncthreads();
    seq = *found;
  } else {
    __syncthreads();
  }

  const int L = context_of(a, seq);
  const int row0 = a.cu_q ? a.cu_q[seq] : seq * a.rows_per_seq;
  const int R = a.cu_q ? a.cu_q[seq + 1] - row0 : a.rows_per_seq;
  const int toks = kRows / G;
  const int tok_lo = blk * toks;
  if (tok_lo >= R || R < a.row_lo || R > a.row_hi) return;   // uniform over the cluster
  if (!rows_lie(row0, R, a.rows, a.max_rows)) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BOUNDS);
    return;
  }
  const int valid = min(toks, R - tok_lo) * G;
  const int past = L - R;                                    // what the sequence had before this call's rows
  // causal: the last row of the block decides how far the walk goes
  const int end = TREE ? L : max(0, past + tok_lo + min(toks, R - tok_lo));
  const int shares = rows_shares(end, gridDim.z);
  const int share_len = rows_share_len(end, shares);
  const int from = min(end, (int)blockIdx.z * share_len), to = (int)blockIdx.z < shares ? min(end, from + share_len) : from;
  const int ntiles = (to - from + kTile - 1) / kTile;

  const int g = lane >> 2, c = lane & 3;
  // of columns (query rows) 8 nt + 2 c + x; g = 2^(m - R)
  float l_run[NT][2], m_run[NT][2], r_run[NT][2], g_run[NT][2];
  float o[NT][MI][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l_run[nt][x] = 0.f;
      m_run[nt][x] = r_run[nt][x] = kUnset;
      g_run[nt][x] = 1.f;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
  }

  if (warp == kWarps) {
    // ---------------- producer ----------------
    const int box = a.page_size < 64 ? a.page_size : 64, box_bits = 31 - __clz(box);
    const int* pages = a.block_table + (size_t)seq * a.max_pages;
    // (page of the table, row in it) of the tile's first token; the table is read 32 pages at a time, a lane each
    int pi0 = from / a.page_size, off0 = from - pi0 * a.page_size, first = pi0 - 32, id = 0;
    int stage = 0;
    uint32_t phase = 0;
    for (int t = 0; t < ntiles; ++t) {
      const int here = min(kTile, to - (from + t * kTile));
      const int boxes = (here + box - 1) >> box_bits;
      if (pi0 + (kTile >> 3) > first + 32) {                  // (a tile has 16 pages at most)
        first = pi0;
        const int pi = first + lane;
        id = pi < a.max_pages ? pages[pi] : -1;
        if (id < 0 || id >= a.pool_pages) {
          if (pi * a.page_size < to) set_error(a.err, ERR_BOUNDS);
          id = 0;
        }
      }
      // box b of the tile
      auto place = [&](int b, int& pi, int& off) {
        pi = pi0;
        off = off0 + (b << box_bits);
        if (box == a.page_size) {
          pi += b;
          off = 0;
        } else if (off >= a.page_size) {                      // (pages of 64 tokens and more: two to a tile at most)
          ++pi;
          off -= a.page_size;
        }
      };
      if (!bar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) {
        set_error(a.err, ERR_WAIT_EMPTY);
        *abort_flag = 1;
        break;
      }
      uint8_t* sk = stages + stage * Cfg::kStage;
      // boxes behind the share's end are not brought: their tokens are masked and their values cleared
      if (lane == 0) mbar_expect_tx(&full_bar[stage], boxes * box * RB * 2);
      __syncwarp();
      {
        int pi, off;
        place(lane >> 1, pi, off);
        const int page = __shfl_sync(0xffffffffu, id, (pi - first) & 31);
        const int b = lane >> 1, which = lane & 1;            // a lane to each box of K and of V
        if (b < boxes) {
#pragma unroll
          for (int cb = 0; cb < RB / Cfg::kBox; ++cb)
            tma_load_3d(sk + which * Cfg::kHalf + cb * (kTile * 128) + (b << box_bits) * Cfg::kBox, kv_map, cb * (Cfg::kBox * D / RB),
                        (which * a.hk + kvh) * a.page_size + off, page, &full_bar[stage]);
        }
      }
      if constexpr (E4M3) {
        const size_t codes = (size_t)2 * a.hk * a.page_size * D;
#pragma unroll
        for (int i = 0; i < 2 * (kTile / 4); i += 32) {
          const int which = (i + lane) / (kTile / 4), i4 = ((i + lane) % (kTile / 4)) * 4;
          int pi, off;
          place(i4 >> box_bits, pi, off);
          const int page = __shfl_sync(0xffffffffu, id, (pi - first) & 31);
          if (i4 < here) {
            const uint8_t* src = a.pool + (size_t)page * (codes + 2 * a.hk * a.page_size) + codes + (size_t)(which * a.hk + kvh) * a.page_size + off + (i4 & (box - 1));
            if (KERN_CHECK(src, 4, SITE_KV_ROW)) async_copy4(smem_u32(scales + stage * Cfg::kScaleBytes + which * kTile + i4), src);
          }
        }
        async_arrive(&full_bar[stage]);
      }
      if (box == a.page_size) {
        pi0 += kTile >> box_bits;
      } else {
        off0 += kTile;
        while (off0 >= a.page_size) {
          off0 -= a.page_size;
          ++pi0;
        }
      }
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
  } else {
    // ---------------- Q's fragments, in the order in which a lane holds the keys ----------------
    uint32_t qf[NT][KS][2];
    float f_col[NT][2];                                      // what turns a column's products into base-2 scores
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + g;
      const bool ok = r < valid;
      const __nv_bfloat16* src = a.q + (size_t)(row0 + tok_lo + (ok ? r / G : 0)) * a.q_stride + (size_t)(kvh * G + (ok ? r % G : 0)) * D;
      float f = a.scale_log2;
      if constexpr (E4M3) {
        // 16 values to a piece: word w of the piece makes k-step 4 i + w
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < KP; ++i)
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            const uint4 v = ok ? *reinterpret_cast<const uint4*>(src + (c + 4 * i) * 16 + h2 * 8) : make_uint4(0, 0, 0, 0);
            qf[nt][4 * i + 2 * h2][0] = v.x;
            qf[nt][4 * i + 2 * h2][1] = v.y;
            qf[nt][4 * i + 2 * h2 + 1][0] = v.z;
            qf[nt][4 * i + 2 * h2 + 1][1] = v.w;
          }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const float2 u = unpack_bf16x2(qf[nt][s][0]), v = unpack_bf16x2(qf[nt][s][1]);
          top = fmaxf(top, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(v.x), fabsf(v.y))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int x = min(max((int)((__float_as_uint(top) >> 23) & 255) - 127, -100), 100);
        const float inv = pow2i(-x);
        f *= pow2i(x);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const float2 u = unpack_bf16x2(qf[nt][s][0]), v = unpack_bf16x2(qf[nt][s][1]);
          qf[nt][s][0] = pack_f16x2(u.x * inv, u.y * inv);
          qf[nt][s][1] = pack_f16x2(v.x * inv, v.y * inv);
        }
      } else {
        // 8 values to a piece: its words make k-steps 2 i and 2 i + 1
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          const uint4 v = ok ? *reinterpret_cast<const uint4*>(src + (c + 4 * i) * 8) : make_uint4(0, 0, 0, 0);
          qf[nt][2 * i][0] = v.x;
          qf[nt][2 * i][1] = v.y;
          qf[nt][2 * i + 1][0] = v.z;
          qf[nt][2 * i + 1][1] = v.w;
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) f_col[nt][x] = __shfl_sync(0xffffffffu, f, (2 * c + x) * 4);
      if constexpr (kQShared) {
        // (the warps write the same values)
#pragma unroll
        for (int s = 0; s < KS; ++s) q_frag[(nt * KS + s) * 32 + lane] = make_uint2(qf[nt][s][0], qf[nt][s][1]);
      }
    }
    __syncwarp();

    // ---------------- products ----------------
    // whether column r of this block sees token j
    auto sees = [&](int j, int r) -> bool {
      if (r >= valid || j >= to) return false;
      const int tk = tok_lo + r / G;
      if constexpr (TREE) {
        if (j < past) return true;
        const int n = j - past;
        return n < a.words * 64 && ((a.masks[(size_t)(row0 + tk) * a.words + (n >> 6)] >> (n & 63)) & 1);
      } else {
        return j <= past + tk;
      }
    };
    // the first token that some row of the block may not see
    const int clear = min(to, TREE ? past : past + tok_lo + 1);
    const int pg = (g & 1) << 2 | (g >> 1);                   // the key row of operand row g: 0, 4, 1, 5, 2, 6, 3, 7
    // of a pair of value rows, which is loaded first: chosen so that a phase's 8 lanes hit different columns of the swizzle
    const int swap = RB == 64 ? (c >> 1) & 1 : (RB == 512 ? 0 : g & 1);
    int stage = 0;
    uint32_t phase = 0;
    for (int t = 0; t < ntiles; ++t) {
      if (!bar_wait(&full_bar[stage], phase, abort_flag)) {
        set_error(a.err, ERR_WAIT_FULL);
        *abort_flag = 1;
        break;
      }
      const uint32_t sk = smem_u32(stages + stage * Cfg::kStage), sv = sk + Cfg::kHalf;
#pragma unroll 1
      for (int part = 0; part < kTile / (16 * kWarps); ++part) {
        const int wtok = (part * kWarps + warp) * 16;               // this warp's 16 tokens of the tile
        const int tok0 = from + t * kTile + wtok;
        if (tok0 >= to) break;
        // ---- S^T = K Q^T: operand rows g and g + 8 are tokens pg and 8 + pg, so that neighbouring rows of a load differ in the
        // bit of the swizzle that a row's own pieces do not reach ----
        float s[NT][4], s2[NT][4];                            // two chains of sums: one would be D / 16 dependent products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[nt][k] = s2[nt][k] = 0.f;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          const uint4 ka = lds128(sk + piece_off<RB, kTile>(wtok + pg, c + 4 * i)), kb = lds128(sk + piece_off<RB, kTile>(wtok + 8 + pg, c + 4 * i));
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
          constexpr int steps = E4M3 ? 4 : 2;
#pragma unroll
          for (int x = 0; x < steps; ++x) {
            uint32_t a0, a1, a2, a3;
            if constexpr (E4M3) {
              codes_f16x4(wa[x], a0, a2);
              codes_f16x4(wb[x], a1, a3);
            } else {
              a0 = wa[2 * x]; a2 = wa[2 * x + 1];
              a1 = wb[2 * x]; a3 = wb[2 * x + 1];
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int ks = steps * i + x;
              uint2 qv;
              if constexpr (kQShared) qv = q_frag[(nt * KS + ks) * 32 + lane];
              else qv = make_uint2(qf[nt][ks][0], qf[nt][ks][1]);
              mma_16816<E4M3>(x & 1 ? s2[nt] : s[nt], a0, a1, a2, a3, qv.x, qv.y);
            }
          }
        }
        // ---- scores of tokens pg and 8 + pg, columns 8 nt + 2 c + x ----
        const bool edge = tok0 + 16 > clear;                  // rows see different tokens, or some are behind the end
        float kscale[2] = {1.f, 1.f}, vscale[2] = {1.f, 1.f};
        if constexpr (E4M3) {
          const uint32_t ss = smem_u32(scales + stage * Cfg::kScaleBytes) + wtok + pg;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            kscale[h] = __uint_as_float(lds8(ss + 8 * h) << 23);
            vscale[h] = __uint_as_float(lds8(ss + kTile + 8 * h) << 23);
          }
        }
        uint32_t see = 0xffffffffu;                           // bit nt * 4 + h * 2 + x
        if (edge) {
          see = 0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const bool ok = sees(tok0 + pg + 8 * (k >> 1), nt * 8 + 2 * c + (k & 1));
              see |= (ok ? 1u : 0u) << (nt * 4 + k);
            }
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (tok0 + pg + 8 * h >= to) kscale[h] = vscale[h] = 1.f;      // (not brought: anything may lie there)
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // (one factor after the other: together they may pass f32's range where a product is 0)
            s[nt][k] = (s[nt][k] + s2[nt][k]) * f_col[nt][k & 1] * kscale[k >> 1];
            if (edge && !(see >> (nt * 4 + k) & 1)) s[nt][k] = -INFINITY;
          }
        float e[NT][4], w[NT][4];
        auto weigh = [&]() {
          float top = 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              e[nt][k] = exp2f(s[nt][k] - m_run[nt][k & 1]);
              top = fmaxf(top, e[nt][k]);
              if constexpr (E4M3) {
                w[nt][k] = e[nt][k] * fminf(g_run[nt][k & 1] * vscale[k >> 1], 3e38f);     // (0 stays 0 beside the largest scales)
                top = fmaxf(top, w[nt][k]);
              } else {
                w[nt][k] = e[nt][k];
              }
            }
          return top;
        };
        if (__any_sync(0xffffffffu, weigh() > kOutgrown)) {
          // a reference moves to its column's maximum (rounded up: factors stay powers of two), and what it scaled with it
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float mx = fmaxf(s[nt][x], s[nt][2 + x]), rx = mx;
              if constexpr (E4M3)
                rx = fmaxf(s[nt][x] + (float)(max((int)(__float_as_uint(vscale[0]) >> 23), kLeastScale) - 127),
                           s[nt][2 + x] + (float)(max((int)(__float_as_uint(vscale[1]) >> 23), kLeastScale) - 127));
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                if constexpr (E4M3) rx = fmaxf(rx, __shfl_xor_sync(0xffffffffu, rx, d));
              }
              const float m = fmaxf(m_run[nt][x], ceilf(mx));
              float co = exp2f(m_run[nt][x] - m);
              l_run[nt][x] *= co;
              m_run[nt][x] = m;
              if constexpr (E4M3) {
                const float r = fmaxf(r_run[nt][x], ceilf(rx) - 7.f);
                co = exp2f(r_run[nt][x] - r);
                r_run[nt][x] = r;
                g_run[nt][x] = exp2f(m - r);
              }
#pragma unroll
              for (int i = 0; i < MI; ++i) {
                o[nt][i][x] *= co;
                o[nt][i][2 + x] *= co;
              }
            }
          weigh();
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            pb[nt][h] = pack_pair<E4M3>(w[nt][2 * h], w[nt][2 * h + 1]);
            // (bf16 weights are summed as the products take them: the rounding of a row's largest falls out of the quotient)
            l_run[nt][0] += E4M3 ? e[nt][2 * h] : __uint_as_float(pb[nt][h] << 16);
            l_run[nt][1] += E4M3 ? e[nt][2 * h + 1] : __uint_as_float(pb[nt][h] & 0xffff0000u);
            pb[nt][h] = transposed(pb[nt][h]);
          }
        // ---- O^T += V^T P^T: the lane's contraction indices are tokens c, c + 4, 8 + c, 12 + c; its channels g * D / 8 onward, two
        // to an operand's rows g and g + 8 ----
        constexpr int VP = VB >= 16 ? VB / 16 : 1;            // loads per token
        constexpr int W = VB >= 16 ? 4 : 2;                   // words per load
#pragma unroll
        for (int h = 0; h < VP; ++h) {
          uint32_t v[2][2][4];                                // [token half][first, second][words]
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int tok = wtok + n * 8 + c + 4 * (x ^ swap);
              if constexpr (VB >= 16) {
                const uint4 q4 = lds128(sv + piece_off<RB, kTile>(tok, g * VP + h));
                v[n][x][0] = q4.x; v[n][x][1] = q4.y; v[n][x][2] = q4.z; v[n][x][3] = q4.w;
              } else {
                const uint2 q2 = lds64(sv + piece_off<RB, kTile>(tok, g >> 1) + (g & 1) * 8);
                v[n][x][0] = q2.x; v[n][x][1] = q2.y; v[n][x][2] = v[n][x][3] = 0;
              }
              if (edge && tok0 - wtok + tok >= to) v[n][x][0] = v[n][x][1] = v[n][x][2] = v[n][x][3] = 0;
            }
          // channels 2 p and 2 p + 1 of word wd: operand rows g and g + 8, the first token of a pair low
          auto operand = [&](int wd, int p, uint32_t (&av)[4]) {
            if constexpr (E4M3) {
              const uint32_t sel = p == 0 ? (swap ? 0x1504u : 0x5140u) : (swap ? 0x3726u : 0x7362u);
              codes_f16x4(__byte_perm(v[0][0][wd], v[0][1][wd], sel), av[0], av[1]);
              codes_f16x4(__byte_perm(v[1][0][wd], v[1][1][wd], sel), av[2], av[3]);
            } else {
              const uint32_t lo = swap ? 0x1054u : 0x5410u, hi = swap ? 0x3276u : 0x7632u;
              av[0] = __byte_perm(v[0][0][wd], v[0][1][wd], lo);
              av[1] = __byte_perm(v[0][0][wd], v[0][1][wd], hi);
              av[2] = __byte_perm(v[1][0][wd], v[1][1][wd], lo);
              av[3] = __byte_perm(v[1][0][wd], v[1][1][wd], hi);
            }
          };
          constexpr int PW = E4M3 ? 2 : 1;                    // channel pairs per word
          if (!edge) {
#pragma unroll
            for (int wd = 0; wd < W; ++wd)
#pragma unroll
              for (int p = 0; p < PW; ++p) {
                uint32_t av[4];
                operand(wd, p, av);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_16816<E4M3>(o[nt][(h * W + wd) * PW + p], av[0], av[1], av[2], av[3], pb[nt][0], pb[nt][1]);
              }
          } else {
            constexpr uint32_t one = E4M3 ? 0x3c003c00u : 0x3f803f80u, inf = E4M3 ? 0x7c00u : 0x7f80u;
            auto ones = [](uint32_t lo, uint32_t hi) { return (lo ? (one & 0xffffu) : 0u) | (hi ? (one & 0xffff0000u) : 0u); };
#pragma unroll
            for (int wd = 0; wd < W; ++wd)
#pragma unroll
              for (int p = 0; p < PW; ++p) {
                uint32_t av[4], bad[4];
                operand(wd, p, av);
#pragma unroll
                for (int k = 0; k < 4; ++k) bad[k] = not_finite<E4M3>(av[k]);
                if (__any_sync(0xffffffffu, (bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
                  // columns that see an infinity or a NaN here get it back: counts of those that pull up (+inf, NaN) and down
                  uint32_t up[4], dn[4];
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    auto pulls = [&](uint32_t half, uint32_t towards) { return half == towards || (half & 0x7fffu) > inf; };
                    up[k] = ones((bad[k] & 1u) && pulls(av[k] & 0xffffu, inf), (bad[k] >> 16) && pulls(av[k] >> 16, inf));
                    dn[k] = ones((bad[k] & 1u) && pulls(av[k] & 0xffffu, inf | 0x8000u), (bad[k] >> 16) && pulls(av[k] >> 16, inf | 0x8000u));
                  }
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t sb = see >> (nt * 4);
                    const uint32_t b0 = transposed(ones(sb & 1u, sb & 2u)), b1 = transposed(ones(sb & 4u, sb & 8u));
                    float nu[4] = {0.f, 0.f, 0.f, 0.f}, nd[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_16816<E4M3>(nu, up[0], up[1], up[2], up[3], b0, b1);
                    mma_16816<E4M3>(nd, dn[0], dn[1], dn[2], dn[3], b0, b1);
                    float (&oo)[4] = o[nt][(h * W + wd) * PW + p];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                      if (nu[k] > 0.f) oo[k] += INFINITY;
                      if (nd[k] > 0.f) oo[k] -= INFINITY;
                    }
                  }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma_16816<E4M3>(o[nt][(h * W + wd) * PW + p], av[0] & ~bad[0], av[1] & ~bad[1], av[2] & ~bad[2], av[3] & ~bad[3], pb[nt][0], pb[nt][1]);
              }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[stage]);
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l_run[nt][x] += __shfl_xor_sync(0xffffffffu, l_run[nt][x], d);
        if constexpr (E4M3) {
          const float f = 1.f / g_run[nt][x];                 // (a power of two)
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            o[nt][i][x] *= f;
            o[nt][i][2 + x] *= f;
          }
        }
      }
  }

  // ---------------- the warps' parts are joined: rows of floats in the ring's memory ----------------
  pdl_launch_dependents();
  __syncthreads();
  if (*abort_flag != 0) {
    const uint64_t t0 = globaltimer_ns();       // let copies in flight land before the memory is used again or goes away
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  constexpr int kPad = D + 4;
  float* mo = reinterpret_cast<float*>(stages);               // [warps][rows][D + 4]
  float* mm = mo + kWarps * kRows * kPad;                     // [warps][rows] references
  float* ml = mm + kWarps * kRows;                            // [warps][rows] sums
  float* jm = ml + kWarps * kRows;                            // [rows] of the CTA
  float* jl = jm + kRows;
  __syncthreads();
  if (warp < kWarps) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = nt * 8 + 2 * c + x;
        if (g == 0) {
          mm[warp * kRows + r] = m_run[nt][x];
          ml[warp * kRows + r] = l_run[nt][x];
        }
        float* dst = mo + (warp * kRows + r) * kPad + g * (D / 8);
#pragma unroll
        for (int i = 0; i < MI; i += 2)
          *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[nt][i][x], o[nt][i][2 + x], o[nt][i + 1][x], o[nt][i + 1][2 + x]);
      }
  }
  __syncthreads();
  auto store = [&](int r, int col, float m, float l, const float (&y)[8], bool whole) {
    const int tk = row0 + tok_lo + r / G, head = kvh * G + r % G;
    if (whole) {
      const float inv = l == 0.f ? 0.f : 1.f / l;             // a row that sees nothing: zeros
      *reinterpret_cast<uint4*>(a.out + (size_t)tk * a.out_stride + (size_t)head * D + col) =
          make_uint4(pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv), pack_bf16x2(y[4] * inv, y[5] * inv),
                     pack_bf16x2(y[6] * inv, y[7] * inv));
    } else {
      const int groups = gridDim.z / a.cluster;
      const size_t at = (ws_row(a.ws_step, seq, row0, tok_lo + r / G) * a.hq + head) * groups + blockIdx.z / a.cluster;
      float4* dst = reinterpret_cast<float4*>(a.ws_o + at * D + col);
      dst[0] = make_float4(y[0], y[1], y[2], y[3]);
      dst[1] = make_float4(y[4], y[5], y[6], y[7]);
      if (col == 0) {
        a.ws_ml[at * 2] = m;
        a.ws_ml[at * 2 + 1] = l;
      }
    }
  };
  const bool whole = shares <= a.cluster;                     // this cluster has the whole context
  for (int i = threadIdx.x; i < valid * (D / 8); i += kThreads) {
    const int r = i / (D / 8), col = (i % (D / 8)) * 8;
    float m = kUnset, l = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, mm[w * kRows + r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float lw = ml[w * kRows + r];
      if (lw == 0.f) continue;                                // a warp that saw nothing of this row
      const float f = exp2f(mm[w * kRows + r] - m);
      l += f * lw;
      const float4* src = reinterpret_cast<const float4*>(mo + (w * kRows + r) * kPad + col);
      const float4 u = src[0], v = src[1];
      y[0] += f * u.x; y[1] += f * u.y; y[2] += f * u.z; y[3] += f * u.w;
      y[4] += f * v.x; y[5] += f * v.y; y[6] += f * v.z; y[7] += f * v.w;
    }
    if (a.cluster == 1) {
      if ((int)blockIdx.z < shares) store(r, col, m, l, y, whole);         // (whole: the one share there is, not those that nobody has)
    } else {
      float4* dst = reinterpret_cast<float4*>(mo + r * kPad + col);       // (in place of what this thread has read)
      dst[0] = make_float4(y[0], y[1], y[2], y[3]);
      dst[1] = make_float4(y[4], y[5], y[6], y[7]);
      if (col == 0) {
        jm[r] = m;
        jl[r] = l;
      }
    }
  }
  if (a.cluster > 1) {
    // ---------------- and the cluster's: every CTA finishes a part of the rows ----------------
    cluster_barrier();
    const int rank = blockIdx.z % a.cluster, first = blockIdx.z - rank;
    const int live = min(a.cluster, shares - first);          // CTAs of this cluster that had a share
    for (int i = rank * kThreads + threadIdx.x; live > 0 && i < valid * (D / 8); i += a.cluster * kThreads) {
      const int r = i / (D / 8), col = (i % (D / 8)) * 8;
      const uint32_t am = smem_u32(jm + r), al = smem_u32(jl + r), ao = smem_u32(mo + r * kPad + col);
      float m = kUnset, l = 0.f, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < live; ++k) m = fmaxf(m, ld_rank(at_rank(am, k)));
#pragma unroll 4
      for (int k = 0; k < live; ++k) {
        const float lk = ld_rank(at_rank(al, k));
        if (lk == 0.f) continue;
        const float f = exp2f(ld_rank(at_rank(am, k)) - m);
        l += f * lk;
        const float4 u = ld_rank4(at_rank(ao, k)), v = ld_rank4(at_rank(ao, k) + 16);
        y[0] += f * u.x; y[1] += f * u.y; y[2] += f * u.z; y[3] += f * u.w;
        y[4] += f * v.x; y[5] += f * v.y; y[6] += f * v.z; y[7] += f * v.w;
      }
      store(r, col, m, l, y, whole);
    }
    cluster_barrier();                                        // no CTA's memory goes before the others have read it
  }
}

// Joins the groups of shares of every row that was cut further than a cluster reaches. A block per (row, head): its four warps take
// every fourth group, D / 32 columns a lane, and are added up in shared memory. grid (max_rows * hq, seqs). What it takes is the
// latency of two dependent loads; what does not come from the launch before it is read ahead of it.
constexpr int kMergeThreads = 128;
template <int D, bool TREE>
KERN_DEVICE void rows_merge(const float* ws_o, const float* ws_ml, __nv_bfloat16* out, const int* seq_lens, const int* cu_q, int rows_per_seq,
                            int hq, int toks, int splits, int cluster, int out_stride, int row_lo, int row_hi, int rows, int max_rows, int ws_step, int capacity) {
  constexpr int N = D / 32;
  __shared__ float y_s[4][D], l_s[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seq = blockIdx.y;
  const int row0 = cu_q ? cu_q[seq] : seq * rows_per_seq, R = cu_q ? cu_q[seq + 1] - row0 : rows_per_seq;
  const int tok = blockIdx.x / hq, head = blockIdx.x % hq;
  const int L = within(seq_lens[seq], capacity), lo = tok / toks * toks;
  const int end = TREE ? L : max(0, L - R + lo + min(toks, R - lo));
  const int shares = rows_shares(end, splits);
  const int groups = splits / cluster, live = (shares + cluster - 1) / cluster;
  const size_t base = (ws_row(ws_step, seq, row0, tok) * hq + head) * groups;
  pdl_wait();                                                 // (in every block: what follows this launch follows the one before it too)
  if (tok >= R || R < row_lo || R > row_hi || !rows_lie(row0, R, rows, max_rows)) return;
  if (shares <= cluster) return;                              // written by its one cluster
  // every warp: the largest reference of all groups
  float m = kUnset;
  for (int s = lane; s < live; s += 32) m = fmaxf(m, ws_ml[(base + s) * 2]);
  m = warp_max(m);
  float y[N], l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = 0.f;
#pragma unroll 8
  for (int s = warp; s < live; s += 4) {
    const float ms = ws_ml[(base + s) * 2], ls = ws_ml[(base + s) * 2 + 1];
    const float f = ls == 0.f ? 0.f : exp2f(ms - m);
    l += f * ls;
    const float* src = ws_o + (base + s) * D + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] += f * src[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) y_s[warp][lane * N + i] = y[i];
  if (lane == 0) l_s[warp] = l;
  __syncthreads();
  l = l_s[0] + l_s[1] + l_s[2] + l_s[3];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __nv_bfloat16* dst = out + (size_t)(row0 + tok) * out_stride + (size_t)head * D;
  for (int c = threadIdx.x * 2; c < D; c += 2 * kMergeThreads)
    *reinterpret_cast<uint32_t*>(dst + c) = pack_bf16x2((y_s[0][c] + y_s[1][c] + y_s[2][c] + y_s[3][c]) * inv,
                                                        (y_s[0][c + 1] + y_s[1][c + 1] + y_s[2][c + 1] + y_s[3][c + 1]) * inv);
}

}  // namespace kern

using namespace kern;

#define KERN_ROWS_ENTRY(D, KIND, E4M3, FORM, TREE, NT)                                                                            \
  extern "C" __global__ void __launch_bounds__(RowsCfg<D, E4M3, NT>::kThreads, RowsCfg<D, E4M3, NT>::kPerSm)                                        \
      kern_attn_rows_##KIND##_##FORM##_d##D##_n##NT(                                                                              \
          const __grid_constant__ CUtensorMap kv_map, const __nv_bfloat16* q, __nv_bfloat16* out, float* ws_o, float* ws_ml,      \
          const uint8_t* pool, const int* block_table, const int* seq_lens, const int* cu_q, const long long* masks, int words,   \
          int rows_per_seq, int hq, int hk, int q_stride, int out_stride, int max_pages, int page_size, int cluster,              \
          int pool_pages, int row_lo, int row_hi, int rows, int max_rows, int ws_step, float scale_log2, int* err) {                           \
    rows_body<D, E4M3, TREE, NT>(&kv_map, RowsArgs{q, out, ws_o, ws_ml, pool, block_table, seq_lens, cu_q, masks, err, words,     \
                                                   rows_per_seq, hq, hk, q_stride, out_stride, max_pages, page_size, cluster,     \
                                                   pool_pages, row_lo, row_hi, rows, max_rows, ws_step, scale_log2});                      \
  }
#define KERN_ROWS_MERGE(D, FORM, TREE)                                                                                            \
  extern "C" __global__ void __launch_bounds__(kMergeThreads) kern_attn_rows_merge_##FORM##_d##D(                                           \
      const float* ws_o, const float* ws_ml, __nv_bfloat16* out, const int* seq_lens, const int* cu_q, int rows_per_seq, int hq,  \
      int toks, int splits, int cluster, int out_stride, int row_lo, int row_hi, int rows, int max_rows, int ws_step, int capacity) { \
    rows_merge<D, TREE>(ws_o, ws_ml, out, seq_lens, cu_q, rows_per_seq, hq, toks, splits, cluster, out_stride, row_lo, row_hi, rows, max_rows, ws_step, capacity); \
  }
#define KERN_ROWS_FORMS(D, NT)                      \
  KERN_ROWS_ENTRY(D, e4m3, true, causal, false, NT) \
  KERN_ROWS_ENTRY(D, e4m3, true, tree, true, NT)    \
  KERN_ROWS_ENTRY(D, bf16, false, tree, true, NT)
#define KERN_ROWS(D)      \
  KERN_ROWS_FORMS(D, 1)   \
  KERN_ROWS_FORMS(D, 2)   \
  KERN_ROWS_MERGE(D, causal, false) \
  KERN_ROWS_MERGE(D, tree, true)
KERN_ROWS(64)
KERN_ROWS(128)
KERN_ROWS(256)
