// Attention of many query rows over a paged cache, bf16 or e4m3, on the 5th-generation tensor cores: prompt chunks (causal) and
// trees of drafted tokens. The formulas, formats and what a row sees are those of attn_rows.cu, which has the few rows.
//
// One CTA = (256 query rows: the G heads of 256 / G tokens, one kv head, a share of the context), 22 working warps of 24:
//
//   warps 0..15        softmax of two 128-row tiles, two threads to a row, 64 of a tile's scores each: scores out of TMEM, weights
//                      back into TMEM over them
//   warps 16..19       halves (a tile of 128 keys, or of values) for the products to read: 8-bit codes become f16 there, in the
//                      swizzle that the tensor cores read; bf16 halves lie as they came, and are only looked through where rows
//                      see different tokens
//   warp 20            issues the products:  S = Q K^T  and  O += P V  (P from TMEM), for the two tiles in turn
//   warp 21            copies by TMA: bf16 halves into a ring of five; codes, with their scale bytes, into two slots, beside a
//                      ring of four halves (three would make every V wait for the products of the K before it)
//
// The two tiles take turns on the tensor cores: while one's products run, the other's exponentials do. At most 128 rows (a small
// tree): both tiles are the same rows, on alternate key tiles, and are added up at the end, so the turns remain. TMEM: S and O of
// both tiles, 512 columns; P overwrites S.
//
// Bound: the products of a tile of keys, 2 * 128 * 128 * D multiply-adds a side, and its 128 * 128 exponentials (16 a clock) take 1024
// clocks each at D = 128, 2048 for both sides if either never paused. But a side's softmax waits for its Q K^T, and its P V for the
// softmax: a pair of tiles takes some 3300 clocks (bf16; 8-bit caches, whose conversions share the schedulers, 3500), which is
// the softmax of one side (1700: 350 to find the largest score, 1200 of exponentials) and what its two products take to come round
// (1500). So what shortens that chain counts: scores are fetched 16 columns ahead of their use, P V starts on the first half of the
// weights, the reference R of a row moves only when a weight has outgrown it (found on the largest score of the row's half, agreed
// between the two warps that share the row; no pass over O but then). Registers are dealt by role, as a spill costs an L2 access
// where shared memory has taken the L1's place.
//
// Measured (8 kv heads, 32 heads of 128): 4 prompts of up to 2048 rows on 8-bit contexts of up to 6000 388 us, 0.60 of the measured
// tensor peak; 18 trees of 128 nodes over 4000 tokens 1100 TFLOP/s (bf16) and 970 (8-bit); 64 trees of up to 32 nodes over bf16
// contexts of up to 8192 210 us, 0.88 of the measured bandwidth.
//
// 8-bit: a tile's rows are brought to one exponent, E = the largest of its scale bytes, as they become f16 (exact for scales down to
// 2^-20 of the largest); 2^E of the keys is then part of the scores' scale, E of the values part of the weights' exponent,
// w_ij = 2^(s_ij + E_t - R_i): no work per score. A block that meets a tile with scales further apart (rows of zeros aside), or
// value tiles whose exponents are more than 100 apart, is computed again, a row to a warp, each key and value row with its own
// scale (tile_wide).
#include "attn_umma.cuh"

namespace kern {

constexpr int kQ = 128, kT = 128;    // query rows of a tile, tokens of a tile
constexpr int kTileThreads = 768;    // (of 24 warps, for warpgroups; the last two only hand over their registers)

template <int D, bool E4M3>
struct TileCfg {
  static constexpr int kQBytes = 2 * kQ * D * 2;
  static constexpr int kHalf = kT * D * 2;                  // a half: a tile of K or of V, as 16-bit values
  static constexpr int kRing = E4M3 ? 4 : 5;                // halves that the products read
  static constexpr int kCodes = E4M3 ? kT * D : 0;          // a half as codes, as it comes
  static constexpr int kSlots = E4M3 ? 2 : 0;               // of which there are so many under way
  static constexpr int kScales = kSlots * 2 * kT;           // with their scale bytes, and V's beside K's
  // (all of the SM's 227 KB are in use: that the base lies on a 1024-byte boundary, as it does in practice, is checked)
  static constexpr int kSmem = kQBytes + kRing * kHalf + kSlots * kCodes + kScales + 4 * kQ * 4 + 512;
  static_assert(kSmem <= 232448, "more shared memory than a CTA has");
};

// D, cache format, tree or causal
template <int D, bool E4M3, bool TREE>
KERN_DEVICE void tile_body(const CUtensorMap* kv_map, const RowsArgs& a, const int seqs) {
  using Cfg = TileCfg<D, E4M3>;
  constexpr int kRing = Cfg::kRing, kSlots = Cfg::kSlots, kCame = E4M3 ? kSlots : kRing;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023) {                                // uniform, before any barrier or allocation
    if (threadIdx.x == 0) set_error(a.err, ERR_BOUNDS);
    return;
  }
  uint8_t* q_s = smem;                                        // two tiles, D / 64 column blocks of [128 rows][128 bytes] each
  uint8_t* h_s = q_s + Cfg::kQBytes;                          // halves
  uint8_t* c_s = h_s + kRing * Cfg::kHalf;                    // (8-bit) codes,
  uint8_t* b_s = c_s + kSlots * Cfg::kCodes;                  // scale bytes [slot][the half's own, V's beside K's][128]
  // [2 sides][2 halves of the columns][128]: at first what turns a side's rows' products into base-2 scores, then maxima and sums
  float* x_s = reinterpret_cast<float*>(b_s + Cfg::kScales);
  uint64_t* full = reinterpret_cast<uint64_t*>(x_s + 4 * kQ); // [ring] a half can be read by the products,
  uint64_t* empty = full + kRing;                             // [ring] has been read;
  uint64_t* came = empty + kRing;                             // [ring; 8-bit: slots] the copy has landed;
  uint64_t* taken = came + kCame;                             // [slots] the codes have been read
  uint64_t* s_full = taken + kCame;                              // per tile of rows: scores in TMEM,
  uint64_t* p_half = s_full + 2;                              // the first half of each thread's weights in TMEM,
  uint64_t* p_full = p_half + 2;                              // the others,
  uint64_t* o_done = p_full + 2;                              // the last P V done
  uint64_t* q_full = o_done + 2;                              // Q in shared memory
  float2* e_s = reinterpret_cast<float2*>(q_full + 2);        // [4] a key tile's (2^E of K, E of V)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(e_s + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* found = reinterpret_cast<int*>(tmem_slot + 2);         // [2] sequence and block of this CTA
  volatile int* bad_s = found + 2;                            // a value that is not finite in a tile whose rows see different tokens
  volatile int* wide_s = found + 3;                           // (8-bit) a tile's scales are further apart than f16 holds

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // (uniform registers for what follows from it)
  const int G = a.hq / a.hk, kvh = blockIdx.x, toks = 2 * kQ / G;
  pdl_wait();
  find_block<TREE>(a, seqs, toks, reinterpret_cast<int*>(q_s), found);
  if (threadIdx.x == 32) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&full[s], 4);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kCame; ++s) {
      mbar_init(&came[s], E4M3 ? 33 : 1);
      mbar_init(&taken[s], 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_half[s], 8);
      mbar_init(&p_full[s], 8);
      mbar_init(&o_done[s], 1);
    }
    mbar_init(q_full, 512);
    *abort_flag = 0;
    *bad_s = 0;
    *wide_s = 0;
    mbar_fence_init();
    tma_prefetch_desc(kv_map);
  }
  __syncthreads();
  const int seq = found[0], blk = found[1];
  if (seq < 0) return;                                        // past the last block: uniform, before any allocation
  const int L = context_of(a, seq);
  const int row0 = a.cu_q ? a.cu_q[seq] : seq * a.rows_per_seq;
  const int R = a.cu_q ? a.cu_q[seq + 1] - row0 : a.rows_per_seq;
  if (!rows_lie(row0, R, a.rows, a.max_rows)) {
    if (threadIdx.x == 0) set_error(a.err, ERR_BOUNDS);
    return;                                                   // (uniform)
  }
  const int tok_lo = blk * toks, tok_n = min(toks, R - tok_lo), valid = tok_n * G, past = L - R;
  const int end = TREE ? L : max(0, past + tok_lo + tok_n);
  const int shares = rows_shares(end, gridDim.z), share_len = rows_share_len(end, shares);
  if ((int)blockIdx.z >= shares) return;
  const int from = min(end, (int)blockIdx.z * share_len), to = min(end, from + share_len);
  const int ntiles = (to - from + kT - 1) / kT;
  const bool twice = valid <= kQ;                             // both tiles are the same rows, on alternate key tiles
  const int clear = min(to, TREE ? past : past + tok_lo + 1); // the first token that some row may not see

  if (warp == 20) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  // the order of the halves: K(0), then K(t + 1) before V(t)
  const int items = 2 * ntiles;
  auto item = [&](int i, int& which, int& t) {
    which = i == items - 1 ? 1 : (i == 0 ? 0 : !(i & 1));
    t = i == items - 1 ? ntiles - 1 : (i == 0 ? 0 : (which ? i / 2 - 1 : (i + 1) / 2));
  };
  auto k_item = [&](int t) { return t == 0 ? 0 : 2 * t - 1; };
  auto v_item = [&](int t) { return t == ntiles - 1 ? items - 1 : 2 * t + 2; };

  // Registers: 80 a thread at launch, 24 * 32 * 80 in all = 16 warps of 88, 4 of 72 and 4 of 56.
  if (warp >= 16 && warp < 20) {
    // ---------------- keys and values ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int tid = threadIdx.x - 512, w4 = warp - 16;
    if constexpr (E4M3) {
      // all of a half's codes are in registers before the half that they go to is free, so its turn is short
      constexpr int kLanes = D / 16, kRowsWarp = 32 / kLanes, kLoads = kT / (4 * kRowsWarp);     // lanes to a row of codes; rows of a lane
      const int c = lane % kLanes, sub = lane / kLanes;
      // a lane's four of a tile's scale bytes (those behind the end are 0), and the largest of all
      auto scale_word = [&](uint32_t at, int here) -> uint32_t {
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at + 4 * lane));
        const int n = here - 4 * lane;
        return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1);
      };
      auto top_byte = [&](uint32_t w) -> int {
        const uint32_t m = __vmaxu4(w, w >> 16);
        return (int)__reduce_max_sync(0xffffffffu, max(m & 255u, (m >> 8) & 255u));
      };
      for (int i = 0; i < items && ok; ++i) {
        int which, t;
        item(i, which, t);
        const int slot = i % kSlots, half = i % kRing, tok0 = from + t * kT;
        if (!bar_wait(&came[slot], (i / kSlots) & 1, abort_flag)) {
          set_error(a.err, ERR_WAIT_FULL);
          *abort_flag = 1;
          ok = false;
          break;
        }
        const uint32_t src = smem_u32(c_s) + slot * Cfg::kCodes, by = smem_u32(b_s) + slot * 2 * kT;
        // a lane: 8 codes of the row's first half and 8 of its second (one piece of 16-bit values each; D = 64: two neighbours)
        constexpr int kApart = D == 64 ? 1 : 8;
        const int p0 = D == 64 ? 2 * c : c, here = to - tok0;
        const bool edge = tok0 + kT > clear;
        const uint32_t word = scale_word(by, here);
        const int top = top_byte(word), vtop = which ? 0 : top_byte(scale_word(by + kT, here));
        // (a row of zeros has the byte -40 + 127)
        if (top > kLeastScale + 20 && (__vcmpgtu4(word, 0u) & __vcmpltu4(word, (uint32_t)(top - 20) * 0x01010101u)) != 0)
          rows_lost<D, 1>(src, 0, lane, word, top, wide_s);
        uint8_t* dst = h_s + half * Cfg::kHalf;
        bool nan = false;
        // rows r0 + j * kStep: all in the same place of the swizzle and of their words of scale bytes
        constexpr int kStep = 4 * kRowsWarp;
        const int r0 = w4 * kRowsWarp + sub;
        uint32_t w[kLoads][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int p = p0 + h * kApart;                      // eight codes: half of a 16-byte piece of the code row
          const uint32_t at = src + r0 * D + (((p >> 1) ^ (D == 64 ? (r0 >> 1) & 3 : r0 & 7)) << 4) + (p & 1) * 8;
#pragma unroll
          for (int j = 0; j < kLoads; ++j)
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[j][2 * h]), "=r"(w[j][2 * h + 1]) : "r"(at + j * kStep * D) : "memory");
        }
        if (edge) {
#pragma unroll
          for (int j = 0; j < kLoads; ++j) {
            if (r0 + j * kStep >= here) w[j][0] = w[j][1] = w[j][2] = w[j][3] = 0;      // (not brought: anything may lie there)
            if (which) {
              // values that are not finite stay out of the product: rows that see them get them at the end
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t m = __vcmpeq4(w[j][k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                nan |= m != 0;
                w[j][k] &= ~m;
              }
            }
          }
        }
        if (!bar_wait(&empty[half], ((i / kRing) & 1) ^ 1, abort_flag)) {
          set_error(a.err, ERR_WAIT_EMPTY);
          *abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t* to0 = dst + (p0 >> 3) * (kT * 128) + r0 * 128 + (((p0 & 7) ^ (r0 & 7)) << 4);
        uint8_t* to1 = dst + ((p0 + kApart) >> 3) * (kT * 128) + r0 * 128 + ((((p0 + kApart) & 7) ^ (r0 & 7)) << 4);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          // 2^(e - E + 6) twice over, as f16: 1 to 21 in the exponent's bits (0: a row of zeros, or one computed again)
          const uint32_t b = __shfl_sync(0xffffffffu, word, (r0 + j * kStep) >> 2) >> (8 * (r0 & 3)) & 255u;
          const uint32_t fj = (uint32_t)max((int)b + 21 - top, 0) * 0x04000400u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t o[4];
            codes_f16x4(w[j][2 * h], o[0], o[1]);
            codes_f16x4(w[j][2 * h + 1], o[2], o[3]);
            *reinterpret_cast<uint4*>((h ? to1 : to0) + j * kStep * 128) =
                make_uint4(mul_f16x2(o[0], fj), mul_f16x2(o[1], fj), mul_f16x2(o[2], fj), mul_f16x2(o[3], fj));
          }
        }
        if (nan) *bad_s = 1;
        if (!which && w4 == 0 && lane == 0) e_s[t & 3] = make_float2(pow2i(top - 127 - 6), (float)(vtop - 127 - 6));
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&full[half]);
          // (not before the codes have been used: behind the loads alone, what the next copy brought was read now and then; and no slower)
          mbar_arrive(&taken[slot]);
        }
      }
    } else {
      for (int i = 0; i < items && ok; ++i) {
        int which, t;
        item(i, which, t);
        const int half = i % kRing, tok0 = from + t * kT;
        if (!bar_wait(&came[half], (i / kRing) & 1, abort_flag)) {
          set_error(a.err, ERR_WAIT_FULL);
          *abort_flag = 1;
          ok = false;
          break;
        }
        if (which && tok0 + kT > clear) {
          // values that are not finite stay out of the product: rows that see them get them at the end
          uint8_t* dst = h_s + half * Cfg::kHalf;
          bool bad = false;
          for (int x = tid; x < kT * (D / 8); x += 128) {
            const int r = x / (D / 8), p = x % (D / 8);
            uint4* at = reinterpret_cast<uint4*>(dst + (p >> 3) * (kT * 128) + r * 128 + (((p & 7) ^ (r & 7)) << 4));
            if (tok0 + r >= to) {
              *at = make_uint4(0, 0, 0, 0);                   // (not brought: anything may lie there)
            } else {
              const uint4 v = *at;
              const uint32_t m0 = not_finite<false>(v.x), m1 = not_finite<false>(v.y), m2 = not_finite<false>(v.z), m3 = not_finite<false>(v.w);
              if (m0 | m1 | m2 | m3) {
                bad = true;
                *at = make_uint4(v.x & ~m0, v.y & ~m1, v.z & ~m2, v.w & ~m3);
              }
            }
          }
          if (bad) *bad_s = 1;
          fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[half]);
      }
    }
  } else if (warp >= 20) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 21) {
      // ---------------- copies: bf16 halves into the ring, 8-bit codes and scale bytes into their slots ----------------
      const size_t codes = (size_t)2 * a.hk * a.page_size * D, page_bytes = codes + 2 * a.hk * a.page_size;
      const int box = a.page_size < 64 ? a.page_size : 64;
      const int* pages = a.block_table + (size_t)seq * a.max_pages;
      // runs of 64 tokens (or of a smaller page's) lie in one page; the table is read 32 pages at a time, a lane each
      const int bits = a.page_size < 64 ? 31 - __clz(a.page_size) : 6, per = a.page_size < 64 ? 1 : a.page_size >> 6;
      auto page_of = [&](int tok) { return per == 1 ? tok >> bits : (tok >> bits) / per; };
      int first = -64, id = 0;
      for (int i = 0; i < items && ok; ++i) {
        int which, t;
        item(i, which, t);
        const int slot = E4M3 ? i % kSlots : i % kRing, tok0 = from + t * kT, here = min(kT, to - tok0), boxes = (here + box - 1) / box;
        if (page_of(tok0) < first || page_of(tok0 + here - 1) >= first + 32) {
          // (the values of the tile before are still to come: a tile has 16 pages at most)
          first = page_of(max(tok0 - kT, from));
          const int pi = first + lane;
          id = pi < a.max_pages ? pages[pi] : -1;
          if (id < 0 || id >= a.pool_pages) {
            if (pi * a.page_size < to) set_error(a.err, ERR_BOUNDS);
            id = 0;
          }
        }
        // page, and row in it, of the eight tokens from 8 lane on
        const int tok = tok0 + 8 * (lane & 15), pi = page_of(tok), off = tok - pi * a.page_size;
        const int page = __shfl_sync(0xffffffffu, id, (pi - first) & 31);
        const int uses = i / (E4M3 ? kSlots : kRing);
        const int b_page = __shfl_sync(0xffffffffu, page, (lane * box >> 3) & 31), b_off = __shfl_sync(0xffffffffu, off, (lane * box >> 3) & 31);
        const int b_row = (which * a.hk + kvh) * a.page_size + b_off;
        // boxes behind the share's end are not brought
        if constexpr (E4M3) {
          const int s_page = __shfl_sync(0xffffffffu, page, lane >> 1), s_off = __shfl_sync(0xffffffffu, off, lane >> 1) + (lane & 1) * 4;
          if (!bar_wait(&taken[slot], (uses & 1) ^ 1, abort_flag)) {
            set_error(a.err, ERR_WAIT_EMPTY);
            *abort_flag = 1;
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect_tx(&came[slot], boxes * box * D);
          __syncwarp();
          if (lane < boxes) tma_load_3d(c_s + slot * Cfg::kCodes + lane * box * D, kv_map, 0, b_row, b_page, &came[slot]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (k && which) break;
            const uint8_t* src = a.pool + (size_t)s_page * page_bytes + codes + (size_t)((k ? 1 : which) * a.hk + kvh) * a.page_size + s_off;
            if (4 * lane < here && KERN_CHECK(src, 4, SITE_KV_ROW))
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(b_s + slot * 2 * kT + k * kT + 4 * lane)), "l"(src) : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&came[slot])) : "memory");
        } else {
          if (!bar_wait(&empty[slot], (uses & 1) ^ 1, abort_flag)) {
            set_error(a.err, ERR_WAIT_EMPTY);
            *abort_flag = 1;
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect_tx(&came[slot], boxes * box * D * 2);
          __syncwarp();
          if (lane < boxes) {
#pragma unroll
            for (int cb = 0; cb < D / 64; ++cb)
              tma_load_3d(h_s + slot * Cfg::kHalf + cb * (kT * 128) + lane * box * 128, kv_map, cb * 64, b_row, b_page, &came[slot]);
          }
        }
      }
    } else if (warp == 20) {
      // ---------------- products: the whole warp walks and waits, one lane issues ----------------
      constexpr uint32_t idesc_qk = tile_idesc<E4M3>(kQ, kT, false), idesc_pv = tile_idesc<E4M3>(kQ, D, true);
      const int steps = twice ? ntiles : 2 * ntiles;
      const uint32_t q_low = desc_low(smem_u32(q_s), 0), h_low = desc_low(smem_u32(h_s), 0), v_low = desc_low(smem_u32(h_s), kT * 128);
      const bool leader = elect_lane();
      float ev_least = 255.f, ev_most = -255.f;               // (8-bit) the value tiles' exponents
      auto qk = [&](int u) -> bool {
        const int side = u & 1, t = twice ? u : u >> 1;
        const int i = k_item(t), half = i % kRing;
        if (!bar_wait(&full[half], (i / kRing) & 1, abort_flag)) return false;
        tc_fence_after();
        const uint32_t sq = q_low + side * (kQ * D * 2 >> 4), sk = h_low + half * (Cfg::kHalf >> 4), s_t = tmem + side * 128;
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_ss(s_t, sq + ((k >> 2) * (kQ * 128) + (k & 3) * 32 >> 4), sk + ((k >> 2) * (kT * 128) + (k & 3) * 32 >> 4), idesc_qk, k != 0);
          tc_commit(&s_full[side]);
          if (twice || side) tc_commit(&empty[half]);
        }
        __syncwarp();
        if constexpr (E4M3) {
          // (here, where a few instructions make nobody wait: 386 us for the prompts above, 404 in the warps that convert)
          const float ev = fmaxf(e_s[t & 3].y, kLeastShift);
          ev_least = fminf(ev_least, ev);
          ev_most = fmaxf(ev_most, ev);
          if (ev_most - ev_least > (float)kTilesApart) *wide_s = 1;
        }
        return true;
      };
      auto pv = [&](int u) -> bool {
        const int side = u & 1, t = twice ? u : u >> 1, n = u >> 1;
        const int i = v_item(t), half = i % kRing;
        if (!bar_wait(&full[half], (i / kRing) & 1, abort_flag)) return false;
        if (!bar_wait(&p_half[side], n & 1, abort_flag)) return false;
        tc_fence_after();
        const uint32_t sv = v_low + half * (Cfg::kHalf >> 4), o_t = tmem + 256 + side * D, p_t = tmem + side * 128;
        if (leader) {
#pragma unroll
          for (int i = 0; i < kT / 32; ++i) {
            const int k = i < kT / 64 ? i : i + kT / 64;      // (a thread's first 32 columns are two steps, of each half of the tile)
            umma_ts(o_t, p_t + (k < 4 ? k : k + 4) * 8, sv + (k * 16 * 128 >> 4), idesc_pv, (n | k) != 0);
          }
        }
        __syncwarp();
        if (!bar_wait(&p_full[side], n & 1, abort_flag)) return false;
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int i = 0; i < kT / 32; ++i) {
            const int k = (i < kT / 64 ? i : i + kT / 64) + 2;
            umma_ts(o_t, p_t + (k < 4 ? k : k + 4) * 8, sv + (k * 16 * 128 >> 4), idesc_pv, 1);
          }
          if (twice || side) tc_commit(&empty[half]);
          if (u + 2 >= steps) tc_commit(&o_done[side]);
        }
        __syncwarp();
        return true;
      };
      if (steps > 0) ok = bar_wait(q_full, 0, abort_flag) && qk(0);
      if (ok && steps > 1) ok = qk(1);
      for (int u = 0; u < steps && ok; ++u) {
        ok = pv(u);
        if (ok && u + 2 < steps) ok = qk(u + 2);                // (overwrites the scores whose weights P V has just been given)
      }
      if (!ok) {
        set_error(a.err, ERR_WAIT_FULL);
        *abort_flag = 1;
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    // ---------------- Q -> shared memory, K-major with the 128-byte swizzle: D / 8 lanes to a row ----------------
    {
      constexpr int kLanes = D / 8, kPass = 512 / kLanes, kPasses = 2 * kQ / kPass;
      const int c = threadIdx.x % kLanes;
      const float per_g = 1.f / (float)G;
      const __nv_bfloat16* q_at = a.q + (size_t)(row0 + tok_lo) * a.q_stride + (size_t)kvh * G * D + c * 8;
      uint4 rows[kPasses];                                    // (all under way together)
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int r = threadIdx.x / kLanes + i * kPass, rr = twice ? r & (kQ - 1) : r;
        const int tok = (int)((rr + 0.5f) * per_g), head = rr - tok * G;      // (rr / G, exact: rr < 256)
        rows[i] = make_uint4(0, 0, 0, 0);
        if (rr < valid) rows[i] = *reinterpret_cast<const uint4*>(q_at + (size_t)tok * a.q_stride + head * D);
      }
#pragma unroll
      for (int i = 0; i < kPasses; ++i) {
        const int r = threadIdx.x / kLanes + i * kPass;
        uint4 v = rows[i];
        float f = a.scale_log2;
        if constexpr (E4M3) {
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          float top = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 u = unpack_bf16x2(w[k]);
            top = fmaxf(top, fmaxf(fabsf(u.x), fabsf(u.y)));
          }
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int x = min(max((int)((__float_as_uint(top) >> 23) & 255) - 127, -100), 100);
          const float inv = pow2i(-x);
          f *= pow2i(x);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 u = unpack_bf16x2(w[k]);
            w[k] = pack_f16x2(u.x * inv, u.y * inv);
          }
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4*>(q_s + (r >> 7) * (kQ * D * 2) + (c >> 3) * (kQ * 128) + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
        if (c == 0) x_s[(r >> 7) * 2 * kQ + (r & 127)] = f;
      }
      fence_proxy_async();
      mbar_arrive(q_full);
      asm volatile("bar.sync 15, 512;" ::: "memory");          // x_s
    }
    // ---------------- softmax: two threads to a row, half of a tile's scores each ----------------
    const int side = (warp >> 2) & 1, part = warp >> 3, row = (warp & 3) * 32 + lane;
    const int r = twice ? row : side * kQ + row;              // of the block's rows
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem + lanes + side * 128 + part * 64, o_t = tmem + lanes + 256 + side * D + part * (D / 2);
    const int tk = tok_lo + (r < valid ? r / G : 0), pos = past + tk;
    const long long* mask = TREE ? a.masks + (size_t)(row0 + tk) * a.words : nullptr;
    const int steps = twice ? (ntiles + 1 - side) / 2 : ntiles;
    const float f = x_s[side * 2 * kQ + row];                 // (read before the side's threads meet, written after)
    float* const own_x = x_s + (side * 2 + part) * kQ + row;  // what the row's two threads tell each other
    float* const his_x = x_s + (side * 2 + 1 - part) * kQ + row;
    const int pair = 1 + (warp & 7);                          // barrier of the two warps that share 32 rows
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory"); };
    auto any_of = [&](bool mine) -> bool {                    // over the two warps' threads
      uint32_t any;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(any)
                   : "r"(pair), "r"((uint32_t)mine)
                   : "memory");
      return any != 0;
    };
    // A reference starts 2^5 under its first tile's maximum and moves, when a weight has outgrown f16
    // (2^30 for bf16 weights). So weights down to 2^-19 of the largest keep all of f16's bits, and where key rows differ in size
    // (by e^0.5) 128 rows move some 9 times in 4096 tokens; 17 times from 2^7 under it and at 2^15.
    constexpr float kGrown = E4M3 ? 15.9f : 30.f, kBelow = E4M3 ? 5.f : 0.f;
    float ref = kUnset, l = 0.f;                              // l: of this thread's columns
    // (a wait that has run out does not leave the walk: the side's threads meet in every step)
    for (int n = 0; n < steps; ++n) {
      const int t = twice ? 2 * n + side : n;
      const int tok0 = from + t * kT;
      if (ok && !bar_wait(&s_full[side], n & 1, abort_flag)) {
        set_error(a.err, ERR_WAIT_TMEM_FULL);
        *abort_flag = 1;
        ok = false;
      }
      tc_fence_after();
      const bool edge = tok0 + kT > clear;                    // uniform
      float scale = f, ev = 0.f;
      if constexpr (E4M3) {
        const float2 e = e_s[t & 3];
        scale = row_scale(f, e.x);
        ev = fmaxf(e.y, kLeastShift);
      }
      if (edge) {
        // the scores that a row does not see become -inf where they lie
#pragma unroll 1
        for (int c = 0; c < 64; c += 32) {
          uint32_t x[32];
          tmem_ld_32x32(s_t + c, x);
          tmem_ld_wait();
          const uint32_t b = seen32<TREE>(mask, a.words, past, pos, to, tok0 + part * 64 + c);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(b >> i & 1)) x[i] = 0xff800000u;
          tmem_st32(s_t + c, x);
        }
        tmem_st_done();
      }
      // ---- the largest score (16 columns on their way while 16 are looked at) ----
      uint32_t x[2][16];
      float m2[2] = {-INFINITY, -INFINITY};
      tmem_ld16(s_t, x[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_ld_wait();
        if (c < 3) tmem_ld16(s_t + (c + 1) * 16, x[(c + 1) & 1]);
#pragma unroll
        for (int i = 0; i < 16; i += 2) m2[(i >> 1) & 1] = max3(m2[(i >> 1) & 1], __uint_as_float(x[c & 1][i]), __uint_as_float(x[c & 1][i + 1]));
      }
      float mx = fmaxf(m2[0], m2[1]);
      mx = fmaf(mx, scale, ev);
      if (any_of(mx > ref + kGrown)) {
        // a row's two threads move its reference together, and each passes over half of O
        *own_x = mx;
        meet();
        mx = fmaxf(mx, *his_x);
        const float to_ref = mx > ref + kGrown ? ceilf(mx) - kBelow : ref, corr = exp2f(ref - to_ref);
        ref = to_ref;
        l *= corr;
        if (n > 0) {
          // (these scores' products were issued behind the last P V: O is quiet)
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 16) {
            uint32_t y[16];
            tmem_ld16(o_t + c, y);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * corr);
            tmem_st16(o_t + c, y);
          }
          tmem_st_done();
        }
        meet();                                               // (the places are free again)
      }
      // ---- weights, over scores of this thread's own that have been read; their sum ----
      const uint64_t scale2 = pair64(scale, scale), shift2 = pair64(ev - ref, ev - ref);
      uint64_t sum2[2] = {0, 0};
      tmem_ld16(s_t, x[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[8];
        tmem_ld_wait();
        if (c < 3) tmem_ld16(s_t + (c + 1) * 16, x[(c + 1) & 1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 y = split64(fma2(pair64(__uint_as_float(x[c & 1][2 * i]), __uint_as_float(x[c & 1][2 * i + 1])), scale2, shift2));
          const float u = exp2f(y.x), v = exp2f(y.y);
          pk[i] = pack_pair<E4M3>(u, v);
          sum2[i & 1] = add2(sum2[i & 1], E4M3 ? pair64(u, v) : pair64(__uint_as_float(pk[i] << 16), __uint_as_float(pk[i] & 0xffff0000u)));
        }
        tmem_st8(s_t + c * 8, pk);
        if (c == 1) {
          tmem_st_done();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[side]);
        }
      }
      const float2 sum = split64(add2(sum2[0], sum2[1]));
      l += E4M3 ? (sum.x + sum.y) * exp2f(-ev) : sum.x + sum.y;
      tmem_st_done();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[side]);
    }
    if (ok && steps > 0 && !bar_wait(&o_done[side], 0, abort_flag)) {
      set_error(a.err, ERR_WAIT_TMEM_FULL);
      *abort_flag = 1;
      ok = false;
    }
    tc_fence_after();
    // ---------------- the rows' end: half of the columns to each of a row's threads ----------------
    *own_x = l;
    meet();
    l += *his_x;
    constexpr int kHalfD = D / 2, kPad = kHalfD + 3;
    float* other = reinterpret_cast<float*>(h_s) + part * (kQ * kPad);    // (twice) the second side's rows: columns, reference, sum
    if (twice) asm volatile("bar.sync 15, 512;" ::: "memory"); // both sides' products are done: the ring is free
    const bool wide = E4M3 && *wide_s != 0;                   // (uniform: every half has been looked at)
    if (twice) {
      if (side == 1) {
        float* mine = other + row * kPad;
        mine[kHalfD] = ref;
        mine[kHalfD + 1] = l;
#pragma unroll 1
        for (int c = 0; c < kHalfD; c += 32) {
          uint32_t x[32];
          tmem_ld_32x32(o_t + c, x);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) mine[c + i] = steps > 0 ? __uint_as_float(x[i]) : 0.f;
        }
      }
      asm volatile("bar.sync 15, 512;" ::: "memory");
    }
    if (wide) {
      if constexpr (E4M3) {
        const RowsArgs args = a;                              // (a copy on the stack, for this call alone)
        if (ok) tile_wide<D, TREE>(args, seq, row0, tok_lo, valid, past, from, to, shares, 16);
      }
    } else if (!(twice && side)) {
      float own = 1.f, his = 0.f, m = ref;
      if (twice) {
        const float* x = other + row * kPad;
        m = fmaxf(ref, x[kHalfD]);
        own = l == 0.f ? 0.f : exp2f(ref - m);
        his = x[kHalfD + 1] == 0.f ? 0.f : exp2f(x[kHalfD] - m);
        l = (l == 0.f ? 0.f : l * own) + (x[kHalfD + 1] == 0.f ? 0.f : x[kHalfD + 1] * his);
      }
      const bool whole = shares == 1, store = r < valid && ok;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (E4M3 && !whole) {
        const float level = level_share(m, l);
        own *= level;
        his *= level;
      }
      const int head = kvh * G + (r < valid ? r % G : 0);
      const size_t at = (ws_row(a.ws_step, seq, row0, tk) * a.hq + head) * gridDim.z + blockIdx.z;
      const bool bad = *bad_s != 0;
#pragma unroll 1
      for (int c = 0; c < kHalfD; c += 32) {
        const int col = part * kHalfD + c;
        uint32_t x[32];
        tmem_ld_32x32(o_t + c, x);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(own != 0.f && steps > 0 ? __uint_as_float(x[i]) * own : 0.f);
        if (twice && his != 0.f) {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) + other[row * kPad + c + i] * his);
        }
        if (bad && store) put_back<D, E4M3, TREE>(a, mask, seq, past, pos, from + max(clear - from, 0) / kT * kT, to, col, x);
        if (!store) continue;
        if (whole) {
          __nv_bfloat16* dst = a.out + (size_t)(row0 + tk) * a.out_stride + (size_t)head * D + col;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = pack_bf16x2(__uint_as_float(x[8 * i + 2 * k]) * inv, __uint_as_float(x[8 * i + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + i * 8) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        } else {
          uint4* dst = reinterpret_cast<uint4*>(a.ws_o + at * D + col);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        }
      }
      if (!whole && store && part == 0) {
        a.ws_ml[at * 2] = m;
        a.ws_ml[at * 2 + 1] = l;
      }
    }
  }

  // ---------------- teardown ----------------
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    const uint64_t t0 = globaltimer_ns();       // let copies and products in flight end before the memory goes away
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  __syncthreads();
  if (warp == 20) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace kern

using namespace kern;

#define KERN_TILE_ENTRY(D, KIND, E4M3, FORM, TREE)                                                                                \
  extern "C" __global__ void __launch_bounds__(kTileThreads, 1) kern_attn_tile_##KIND##_##FORM##_d##D(                            \
      const __grid_constant__ CUtensorMap kv_map, const __nv_bfloat16* q, __nv_bfloat16* out, float* ws_o, float* ws_ml,          \
      const uint8_t* pool, const int* block_table, const int* seq_lens, const int* cu_q, const long long* masks, int words,       \
      int rows_per_seq, int hq, int hk, int q_stride, int out_stride, int max_pages, int page_size, int seqs, int pool_pages,     \
      int row_lo, int row_hi, int rows, int max_rows, int ws_step, float scale_log2, int* err) {                                               \
    tile_body<D, E4M3, TREE>(&kv_map, RowsArgs{q, out, ws_o, ws_ml, pool, block_table, seq_lens, cu_q, masks, err, words,         \
                                               rows_per_seq, hq, hk, q_stride, out_stride, max_pages, page_size, 1, pool_pages,   \
                                               row_lo, row_hi, rows, max_rows, ws_step, scale_log2},                                       \
                             seqs);                                                                                               \
  }
#define KERN_TILE(D)                            \
  KERN_TILE_ENTRY(D, e4m3, true, causal, false) \
  KERN_TILE_ENTRY(D, e4m3, true, tree, true)    \
  KERN_TILE_ENTRY(D, bf16, false, tree, true)
KERN_TILE(64)
KERN_TILE(128)
