// Attention of many query rows over a paged cache for head_dim 256: attn_tile.cu's formulas and formats, another shape. O of 128 rows
// takes half of TMEM there, so a CTA has one tile of 128 query rows, and pauses are filled from its own next tile: scores have two
// places, and Q K^T of the next 64 keys runs while a tile's softmax does.
//
//   warps 0..7      softmax, two threads to a row, 32 of a tile's 64 scores each, held in registers from the maximum to the weights
//   warps 8..15     two teams of four, a half (64 keys, or values) each in turn: 8-bit codes become f16, as in attn_tile.cu; one team
//                   looks through bf16 halves where rows see different tokens
//   warp 16         issues the products in the order Q K^T(t + 2) behind P V(t); O is quiet for a reference to move once the P V before
//                   has ended, which a barrier of its own tells
//   warp 17         copies by TMA: codes into two slots, a team's each, beside a ring of four halves; bf16 halves into a ring of five
//
// TMEM: O in columns 0..255, scores in 256..319 and 320..383, the weights over them (a thread's 32 over its own columns).
//
// Bound: 2 * 128 * 64 * 256 multiply-adds a tile take 1024 clocks, its exponentials 512; 32 KB of f16 values a half go through shared
// memory for 128 query rows where attn_tile.cu has 256, so the conversions weigh twice as much. Measured: 4 prompts of 1024 rows on 4000
// tokens, 8-bit, 24 heads over 4, 424 us, 830 TFLOP/s (16 query rows at a time in the few-row kernel: 3100 us).
#include "attn_umma.cuh"

namespace kern {

constexpr int kWide = 256, kQRows = 128, kKeys = 64, kWideThreads = 576;

template <bool E4M3>
struct Tile256Cfg {
  static constexpr int kQBytes = kQRows * kWide * 2;
  static constexpr int kHalf = kKeys * kWide * 2;
  static constexpr int kRing = E4M3 ? 4 : 5;
  static constexpr int kSlots = E4M3 ? 2 : 0, kCodes = E4M3 ? kKeys * kWide : 0, kScales = kSlots * 2 * kKeys;
  static constexpr int kSmem = kQBytes + kRing * kHalf + kSlots * kCodes + kScales + 2 * kQRows * 4 + 512;
  static_assert(kSmem <= 232448, "more shared memory than a CTA has");
};

// An arrival that says that a warp's loads from shared memory are done, before anything has used them. The address takes in every lane's
// values (`zero` is 0, which the compiler does not know; `others`: what else was loaded from the slot): behind the loads alone the arrival
// came before some of them now and then, and they read what the next copy brought.
template <int N>
KERN_DEVICE void arrive_loaded(uint64_t* bar, const uint32_t (&w)[N][4], uint32_t others, uint32_t zero) {
  uint32_t all = others;
#pragma unroll
  for (int i = 0; i < N; ++i) all |= w[i][0] | w[i][1] | w[i][2] | w[i][3];
  const uint32_t off = __reduce_or_sync(0xffffffffu, all & zero);
  if ((threadIdx.x & 31) == 0) mbar_arrive(reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(bar) + off));
}

// cache format, tree or causal
template <bool E4M3, bool TREE>
KERN_DEVICE void tile256_body(const CUtensorMap* kv_map, const RowsArgs& a, const int seqs) {
  using Cfg = Tile256Cfg<E4M3>;
  constexpr int D = kWide, kRing = Cfg::kRing, kSlots = Cfg::kSlots, kCame = E4M3 ? kSlots : kRing;
  constexpr int kBlock = kKeys * 128, kQBlock = kQRows * 128;  // 64 columns of a half, of Q
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023) {                                // uniform, before any barrier or allocation
    if (threadIdx.x == 0) set_error(a.err, ERR_BOUNDS);
    return;
  }
  uint8_t* q_s = smem;                                        // four column blocks of [128 rows][128 bytes]
  uint8_t* h_s = q_s + Cfg::kQBytes;                          // halves: four column blocks of [64 rows][128 bytes]
  uint8_t* c_s = h_s + kRing * Cfg::kHalf;                    // (8-bit) codes: two of [64 rows][128 bytes],
  uint8_t* b_s = c_s + kSlots * Cfg::kCodes;                  // scale bytes [slot][the half's own, V's beside K's][64]
  float* x_s = reinterpret_cast<float*>(b_s + Cfg::kScales);  // [2 halves of the columns][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(x_s + 2 * kQRows);
  uint64_t* empty = full + kRing;
  uint64_t* came = empty + kRing;
  uint64_t* taken = came + kCame;
  uint64_t* s_full = taken + kCame;                           // [2] scores in TMEM,
  uint64_t* p_full = s_full + 2;                              // [2] weights in TMEM,
  uint64_t* o_quiet = p_full + 2;                             // [2] the P V has ended
  uint64_t* q_full = o_quiet + 2;
  float2* e_s = reinterpret_cast<float2*>(q_full + 1);        // [4] a key tile's (2^E of K, E of V)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(e_s + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* found = reinterpret_cast<int*>(tmem_slot + 2);         // [2] sequence and block of this CTA
  volatile int* bad_s = found + 2;
  volatile int* wide_s = found + 3;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int G = a.hq / a.hk, kvh = blockIdx.x, toks = kQRows / G;
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
      mbar_init(&p_full[s], 8);
      mbar_init(&o_quiet[s], 1);
    }
    mbar_init(q_full, 256);
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
  const int ntiles = (to - from + kKeys - 1) / kKeys;
  const int clear = min(to, TREE ? past : past + tok_lo + 1); // the first token that some row may not see

  if (warp == 16) {
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

  if (warp >= 8 && warp < 16) {
    // ---------------- keys and values: item i is team i & 1's, so a place of the ring is always the same team's, which has seen every
    // turn of its barriers (8-bit; of five places each would change hands: bf16 halves, which take next to no work, have one team) ------
    const int team = (warp >> 2) & 1, w4 = warp & 3;
    const uint32_t zero = (uint32_t)(a.rows >> 31);
    static_assert(!E4M3 || kRing % 2 == 0, "a place belongs to one team");
    for (int i = E4M3 || !team ? team : items; i < items && ok; i += E4M3 ? 2 : 1) {
      int which, t;
      item(i, which, t);
      const int half = i % kRing, tok0 = from + t * kKeys, here = to - tok0;
      const bool edge = tok0 + kKeys > clear;
      uint8_t* dst = h_s + half * Cfg::kHalf;
      bool bad = false;
      if constexpr (E4M3) {
        const int slot = team;                                // (i % 2)
        if (!bar_wait(&came[slot], (i / kSlots) & 1, abort_flag)) {
          set_error(a.err, ERR_WAIT_FULL);
          *abort_flag = 1;
          ok = false;
          break;
        }
        const uint32_t src = smem_u32(c_s) + slot * Cfg::kCodes, by = smem_u32(b_s) + slot * 2 * kKeys;
        // a lane's four of the tile's scale bytes (those behind the end are 0; 16 lanes have some), and the largest of all
        auto scale_word = [&](uint32_t at) -> uint32_t {
          uint32_t w;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(at + 4 * (lane & 15)));
          const int n = lane < 16 ? here - 4 * lane : 0;
          return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1);
        };
        auto top_byte = [&](uint32_t w) -> int {
          const uint32_t m = __vmaxu4(w, w >> 16);
          return (int)__reduce_max_sync(0xffffffffu, max(m & 255u, (m >> 8) & 255u));
        };
        const uint32_t word = scale_word(by), v_word = which ? 0u : scale_word(by + kKeys);
        const int top = top_byte(word), vtop = top_byte(v_word);
        // (a row of zeros has the byte -40 + 127)
        if (top > kLeastScale + 20 && (__vcmpgtu4(word, 0u) & __vcmpltu4(word, (uint32_t)(top - 20) * 0x01010101u)) != 0)
          rows_lost<128, 2>(src, kBlock, lane, word, top, wide_s);
        // a lane: 8 codes of the row's first 128 and 8 of its second (a piece of 16-bit values each), in rows r0 + 8 j: all in the
        // same place of the swizzle and of their words of scale bytes
        constexpr int kLoads = kKeys / 8;
        const int c = lane & 15, r0 = w4 * 2 + (lane >> 4);
        const uint32_t at = src + r0 * 128 + (((c >> 1) ^ (r0 & 7)) << 4) + (c & 1) * 8;
        uint32_t w[kLoads][4];
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[j][2 * h]), "=r"(w[j][2 * h + 1]) : "r"(at + h * kBlock + j * 8 * 128) : "memory");
        arrive_loaded(&taken[slot], w, word | v_word, zero);                 // (once the codes have been used: 473 us, not 424, for the prompts above)
        if (edge) {
#pragma unroll
          for (int j = 0; j < kLoads; ++j) {
            if (r0 + j * 8 >= here) w[j][0] = w[j][1] = w[j][2] = w[j][3] = 0;      // (not brought: anything may lie there)
            if (which) {
              // values that are not finite stay out of the product: rows that see them get them at the end
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t m = __vcmpeq4(w[j][k] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                bad |= m != 0;
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
        // piece c of the row's 32: column block c >> 3, and two blocks on for the second 128 columns
        uint8_t* to0 = dst + (c >> 3) * kBlock + r0 * 128 + (((c & 7) ^ (r0 & 7)) << 4);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          // 2^(e - E + 6) twice over, as f16: 1 to 21 in the exponent's bits (0: a row of zeros, or one computed again)
          const uint32_t b = __shfl_sync(0xffffffffu, word, (r0 + j * 8) >> 2) >> (8 * (r0 & 3)) & 255u;
          const uint32_t fj = (uint32_t)max((int)b + 21 - top, 0) * 0x04000400u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t o[4];
            codes_f16x4(w[j][2 * h], o[0], o[1]);
            codes_f16x4(w[j][2 * h + 1], o[2], o[3]);
            *reinterpret_cast<uint4*>(to0 + h * 2 * kBlock + j * 8 * 128) =
                make_uint4(mul_f16x2(o[0], fj), mul_f16x2(o[1], fj), mul_f16x2(o[2], fj), mul_f16x2(o[3], fj));
          }
        }
        if (!which && w4 == 0 && lane == 0) e_s[t & 3] = make_float2(pow2i(top - 127 - 6), (float)(vtop - 127 - 6));
        fence_proxy_async();
      } else {
        if (!bar_wait(&came[half], (i / kRing) & 1, abort_flag)) {
          set_error(a.err, ERR_WAIT_FULL);
          *abort_flag = 1;
          ok = false;
          break;
        }
        if (which && edge) {
          // values that are not finite stay out of the product: rows that see them get them at the end
          for (int x = w4 * 32 + lane; x < kKeys * (D / 8); x += 128) {
            const int r = x / (D / 8), p = x % (D / 8);
            uint4* at = reinterpret_cast<uint4*>(dst + (p >> 3) * kBlock + r * 128 + (((p & 7) ^ (r & 7)) << 4));
            if (r >= here) {
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
          fence_proxy_async();
        }
      }
      if (bad) *bad_s = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[half]);
    }
  } else if (warp == 17) {
    // ---------------- copies ----------------
    const size_t codes = (size_t)2 * a.hk * a.page_size * D, page_bytes = codes + 2 * a.hk * a.page_size;
    const int box = a.page_size < 64 ? a.page_size : 64;
    const int* pages = a.block_table + (size_t)seq * a.max_pages;
    const int bits = a.page_size < 64 ? 31 - __clz(a.page_size) : 6, per = a.page_size < 64 ? 1 : a.page_size >> 6;
    auto page_of = [&](int tok) { return per == 1 ? tok >> bits : (tok >> bits) / per; };
    int first = -64, id = 0;
    for (int i = 0; i < items && ok; ++i) {
      int which, t;
      item(i, which, t);
      const int slot = E4M3 ? i % kSlots : i % kRing, uses = i / (E4M3 ? kSlots : kRing);
      const int tok0 = from + t * kKeys, here = min(kKeys, to - tok0), boxes = (here + box - 1) / box;
      if (page_of(tok0) < first || page_of(tok0 + here - 1) >= first + 32) {
        // the table, 32 pages at a time (the values of the tile before are still to come: a tile has 8 pages at most)
        first = page_of(max(tok0 - kKeys, from));
        const int pi = first + lane;
        id = pi < a.max_pages ? pages[pi] : -1;
        if (id < 0 || id >= a.pool_pages) {
          if (pi * a.page_size < to) set_error(a.err, ERR_BOUNDS);
          id = 0;
        }
      }
      // page, and row in it, of the eight tokens from 8 lane on
      const int tok = tok0 + 8 * (lane & 7), pi = page_of(tok), off = tok - pi * a.page_size;
      const int page = __shfl_sync(0xffffffffu, id, (pi - first) & 31);
      const int b_page = __shfl_sync(0xffffffffu, page, (lane * box >> 3) & 31), b_off = __shfl_sync(0xffffffffu, off, (lane * box >> 3) & 31);
      const int b_row = (which * a.hk + kvh) * a.page_size + b_off;
      if (!bar_wait(E4M3 ? &taken[slot] : &empty[slot], (uses & 1) ^ 1, abort_flag)) {
        set_error(a.err, ERR_WAIT_EMPTY);
        *abort_flag = 1;
        ok = false;
        break;
      }
      // boxes behind the share's end are not brought
      if (lane == 0) mbar_expect_tx(&came[slot], boxes * box * D * (E4M3 ? 1 : 2));
      __syncwarp();
      if (lane < boxes) {
#pragma unroll
        for (int cb = 0; cb < (E4M3 ? 2 : 4); ++cb)
          tma_load_3d((E4M3 ? c_s + slot * Cfg::kCodes : h_s + slot * Cfg::kHalf) + cb * kBlock + lane * box * 128, kv_map, cb * (E4M3 ? 128 : 64), b_row, b_page,
                      &came[slot]);
      }
      if constexpr (E4M3) {
        const int s_page = __shfl_sync(0xffffffffu, page, (lane >> 1) & 7), s_off = __shfl_sync(0xffffffffu, off, (lane >> 1) & 7) + (lane & 1) * 4;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (k && which) break;
          const uint8_t* src = a.pool + (size_t)s_page * page_bytes + codes + (size_t)((k ? 1 : which) * a.hk + kvh) * a.page_size + s_off;
          if (4 * lane < here && KERN_CHECK(src, 4, SITE_KV_ROW))
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(b_s + slot * 2 * kKeys + k * kKeys + 4 * lane)), "l"(src) : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&came[slot])) : "memory");
      }
    }
  } else if (warp == 16) {
    // ---------------- products: the whole warp walks and waits, one lane issues ----------------
    constexpr uint32_t idesc_qk = tile_idesc<E4M3>(kQRows, kKeys, false), idesc_pv = tile_idesc<E4M3>(kQRows, D, true);
    const uint32_t q_low = desc_low(smem_u32(q_s), 0), h_low = desc_low(smem_u32(h_s), 0), v_low = desc_low(smem_u32(h_s), kBlock);
    const bool leader = elect_lane();
    float ev_least = 255.f, ev_most = -255.f;                 // (8-bit) the value tiles' exponents
    auto qk = [&](int t) -> bool {
      const int i = k_item(t), half = i % kRing;
      if (!bar_wait(&full[half], (i / kRing) & 1, abort_flag)) return false;
      tc_fence_after();
      const uint32_t sk = h_low + half * (Cfg::kHalf >> 4), s_t = tmem + D + (t & 1) * kKeys;
      if (leader) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_ss(s_t, q_low + ((k >> 2) * kQBlock + (k & 3) * 32 >> 4), sk + ((k >> 2) * kBlock + (k & 3) * 32 >> 4), idesc_qk, k != 0);
        tc_commit(&s_full[t & 1]);
        tc_commit(&empty[half]);
      }
      __syncwarp();
      if constexpr (E4M3) {
        // (here, where a few instructions make nobody wait, as in attn_tile.cu)
        const float ev = fmaxf(e_s[t & 3].y, kLeastShift);
        ev_least = fminf(ev_least, ev);
        ev_most = fmaxf(ev_most, ev);
        if (ev_most - ev_least > (float)kTilesApart) *wide_s = 1;
      }
      return true;
    };
    auto pv = [&](int t) -> bool {
      const int i = v_item(t), half = i % kRing;
      if (!bar_wait(&full[half], (i / kRing) & 1, abort_flag)) return false;
      if (!bar_wait(&p_full[t & 1], (t >> 1) & 1, abort_flag)) return false;
      tc_fence_after();
      const uint32_t sv = v_low + half * (Cfg::kHalf >> 4), p_t = tmem + D + (t & 1) * kKeys;
      if (leader) {
        // (a thread's 32 columns are two steps, in 16 of its 32 places)
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k) umma_ts(tmem, p_t + (k < 2 ? k : k + 2) * 8, sv + (k * 16 * 128 >> 4), idesc_pv, (t | k) != 0);
        tc_commit(&empty[half]);
        tc_commit(&o_quiet[t & 1]);
      }
      __syncwarp();
      return true;
    };
    if (ntiles > 0) ok = bar_wait(q_full, 0, abort_flag) && qk(0);
    if (ok && ntiles > 1) ok = qk(1);
    for (int t = 0; t < ntiles && ok; ++t) {
      ok = pv(t);
      if (ok && t + 2 < ntiles) ok = qk(t + 2);               // (overwrites the scores whose weights P V has just been given)
    }
    if (!ok) {
      set_error(a.err, ERR_WAIT_FULL);
      *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp < 8) {
    // ---------------- Q -> shared memory, K-major with the 128-byte swizzle: a warp to a row ----------------
    const float per_g = 1.f / (float)G;
    const __nv_bfloat16* q_at = a.q + (size_t)(row0 + tok_lo) * a.q_stride + (size_t)kvh * G * D + lane * 8;
#pragma unroll 1
    for (int r1 = warp; r1 < kQRows; r1 += 64) {
      uint4 rows[8];                                          // (all under way together)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r1 + i * 8;
        const int tok = (int)((r + 0.5f) * per_g), head = r - tok * G;        // (r / G, exact: r < 128)
        rows[i] = make_uint4(0, 0, 0, 0);
        if (r < valid) rows[i] = *reinterpret_cast<const uint4*>(q_at + (size_t)tok * a.q_stride + head * D);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r1 + i * 8;
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
          top = warp_max(top);
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
        *reinterpret_cast<uint4*>(q_s + (lane >> 3) * kQBlock + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = v;
        if (lane == 0) x_s[r] = f;
      }
    }
    fence_proxy_async();
    mbar_arrive(q_full);
    asm volatile("bar.sync 15, 256;" ::: "memory");           // x_s
    // ---------------- softmax: two threads to a row, half of a tile's scores each ----------------
    const int part = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, o_t = tmem + lanes + part * (D / 2);
    const int tk = tok_lo + (row < valid ? row / G : 0), pos = past + tk;
    const long long* mask = TREE ? a.masks + (size_t)(row0 + tk) * a.words : nullptr;
    const float f = x_s[row];                                 // (read before the row's threads meet, written after)
    float* const own_x = x_s + part * kQRows + row;           // what the row's two threads tell each other
    float* const his_x = x_s + (1 - part) * kQRows + row;
    const int pair = 1 + (warp & 3);                          // barrier of the two warps that share 32 rows
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory"); };
    auto any_of = [&](bool mine) -> bool {                    // over the two warps' threads
      uint32_t any;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(any)
                   : "r"(pair), "r"((uint32_t)mine)
                   : "memory");
      return any != 0;
    };
    constexpr float kGrown = E4M3 ? 15.9f : 30.f, kBelow = E4M3 ? 5.f : 0.f;      // (attn_tile.cu)
    float ref = kUnset, l = 0.f;                              // l: of this thread's columns
    // P V of tile t has ended (that of tile t - 2, whose place the scores of tile t took, has before those came)
    auto quiet = [&](int t) -> bool { return bar_wait(&o_quiet[t & 1], (t >> 1) & 1, abort_flag); };
    // (a wait that has run out does not leave the walk: the two warps meet in every step)
    for (int t = 0; t < ntiles; ++t) {
      const int tok0 = from + t * kKeys;
      const uint32_t s_t = tmem + lanes + D + (t & 1) * kKeys + part * 32;
      if (ok && !bar_wait(&s_full[t & 1], (t >> 1) & 1, abort_flag)) {
        set_error(a.err, ERR_WAIT_TMEM_FULL);
        *abort_flag = 1;
        ok = false;
      }
      tc_fence_after();
      float scale = f, ev = 0.f;
      if constexpr (E4M3) {
        const float2 e = e_s[t & 3];
        scale = row_scale(f, e.x);
        ev = fmaxf(e.y, kLeastShift);
      }
      uint32_t x[32];
      tmem_ld_32x32(s_t, x);
      tmem_ld_wait();
      if (tok0 + kKeys > clear) {                             // (uniform) rows see different tokens
        const uint32_t b = seen32<TREE>(mask, a.words, past, pos, to, tok0 + part * 32);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!(b >> i & 1)) x[i] = 0xff800000u;
      }
      float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 32; i += 2) m2[(i >> 1) & 1] = max3(m2[(i >> 1) & 1], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
      float mx = fmaf(fmaxf(m2[0], m2[1]), scale, ev);
      if (any_of(mx > ref + kGrown)) {
        // a row's two threads move its reference together, and each passes over half of O once the P V before has ended
        *own_x = mx;
        meet();
        mx = fmaxf(mx, *his_x);
        const float to_ref = mx > ref + kGrown ? ceilf(mx) - kBelow : ref, corr = exp2f(ref - to_ref);
        ref = to_ref;
        l *= corr;
        if (t > 0) {
          if (ok && !quiet(t - 1)) {
            set_error(a.err, ERR_WAIT_TMEM_FULL);
            *abort_flag = 1;
            ok = false;
          }
          tc_fence_after();
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
      const uint64_t scale2 = pair64(scale, scale), shift2 = pair64(ev - ref, ev - ref);
      uint64_t sum2[2] = {0, 0};
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 y = split64(fma2(pair64(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2, shift2));
        const float u = exp2f(y.x), v = exp2f(y.y);
        pk[i] = pack_pair<E4M3>(u, v);
        sum2[i & 1] = add2(sum2[i & 1], E4M3 ? pair64(u, v) : pair64(__uint_as_float(pk[i] << 16), __uint_as_float(pk[i] & 0xffff0000u)));
      }
      tmem_st16(s_t, pk);
      const float2 sum = split64(add2(sum2[0], sum2[1]));
      l += E4M3 ? (sum.x + sum.y) * exp2f(-ev) : sum.x + sum.y;
      tmem_st_done();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t & 1]);
    }
    if (ok && ntiles > 0 && !quiet(ntiles - 1)) {
      set_error(a.err, ERR_WAIT_TMEM_FULL);
      *abort_flag = 1;
      ok = false;
    }
    tc_fence_after();
    // ---------------- the rows' end: half of the columns to each of a row's threads ----------------
    *own_x = l;
    meet();
    l += *his_x;
    if (E4M3 && *wide_s != 0) {                               // (uniform: every half has been looked at)
      if constexpr (E4M3) {
        const RowsArgs args = a;                              // (a copy on the stack, for this call alone)
        if (ok) tile_wide<D, TREE>(args, seq, row0, tok_lo, valid, past, from, to, shares, 8);
      }
    } else {
      const bool whole = shares == 1, store = row < valid && ok, bad = *bad_s != 0;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float level = E4M3 && !whole ? level_share(ref, l) : 1.f;
      const int head = kvh * G + (row < valid ? row % G : 0);
      const size_t at = (ws_row(a.ws_step, seq, row0, tk) * a.hq + head) * gridDim.z + blockIdx.z;
#pragma unroll 1
      for (int c = 0; c < D / 2; c += 32) {
        const int col = part * (D / 2) + c;
        uint32_t x[32];
        tmem_ld_32x32(o_t + c, x);
        tmem_ld_wait();
        if (ntiles == 0) {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0;
        }
        if (bad && store) put_back<D, E4M3, TREE>(a, mask, seq, past, pos, from + max(clear - from, 0) / kKeys * kKeys, to, col, x);
        if (!store) continue;
        if (whole) {
          __nv_bfloat16* dst = a.out + (size_t)(row0 + tk) * a.out_stride + (size_t)head * D + col;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              o[k] = l == 0.f ? 0u : pack_bf16x2(__uint_as_float(x[8 * i + 2 * k]) * inv, __uint_as_float(x[8 * i + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + i * 8) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        } else {
          uint4* dst = reinterpret_cast<uint4*>(a.ws_o + at * D + col);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (E4M3) {
#pragma unroll
              for (int k = 0; k < 4; ++k) x[4 * i + k] = __float_as_uint(__uint_as_float(x[4 * i + k]) * level);
            }
            dst[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          }
        }
      }
      if (!whole && store && part == 0) {
        a.ws_ml[at * 2] = ref;
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
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace kern

using namespace kern;

#define KERN_TILE256_ENTRY(KIND, E4M3, FORM, TREE)                                                                                \
  extern "C" __global__ void __launch_bounds__(kWideThreads, 1) kern_attn_tile_##KIND##_##FORM##_d256(                            \
      const __grid_constant__ CUtensorMap kv_map, const __nv_bfloat16* q, __nv_bfloat16* out, float* ws_o, float* ws_ml,          \
      const uint8_t* pool, const int* block_table, const int* seq_lens, const int* cu_q, const long long* masks, int words,       \
      int rows_per_seq, int hq, int hk, int q_stride, int out_stride, int max_pages, int page_size, int seqs, int pool_pages,     \
      int row_lo, int row_hi, int rows, int max_rows, int ws_step, float scale_log2, int* err) {                                               \
    tile256_body<E4M3, TREE>(&kv_map, RowsArgs{q, out, ws_o, ws_ml, pool, block_table, seq_lens, cu_q, masks, err, words,         \
                                               rows_per_seq, hq, hk, q_stride, out_stride, max_pages, page_size, 1, pool_pages,   \
                                               row_lo, row_hi, rows, max_rows, ws_step, scale_log2},                                       \
                             seqs);                                                                                               \
  }
KERN_TILE256_ENTRY(e4m3, true, causal, false)
KERN_TILE256_ENTRY(e4m3, true, tree, true)
KERN_TILE256_ENTRY(bf16, false, tree, true)
