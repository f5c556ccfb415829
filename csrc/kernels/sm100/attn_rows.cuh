// What the kernels of attention over a cache in either format share (attn_rows.cu: few query rows, attn_tile.cu: many): their
// arguments, conversions, and how a context is dealt out.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace kern {

constexpr float kUnset = -1e30f;     // a reference before its first score
constexpr float kOutgrown = 32768.f; // the weight at which references move: f16 holds twice that

// the scale byte of a row of zeros, and of the smallest rows: -40 + 127. A page that nobody has written to has bytes of 0 (and codes of
// 0): references and a value tile's exponent take these for the least, or what undoes their 2^-127 would pass f32's range
constexpr int kLeastScale = 87;

struct RowsArgs {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  float* ws_o;               // partials [place][head][groups][D] (one group: none)
  float* ws_ml;              // [place][head][groups][2]
  const uint8_t* pool;       // (8-bit) scale bytes are read from here
  const int* block_table;
  const int* seq_lens;
  const int* cu_q;
  const long long* masks;    // (tree) [row][words]
  int* err;
  int words, rows_per_seq, hq, hk, q_stride, out_stride, max_pages, page_size, cluster, pool_pages;
  int row_lo, row_hi;        // sequences of other row counts are another launch's
  int rows;                  // of q and out: a sequence's have to lie in them
  int max_rows;              // the most rows of one sequence, by which blocks were counted
  int ws_step;               // places of partials to a sequence; 0: they lie as the rows of q
  float scale_log2;
};

// A wait bounded by the SM's own clock (some 2 s), which is read in a few cycles.
KERN_DEVICE bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 0x3f) == 0x3f && (*abort_flag != 0 || clock64() - t0 > 4000000000ll)) return false;
  }
}

// four e4m3 codes -> two pairs of f16, exact
KERN_DEVICE void codes_f16x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
KERN_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool F16>
KERN_DEVICE uint32_t pack_pair(float lo, float hi) {
  if constexpr (F16) return pack_f16x2(lo, hi);
  else return pack_bf16x2(lo, hi);
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

// A sequence's tokens: no more than its row of the table has pages for, or a length that is not one would be walked to its end, seconds
// of it. (capacity: below 2^31 - 256, so that lengths can be rounded up)
KERN_DEVICE int within(int len, int capacity) { return min(max(len, 0), capacity); }
KERN_DEVICE int context_of(const RowsArgs& a, int seq) {
  const int len = a.seq_lens[seq], capacity = a.max_pages * a.page_size;
  if (len > capacity) set_error(a.err, ERR_BOUNDS);
  return within(len, capacity);
}

// whether R rows from row0 on are rows of the call, and no more than it has said
KERN_DEVICE bool rows_lie(int row0, int R, int rows, int max_rows) { return row0 >= 0 && R >= 0 && R <= rows - row0 && R <= max_rows; }

// where the partials of a sequence's row `tok` lie: q may have many rows that are nobody's in this call
KERN_DEVICE size_t ws_row(int ws_step, int seq, int row0, int tok) { return ws_step ? (size_t)seq * ws_step + tok : (size_t)(row0 + tok); }

KERN_DEVICE float pow2i(int e) { return __uint_as_float((uint32_t)(min(max(e, -126), 127) + 127) << 23); }

// A context is dealt out in runs of whole 128-token units: how many shares `end` tokens are cut into, and the tokens
// of each.
KERN_DEVICE int rows_shares(int end, int splits) { return min(splits, max(1, (end + 127) / 128)); }
KERN_DEVICE int rows_share_len(int end, int shares) { return ((end + 127) / 128 + shares - 1) / shares * 128; }

KERN_DEVICE unsigned sm_count() {
  unsigned n;
  asm("mov.u32 %0, %%nsmid;" : "=r"(n));
  return n;
}
// Of n <= 256 sequences (and a thread to each): the rank of this thread's by length, the longest first; -1 in further threads. Every
// thread of the block calls; keys: 256 places in shared memory.
KERN_DEVICE int by_length(const int* seq_lens, int n, int* keys) {
  const int t = threadIdx.x, own = t < n ? min(max(seq_lens[t], 0), 0x7fffff) << 8 | (255 - t) : -1;
  if (t < 256) keys[t] = own;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < n; i += 4) {
    const int4 k = *reinterpret_cast<const int4*>(keys + i);
    before += (k.x > own) + (k.y > own) + (k.z > own) + (k.w > own);
  }
  return t < n ? before : -1;
}

}  // namespace kern
