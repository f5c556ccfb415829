// The host side of the operators whose calls are as short as their launches: 8-bit caching, attention over either cache, drafted
// trees. A call checks its tensors, allocates what it returns, packs the kernel's parameter block and launches it, all here: in
// Python the same took two to four times the kernel's own time at small sizes. Linked against PyTorch's libraries (tensors,
// allocator, current stream); kernels are those that `kern_b200.ops.launcher` has loaded, and are launched through the same device
// layer.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/full.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cmath>
#include <cstring>
#include <memory>
#include <optional>
#include <string>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "runtime/device.hpp"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

constexpr int64_t kTile = 64, kMaxNodes = 256, kMaxPools = 128;
constexpr double kLog2e = 1.4426950408889634;

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }
std::string n(int64_t v) { return std::to_string(v); }

// ---- one GPU's kernels -----------------------------------------------------------------------------------------------------------
struct Host {
  std::shared_ptr<kern::Device> dev;
  int sms = 0;
  uint64_t err = 0;
  py::object resolve;                                        // (module, entry) -> function handle
  std::unordered_map<std::string, CUfunction> functions;
  int64_t launches = 0;

  CUfunction function(const char* module, const std::string& entry) {
    auto it = functions.find(entry);
    if (it != functions.end()) return it->second;
    const CUfunction f = reinterpret_cast<CUfunction>(resolve(module, entry).cast<uint64_t>());
    functions.emplace(entry, f);
    return f;
  }
};
std::array<std::unique_ptr<Host>, 64>& hosts() {
  static std::array<std::unique_ptr<Host>, 64> h;
  return h;
}
py::object& missing() {
  static py::object* f = new py::object();                   // (never freed: the interpreter may be gone by then)
  return *f;
}
Host& host_of(int gpu) {
  if (gpu >= (int)hosts().size()) refuse("device index " + n(gpu));
  if (!hosts()[gpu]) missing()(gpu);
  if (!hosts()[gpu]) throw std::runtime_error("no kernels for GPU " + n(gpu));
  return *hosts()[gpu];
}

// A kernel's parameters, each at its natural alignment.
struct Block {
  alignas(64) uint8_t data[2048];
  size_t size = 0;
  template <typename T>
  Block& put(const T& v) {
    size = (size + alignof(T) - 1) / alignof(T) * alignof(T);
    std::memcpy(data + size, &v, sizeof(T));
    size += sizeof(T);
    return *this;
  }
  Block& at(const Tensor& t) { return put<uint64_t>(reinterpret_cast<uint64_t>(t.data_ptr())); }
  Block& at(const Maybe& t) { return put<uint64_t>(t ? reinterpret_cast<uint64_t>(t->data_ptr()) : 0); }
  template <typename... I>
  Block& ints(I... v) {
    (put<int32_t>((int32_t)v), ...);
    return *this;
  }
  Block& bytes(const void* p, size_t count) {
    std::memcpy(data + size, p, count);
    size += count;
    return *this;
  }
};

void launch(Host& h, const char* module, const std::string& entry, int64_t gx, int64_t gy, int64_t gz, unsigned threads, Block& b,
            unsigned shared = 0, bool pdl = false, unsigned cluster = 1) {
  kern::LaunchDims dims;
  dims.grid[0] = (unsigned)gx;
  dims.grid[1] = (unsigned)gy;
  dims.grid[2] = (unsigned)gz;
  dims.block[0] = threads;
  dims.cluster[2] = cluster;
  dims.shared_mem = shared;
  dims.pdl = pdl;
  h.dev->launch(h.function(module, entry), dims, c10::cuda::getCurrentCUDAStream(h.dev->gpu()).stream(), nullptr, b.data, b.size);
  ++h.launches;
}

// ---- checks ----------------------------------------------------------------------------------------------------------------------
bool whole(const Tensor& t) { return t.is_contiguous(); }
bool on16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// a bf16 row tensor that the kernels read 16 bytes at a time; (rows, elements from one row to the next)
std::pair<int64_t, int64_t> rows_of(const Tensor& t, int64_t width, const char* name) {
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 2) refuse(std::string(name) + " is a bf16 [rows, >= " + n(width) + "] tensor");
  if (t.size(1) < width || (t.stride(1) != 1 && t.size(1) > 1)) refuse(std::string(name) + " is a bf16 [rows, >= " + n(width) + "] tensor whose columns are neighbours");
  if ((t.size(0) > 1 && (t.stride(0) % 8 || t.stride(0) < width)) || !on16(t)) refuse(std::string(name) + ": rows start on 16 bytes and do not overlap");
  if (t.stride(0) > INT32_MAX) refuse(std::string(name) + ": rows too far apart");
  return {t.size(0), t.size(0) > 1 ? t.stride(0) : width};
}
void numbers(const Tensor& t, at::ScalarType type, int64_t count, const char* name) {
  if (t.scalar_type() != type || t.numel() < count || !whole(t)) refuse(std::string(name) + ": contiguous " + (type == at::kInt ? "i32" : "i64") + ", " + n(count) + " of them");
}
void table_of(const Tensor& t, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || !whole(t)) refuse(std::string(name) + ": contiguous i32 [seqs, pages]");
  if (t.size(0) > 65535 || (t.size(0) > 0 && t.size(1) < 1)) refuse(std::string(name) + " [" + n(t.size(0)) + ", " + n(t.size(1)) + "]: at most 65535 sequences, a page to a row");
}
void heads(int64_t hq, int64_t hk, int64_t d, int64_t page, bool attends) {
  if (hk < 1 || hq < 1 || hq % hk || (attends && hq > 16 * hk))
    refuse(n(hq) + " query heads over " + n(hk) + " kv heads: a whole group" + (attends ? " of at most 16" : ""));
  if (d != 64 && d != 128 && d != 256) refuse("head_dim " + n(d) + ": built for 64, 128, 256");
  if (page < 8 || (page <= kTile ? kTile % page : page % kTile)) refuse("page_size " + n(page) + ": 8, 16, 32, or a multiple of 64");
  if (hq > 4096 || page > (1 << 20) || 2 * hk * page * (d + 1) > INT32_MAX) refuse("heads or pages past 32 bits");
}
// pages of a pool in the 8-bit format, or in either
int64_t pages8(const Tensor& p, int64_t hk, int64_t page, int64_t d) {
  const int64_t bytes = 2 * hk * page * (d + 1);
  if (p.scalar_type() != at::kByte || p.dim() != 2 || p.size(1) != bytes || !whole(p))
    refuse("an 8-bit pool is a contiguous uint8 [pages, " + n(bytes) + "] tensor for these heads and pages");
  if (p.size(0) < 1 || !on16(p)) refuse("the pool has a page, and starts on 16 bytes");
  if (p.size(0) * page > INT32_MAX) refuse("a pool of 2^31 tokens or more");
  return p.size(0);
}
int64_t pages_any(const Tensor& p, int64_t hk, int64_t page, int64_t d) {
  if (p.scalar_type() == at::kByte) return pages8(p, hk, page, d);
  if (p.scalar_type() != at::kBFloat16 || p.dim() != 5 || p.size(1) != 2 || p.size(2) != hk || p.size(3) != page || p.size(4) != d || !whole(p))
    refuse("a bf16 pool is a contiguous [pages, 2, " + n(hk) + ", " + n(page) + ", " + n(d) + "] tensor");
  if (p.size(0) < 1 || !on16(p)) refuse("the pool has a page, and starts on 16 bytes");
  if (p.size(0) * page > INT32_MAX) refuse("a pool of 2^31 tokens or more");
  return p.size(0);
}
struct Same {
  int gpu;
  explicit Same(const Tensor& t) : gpu(t.is_cuda() ? t.get_device() : -1) {
    if (gpu < 0) refuse("the tensors of this call live on a CUDA device");
  }
  Same& operator()(const Tensor& t) {
    if (!t.is_cuda() || t.get_device() != gpu) refuse("the tensors of a call live on one device");
    return *this;
  }
  Same& operator()(const Maybe& t) { return t ? (*this)(*t) : *this; }
};
at::TensorOptions typed(const Tensor& like, at::ScalarType type) { return like.options().dtype(type).layout(at::kStrided).requires_grad(false); }

// ---- the 8-bit cache ----------------------------------------------------------------------------------------------------------------
Tensor append(const Tensor& qkv, const Tensor& pool, const Tensor& positions, const Tensor& slots, const Tensor& cos, const Tensor& sin, int64_t hq,
              int64_t hk, int64_t d, int64_t page, std::optional<int64_t> rot_, const std::string& pairs, const Maybe& q_norm, const Maybe& k_norm,
              double eps, bool plus_one, std::optional<int64_t> tokens, const Maybe& q_out) {
  heads(hq, hk, d, page, false);
  const int64_t pages = pages8(pool, hk, page, d);
  auto [t, step] = rows_of(qkv, (hq + 2 * hk) * d, "qkv");
  if (tokens) {
    if (*tokens < 0 || *tokens > t) refuse(n(*tokens) + " tokens of " + n(t) + " rows");
    t = *tokens;
  }
  const int64_t rot = rot_.value_or(d);
  if (rot < 0 || rot > d || rot % 16) refuse("rot " + n(rot) + ": a multiple of 16 up to the head's " + n(d));
  if (pairs != "half" && pairs != "interleaved") refuse("pairs '" + pairs + "': half or interleaved");
  numbers(positions, at::kLong, t, "positions");
  numbers(slots, at::kLong, t, "slots");
  for (const Tensor* x : {&cos, &sin})
    if (x->scalar_type() != at::kFloat || x->dim() != 2 || !whole(*x) || x->size(1) != rot / 2 || !on16(*x))
      refuse("cos and sin: contiguous f32 [max_pos, rot / 2] tables");
  const int64_t max_pos = cos.size(0);
  if (max_pos < 1 || sin.size(0) != max_pos || max_pos > INT32_MAX) refuse("the tables have the same positions, one at least");
  for (const Maybe* x : {&q_norm, &k_norm})
    if (*x && ((*x)->scalar_type() != at::kBFloat16 || (*x)->numel() != d || !whole(**x) || !on16(**x))) refuse("q_norm and k_norm: bf16 [" + n(d) + "]");
  const Tensor& dst = q_out ? *q_out : qkv;
  int64_t dst_step = step;
  if (q_out) {
    const auto [m, s] = rows_of(dst, hq * d, "q_out");
    if (m < t) refuse("q_out has a row for each token");
    dst_step = s;
  }
  const int gpu = Same(qkv)(pool)(positions)(slots)(cos)(sin)(q_norm)(k_norm)(dst).gpu;
  if (t) {
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)gpu);
    Host& h = host_of(gpu);
    Block b;
    b.at(qkv).at(dst).at(pool).at(positions).at(slots).at(cos).at(sin).at(q_norm).at(k_norm).ints(hq, hk, rot, page).put((float)eps).ints(plus_one);
    b.put<int64_t>(pages * page).ints(max_pos, step, dst_step).put(h.err);
    launch(h, "kv_e4m3", "kern_rope_kv_append_e4m3_" + pairs + (q_norm || k_norm ? "_norm_d" : "_d") + n(d), t, 1, 1, 128, b);
  }
  if (dst.size(0) == t && dst.size(1) == hq * d) return dst;
  return dst.narrow(0, 0, t).narrow(1, 0, hq * d);
}

Tensor read_rows(const Tensor& pool, const Tensor& slots, int64_t hk, int64_t d, int64_t page, const Maybe& out_) {
  heads(hk, hk, d, page, false);
  const int64_t pages = pages8(pool, hk, page, d);
  if (slots.scalar_type() != at::kLong || slots.dim() != 1 || !whole(slots)) refuse("slots: i64 [tokens]");
  const int64_t t = slots.numel();
  if (out_ && (out_->scalar_type() != at::kBFloat16 || out_->dim() != 4 || out_->size(0) != t || out_->size(1) != 2 || out_->size(2) != hk ||
               out_->size(3) != d || !whole(*out_) || !on16(*out_)))
    refuse("out: contiguous bf16 [" + n(t) + ", 2, " + n(hk) + ", " + n(d) + "]");
  const int gpu = Same(pool)(slots)(out_).gpu;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)gpu);
  const Tensor out = out_ ? *out_ : at::empty({t, 2, hk, d}, typed(pool, at::kBFloat16));
  if (t) {
    Host& h = host_of(gpu);
    Block b;
    b.at(pool).at(slots).at(out).ints(t, hk, page).put<int64_t>(pages * page).put(h.err);
    launch(h, "kv_e4m3", "kern_kv_read_e4m3_d" + n(d), t, 1, 1, 128, b);
  }
  return out;
}

// ---- attention ------------------------------------------------------------------------------------------------------------------------
// The few-row kernel with 8 * nt query rows to a CTA: dynamic shared memory (a ring of tiles of 128 tokens, 64 where a row is over
// 128 bytes; scale bytes; Q's fragments at head_dim 256 and 16 rows; barriers), and CTAs on an SM.
struct RowsForm {
  unsigned shared;
  int per_sm;
};
RowsForm rows_form(int64_t d, bool e4m3, int64_t nt) {
  const int64_t row = d * (e4m3 ? 1 : 2), tile = row <= 128 ? 128 : 64, stage = 2 * tile * row;
  const int per_sm = d == 256 ? 1 : 2;
  const int64_t stages = stage >= 65536 ? 3 : (per_sm == 1 ? 196608 : 98304) / stage;
  return {(unsigned)(1024 + stages * (stage + (e4m3 ? 2 * tile : 0)) + (d == 256 && nt > 1 ? nt * d * 16 : 0) + 256), per_sm};
}
// Shares that a row's context is cut into, and CTAs of a cluster: as many as fill the SMs once, none of under 128 tokens, and one where
// the rows alone fill them, the longest first then. Up to 8 shares are one cluster; more are on their own, and joined by a second
// launch. Microseconds of decode, 8 kv heads, head_dim 128, by shares (* the rule's):
//   sequences of tokens    1      2      4      8     16     32          sequences of tokens (ragged: up to)    1       2       4
//     1 of 1000          10.6    9.8    8.6    7.8*                       64 of 4000                            90.9*  101.6   114.6
//     1 of 30000          192    100   54.1   31.5   20.1   19.0*         64 of up to 4000                      48.3*   60.2    81.5
//     4 of 4000          30.1   18.8   12.9   13.1*  15.5                 48 of up to 4000                      41.0*   54.9    66.0
//    16 of 4000          32.7   29.5*  34.8   47.1   45.0                 48 of 4000                            86.8*   79.0    89.7
//     2 of 100000         631    324    166    116   71.7*  77.4          128 of up to 8000                    167.9*  183.5   225.3
std::pair<int64_t, int64_t> rows_shares(int64_t ctas, int64_t max_len, int64_t resident) {
  const int64_t most = std::max<int64_t>(1, (max_len + 127) / 128);
  const int64_t want = std::min<int64_t>({most, std::max<int64_t>(1, resident / ctas), 256});
  if (want > 8) return {want, 1};
  const int64_t cluster = want >= 8 ? 8 : want >= 4 ? 4 : want >= 2 ? 2 : 1;
  return {cluster, cluster};
}
// The many-row kernels: two tiles of Q (head_dim 256: one, and halves of 64 tokens), a ring of K and V halves as 16-bit values (four, or five where they are copied as they are),
// two halves of codes with their scale bytes, barriers.
int64_t tile_rows(int64_t d) { return d == 256 ? 128 : 256; }        // query rows of a CTA
int64_t tile_threads(int64_t d) { return d == 256 ? 576 : 768; }
const char* tile_module(int64_t d) { return d == 256 ? "attn_tile256" : "attn_tile"; }
unsigned tile_shared(int64_t d, bool e4m3) {
  if (d == 256) return (unsigned)(128 * d * 2 + (e4m3 ? 4 : 5) * 64 * d * 2 + (e4m3 ? 2 * (64 * d + 128) : 0) + 2 * 128 * 4 + 512);
  return (unsigned)(2 * 128 * d * 2 + (e4m3 ? 4 : 5) * 128 * d * 2 + (e4m3 ? 2 * (128 * d + 256) : 0) + 4 * 128 * 4 + 512);
}
// Shares of the many-row kernel: as many as fill the SMs once. Microseconds, 64 rows of 4 heads each, by shares (* the rule's):
//   sequences of tokens    1      2      4      8     16     32
//     1 of 8000           134   78.6   48.3   33.9   28.3*  43.8
//     4 of 4000          76.2   56.9   42.2*  56.5   86.0
//     9 of 4000          77.4   69.2*  82.7    112
//    16 of 4000          79.1*   127    154
// (a CTA takes the SM's whole memory, so a second wave begins with copies that nothing hides)
int64_t tile_shares(int64_t ctas, int64_t max_len, int64_t sms) {
  return std::max<int64_t>(1, std::min<int64_t>({sms / ctas, (max_len + 255) / 256, 64}));
}
// Query rows of a sequence and kv head up to which the few-row kernel runs; the many-row kernel above them.
// Microseconds of the few-row kernel : of the many-row kernel, 8 kv heads, head_dim 128:
//   8-bit cache, causal          16 rows       32 rows            bf16 cache, tree       16 rows       24 rows
//     1 sequence  of 1000      10.0 :  13.1   14.4 :  14.0           1 of 1000           10.4 :  11.8    14.0 :  11.9
//    16 sequences of 4000      39.0 :  74.9   74.2 :  75.1          16 of 4000           47.9 :  46.6    85.0 :  46.6
//    64 sequences of 2000      88.8 : 159     206  : 161            64 of 2000          106.8 : 107.2   216.8 : 107.8
// and head_dim 256, 16 sequences of 4000: 12 rows 42.5 : 54.3, 18 rows 66.0 : 54.8.
// (the few-row kernel's matrix instructions take time for every eight rows, the other's are the same up to 128)
constexpr int64_t kFewRows = 16;

// 3-D descriptor over a pool of either format: (value, row of a page's k | v x head x token, page)
std::array<uint8_t, 128> pool_map(Host& h, const Tensor& pool, bool e4m3, int64_t pages, int64_t hk, int64_t d, int64_t page) {
  const int64_t es = e4m3 ? 1 : 2, cols = std::min<int64_t>(d * es, 128);
  kern::TensorMapSpec s;
  s.dtype = e4m3 ? 0 : 9;                                    // u8, bf16
  s.dims = {(uint64_t)d, (uint64_t)(2 * hk * page), (uint64_t)pages};
  s.strides = {(uint64_t)(d * es), (uint64_t)(e4m3 ? 2 * hk * page * (d + 1) : 2 * hk * page * d * 2)};
  s.box = {(uint32_t)(cols / es), (uint32_t)std::min<int64_t>(page, kTile), 1};
  s.swizzle = (int)cols;
  s.l2_promotion = 256;
  s.oob_nan = false;
  return h.dev->encode_tensor_map(reinterpret_cast<uint64_t>(pool.data_ptr()), s);
}

Tensor attend(const Tensor& q, const Tensor& pool, const Tensor& table, const Tensor& lens, const Maybe& masks, const Maybe& cu_q, int64_t hq,
              int64_t hk, int64_t d, int64_t page, const Maybe& out_, int64_t rows_per_seq, std::optional<int64_t> max_rows_, std::optional<int64_t> max_len_,
              std::optional<double> scale_) {
  heads(hq, hk, d, page, true);
  const int64_t pages = masks ? pages_any(pool, hk, page, d) : pages8(pool, hk, page, d);
  const bool e4m3 = pool.scalar_type() == at::kByte;
  const auto [rows, q_step] = rows_of(q, hq * d, "q");
  table_of(table, "block_table");
  const int64_t seqs = table.size(0), width = table.size(1);
  numbers(lens, at::kInt, seqs, "seq_lens");
  int64_t max_rows = rows_per_seq;
  if (cu_q) {
    numbers(*cu_q, at::kInt, seqs + 1, "cu_q");
    rows_per_seq = 1;
    max_rows = max_rows_.value_or(rows);
  } else if (masks) {
    refuse("cu_q: i32 [seqs + 1]");
  } else if (rows_per_seq < 1 || rows < seqs * rows_per_seq) {
    refuse("q has rows_per_seq rows for each sequence");
  }
  if (seqs && (max_rows < 0 || max_rows > rows)) refuse("max_rows " + n(max_rows) + ": the most rows of one sequence, of " + n(rows));
  if (masks && (masks->scalar_type() != at::kLong || masks->dim() != 2 || masks->size(0) < rows || masks->size(1) < 1 || masks->size(1) > kMaxNodes / 64 || !whole(*masks)))
    refuse("masks: contiguous i64 [rows, words], up to " + n(kMaxNodes / 64) + " words");
  int64_t out_step = hq * d;
  if (out_) {
    const auto [m, s] = rows_of(*out_, hq * d, "out");
    if (m < rows) refuse("out has a row for each of q's");
    out_step = s;
  }
  if (width * page > INT32_MAX - 256) refuse("a table of " + n(width) + " pages: contexts past 32 bits");
  const int64_t max_len = max_len_.value_or(width * page);
  if (max_len < 0) refuse("max_len " + n(max_len));
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)d);
  const float scale_log2 = (float)(scale * kLog2e);
  if (!(scale > 0) || !std::isnormal(scale_log2)) refuse("scale: above zero, and a number that f32 holds");
  const int gpu = Same(q)(pool)(table)(lens)(cu_q)(masks)(out_).gpu;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)gpu);
  const Tensor out = out_ ? *out_ : at::empty({rows, hq * d}, typed(q, at::kBFloat16));
  if (!seqs || !rows) return out;
  Host& h = host_of(gpu);
  const int64_t g = hq / hk;
  const auto map = pool_map(h, pool, e4m3, pages, hk, d, page);
  const std::string form = std::string(e4m3 ? "_e4m3" : "_bf16") + (masks ? "_tree_d" : "_causal_d") + n(d);
  const int64_t all = INT32_MAX, few = std::max<int64_t>(1, 8 / g);
  // one kernel over the sequences of lo .. hi rows
  auto run = [&](bool tiled, int64_t lo, int64_t hi) {
    const int64_t most = std::max<int64_t>(1, std::min(max_rows, hi));       // (max_rows 0: the kernels see whether that is so)
    int64_t toks, cluster = 1, shares, gx, gy;
    unsigned shared;
    std::string name;
    if (tiled) {
      toks = tile_rows(d) / g;
      gy = std::min(rows / toks + seqs, seqs * ((most + toks - 1) / toks));                // blocks of all sequences, at most
      shares = tile_shares(hk * gy, max_len, h.sms);
      gx = hk;
      shared = tile_shared(d, e4m3);
      name = "kern_attn_tile" + form;
    } else {
      const int64_t nt = g * most <= 8 ? 1 : 2;              // query rows of a CTA, in eights
      toks = 8 * nt / g;
      const int64_t blocks = (most + toks - 1) / toks;
      const RowsForm f = rows_form(d, e4m3, nt);
      std::tie(shares, cluster) = rows_shares(hk * blocks * seqs, max_len, (int64_t)h.sms * f.per_sm);
      // among sequences of more rows, whose CTAs leave at once: two shares at least, and no second launch for what may be none
      if (hi < all && max_len > 128) shares = cluster = std::min<int64_t>(std::max<int64_t>(shares, 2), 8);
      gx = hk * blocks;
      gy = seqs;
      shared = f.shared;
      name = "kern_attn_rows" + form + "_n" + n(nt);
    }
    if (gy > 65535) refuse("more blocks of rows than a launch has: split the call");
    Tensor ws;
    uint64_t ws_o = 0, ws_ml = 0;
    const int64_t groups = shares / cluster;
    const int64_t ws_step = seqs * most < rows ? most : 0, places = std::min(rows, seqs * most);
    if (groups > 1) {
      ws = at::empty({places * hq * groups * (d + 2)}, typed(q, at::kFloat));
      ws_o = reinterpret_cast<uint64_t>(ws.data_ptr());
      ws_ml = ws_o + 4 * (uint64_t)(places * hq * groups * d);
    }
    Block b;
    b.bytes(map.data(), map.size()).at(q).at(out).put(ws_o).put(ws_ml).at(pool).at(table).at(lens).at(cu_q).at(masks);
    b.ints(masks ? masks->size(1) : 0, rows_per_seq, hq, hk, q_step, out_step, width, page, tiled ? seqs : cluster, pages, lo, hi, rows, max_rows, ws_step);
    b.put(scale_log2).put(h.err);
    launch(h, tiled ? tile_module(d) : "attn_rows", name, gx, gy, shares, tiled ? (unsigned)tile_threads(d) : 160, b, shared, !tiled && hi < all, (unsigned)cluster);
    if (groups > 1) {
      Block m;
      m.put(ws_o).put(ws_ml).at(out).at(lens).at(cu_q).ints(rows_per_seq, hq, toks, shares, cluster, out_step, lo, hi, rows, max_rows, ws_step, width * page);
      launch(h, "attn_rows", std::string("kern_attn_rows_merge_") + (masks ? "tree_d" : "causal_d") + n(d), most * hq, seqs, 1, 128, m, 0, true);
    }
  };
  if (g * max_rows <= kFewRows) {
    run(false, 1, all);
  } else if (masks || !cu_q || seqs == 1 || rows + few >= seqs * max_rows) {
    run(true, 1, all);                                       // (rows alike; trees of a node or two among the others end before those)
  } else {
    // sequences of single tokens among prompt chunks keep the few-row kernel, which cuts their contexts into shares
    run(true, few + 1, all);
    run(false, 1, few);
  }
  return out;
}

// ---- trees ------------------------------------------------------------------------------------------------------------------------------
int64_t glue(const Tensor& parents, const Tensor& cu, const Tensor& base, const Tensor& table, int64_t page, std::optional<int64_t> max_rows) {
  if (parents.scalar_type() != at::kInt || parents.dim() != 1 || !whole(parents)) refuse("parents: i32 [nodes]");
  table_of(table, "block_table");
  numbers(cu, at::kInt, table.size(0) + 1, "cu");
  numbers(base, at::kLong, table.size(0), "base");
  if (page < 1 || page > (1 << 20)) refuse("page_size " + n(page));
  const int64_t most = max_rows ? *max_rows : std::min<int64_t>(kMaxNodes, parents.size(0));
  if (most < 0 || most > kMaxNodes) refuse(n(most) + " nodes: at most " + n(kMaxNodes) + " in a tree");
  return most;
}

py::tuple tree_rows(const Tensor& parents, const Tensor& cu, const Tensor& base, const Tensor& table, int64_t page, std::optional<int64_t> max_rows) {
  const int64_t most = glue(parents, cu, base, table, page, max_rows), words = std::max<int64_t>(1, (most + 63) / 64);
  const int gpu = Same(parents)(cu)(base)(table).gpu;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)gpu);
  const int64_t nodes = parents.size(0), seqs = table.size(0);
  const auto i64 = typed(parents, at::kLong);
  if (!seqs || !nodes)                                       // no launch that would fill them
    return py::make_tuple(at::zeros({nodes}, i64), at::full({nodes}, -1, i64), base.narrow(0, 0, seqs).clamp_min(0).to(at::kInt), at::zeros({nodes, words}, i64));
  const Tensor positions = at::empty({nodes}, i64), slots = at::empty({nodes}, i64), masks = at::empty({nodes, words}, i64),
               lens = at::empty({seqs}, typed(parents, at::kInt));
  Host& h = host_of(gpu);
  Block b;
  b.at(parents).at(cu).at(base).at(table).at(positions).at(slots).at(lens).at(masks).ints(nodes, most, words, table.size(1), page).put(h.err);
  launch(h, "tree", "kern_tree_rows", seqs, 1, 1, 256, b);
  return py::make_tuple(positions, slots, lens, masks);
}

py::tuple tree_keep(const Tensor& ids, const Tensor& parents, const Tensor& verify, const Tensor& cu, const Tensor& base, const Tensor& table,
                    const std::vector<Tensor>& pools, int64_t hk, int64_t d, int64_t page, std::optional<int64_t> max_rows) {
  heads(hk, hk, d, page, false);
  const int64_t most = glue(parents, cu, base, table, page, max_rows);
  const int64_t nodes = parents.size(0), seqs = table.size(0);
  numbers(ids, at::kLong, nodes, "ids");
  numbers(verify, at::kLong, nodes, "verify");
  if ((int64_t)pools.size() > kMaxPools) refuse(n(pools.size()) + " pools: at most " + n(kMaxPools));
  int64_t pages = 0;
  uint64_t where[kMaxPools] = {};
  std::unordered_set<uint64_t> seen;
  for (size_t i = 0; i < pools.size(); ++i) {
    pages = pages_any(pools[i], hk, page, d);
    if (pools[i].scalar_type() != pools[0].scalar_type() || pages != pools[0].size(0)) refuse("the pools of a call are alike");
    where[i] = reinterpret_cast<uint64_t>(pools[i].data_ptr());
    if (!seen.insert(where[i]).second) refuse("a pool is named once");
  }
  Same same(parents);
  same(ids)(verify)(cu)(base)(table);
  for (auto& p : pools) same(p);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)same.gpu);
  const auto i32 = typed(parents, at::kInt), i64 = typed(parents, at::kLong);
  if (!seqs || !nodes)                                       // no launch that would fill them
    return py::make_tuple(at::zeros({seqs}, i32), at::full({nodes}, -1, i32), at::zeros({nodes}, i64));
  const Tensor count = at::empty({seqs}, i32), path = at::empty({nodes}, i32), emitted = at::empty({nodes}, i64);
  Host& h = host_of(same.gpu);
  const bool e4m3 = !pools.empty() && pools[0].scalar_type() == at::kByte;
  Block b;
  b.bytes(where, sizeof(where)).at(ids).at(parents).at(verify).at(cu).at(base).at(table).at(count).at(path).at(emitted);
  b.ints(nodes, most, pools.size(), table.size(1), page, hk, d, e4m3, pages).put(h.err);
  launch(h, "tree", "kern_tree_keep", seqs, std::max<int64_t>(1, pools.size()), 1, 128, b);
  return py::make_tuple(count, path, emitted);
}

}  // namespace

PYBIND11_MODULE(_ops_host, m) {
  m.doc() = "Host side of the operators over 8-bit caches and drafted trees";
  m.attr("torch_version") = KERN_TORCH_VERSION;              // that it was built for
  m.def("on_missing", [](py::object f) { missing() = std::move(f); });
  m.def("provide", [](int gpu, int sms, uint64_t err, py::object resolve) {
    auto h = std::make_unique<Host>();
    h->dev = std::make_shared<kern::Device>(gpu);
    h->sms = sms;
    h->err = err;
    h->resolve = std::move(resolve);
    hosts().at(gpu) = std::move(h);
  });
  m.def("launches", [](int gpu) { return hosts().at(gpu) ? hosts()[gpu]->launches : 0; });
  m.def("rows_form", [](int64_t d, bool e4m3, int64_t nt) { const RowsForm f = rows_form(d, e4m3, nt); return py::make_tuple(f.shared, f.per_sm); });
  m.def("tile_form", [](int64_t d, bool e4m3) { return py::make_tuple(tile_module(d), tile_rows(d), tile_threads(d), tile_shared(d, e4m3)); });
  m.def("append", &append);
  m.def("read_rows", &read_rows);
  m.def("attend", &attend);
  m.def("tree_rows", &tree_rows);
  m.def("tree_keep", &tree_keep);
  // (the interpreter's end: what holds Python objects goes before it)
  auto atexit = py::module_::import("atexit");
  atexit.attr("register")(py::cpp_function([] {
    for (auto& h : hosts()) h.reset();
    missing() = py::object();
  }));
}
