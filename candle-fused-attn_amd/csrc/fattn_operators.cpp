// The C ABI of the operators around self-attention (include/fattn.h): argument validation and the
// launches. Validation runs before any HIP call, as in fattn_api.cpp.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "fattn.h"
#include "fattn_internal.h"

namespace {

using fattn::set_error;

// Workgroups of 256 threads in a grid of fewer than 2^32 threads.
constexpr int64_t kMaxGrid = (int64_t{1} << 24) - 1;
constexpr int64_t kMaxHeads = 65535;

bool known(int dtype) { return dtype == FATTN_F32 || dtype == FATTN_F16 || dtype == FATTN_BF16; }
int64_t size_of(int dtype) { return dtype == FATTN_F32 ? 4 : dtype == FATTN_FP4 ? 1 : 2; }
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
void copy3(int64_t to[3], const int64_t from[3]) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}
// Strides {.., .., ..} of dimensions of n0, n1, n2: those of one entry (or none) are never used.
void used3(int64_t to[3], const int64_t from[3], int64_t n0, int64_t n1, int64_t n2) {
  to[0] = n0 > 1 ? from[0] : 0, to[1] = n1 > 1 ? from[1] : 0, to[2] = n2 > 1 ? from[2] : 0;
}
bool multiples(const int64_t st[3], int64_t of) {
  return st[0] % of == 0 && st[1] % of == 0 && st[2] % of == 0;
}
bool negative(const int64_t* x, int n) {
  for (int i = 0; i < n; ++i) {
    if (x[i] < 0) return true;
  }
  return false;
}

int check_dim(const char* who, int64_t d) {
  if (fattn::head_dim_supported(d)) return 0;
  return set_error(FATTN_EHEADDIM, "%s: the HIP kernels take head_dim 32, 64 or 128, got %lld", who,
                   static_cast<long long>(d));
}
int check_types(const char* who, int dtype, int cache_dtype) {
  if (!known(dtype) || !(known(cache_dtype) || cache_dtype == FATTN_FP4)) {
    return set_error(FATTN_EINVAL, "%s: f32, f16 or bf16 only", who);
  }
  if (dtype != FATTN_F32 && cache_dtype != dtype && cache_dtype != FATTN_FP4) {
    return set_error(FATTN_EINVAL, "%s: a cache of another type than 16-bit activations", who);
  }
  return 0;
}
// (No query heads at all: an append without queries, or an empty call.)
int check_heads(const char* who, int64_t heads, int64_t kv_heads, bool none) {
  if (heads < 0 || kv_heads < 0 || heads > kMaxHeads || kv_heads > kMaxHeads) {
    return set_error(FATTN_ERANGE, "%s: at most %lld heads", who, static_cast<long long>(kMaxHeads));
  }
  if (heads == 0 && none) return 0;
  if (kv_heads == 0 || heads == 0 || heads % kv_heads != 0) {
    return set_error(FATTN_EINVAL, "%s: %lld query heads are no multiple of %lld key heads", who,
                     static_cast<long long>(heads), static_cast<long long>(kv_heads));
  }
  return 0;
}

constexpr float kLog2e = 1.44269504088896340736f;
// The cap of scores: 0 (none), or such that it and its inverse are floats in units of log2 e too.
int check_cap(const char* who, float cap) {
  if (cap == 0.0f || (cap >= 1e-30f && cap <= 1e30f)) return 0;
  return set_error(FATTN_EINVAL, "%s: a cap from 1e-30 to 1e30 expected, got %g", who, static_cast<double>(cap));
}

// The pages, their table and the lengths of a cache; ks, vs: the strides that its indices use.
int check_cache(const char* who, int cache_dtype, const void* k, const int64_t k_strides[3],
                const void* v, const int64_t v_strides[3], int64_t pages, int64_t kv_heads,
                int64_t page_size, const int32_t* table, int64_t table_stride, int64_t table_width,
                const int32_t* lengths, int64_t ks[3], int64_t vs[3]) {
  if (!k || !v || !k_strides || !v_strides || !table || !lengths) {
    return set_error(FATTN_EINVAL, "%s: null operand", who);
  }
  if (pages <= 0 || page_size <= 0 || page_size % 16 != 0 || table_width <= 0 || table_stride < 0) {
    return set_error(FATTN_EINVAL, "%s: pages of a multiple of 16 slots and a table of them expected, "
                     "got %lld pages of %lld slots, a table %lld wide", who,
                     static_cast<long long>(pages), static_cast<long long>(page_size),
                     static_cast<long long>(table_width));
  }
  if (pages > INT32_MAX || page_size > INT32_MAX / 2 || table_width > INT32_MAX) {
    return set_error(FATTN_ERANGE, "%s: the cache exceeds 32-bit indexing", who);
  }
  // (4-bit rows are words of 4 bytes, 68 of d 128.)
  const int64_t size = size_of(cache_dtype), unit = cache_dtype == FATTN_FP4 ? 4 : 16, per = unit / size;
  used3(ks, k_strides, pages, kv_heads, page_size);
  used3(vs, v_strides, pages, kv_heads, page_size);
  if (negative(ks, 3) || negative(vs, 3)) return set_error(FATTN_EINVAL, "%s: negative strides", who);
  if (!aligned(k, unit) || !aligned(v, unit) || !multiples(ks, per) || !multiples(vs, per)) {
    return set_error(FATTN_EALIGN, "%s: the cache's rows must be %d-byte aligned", who, static_cast<int>(unit));
  }
  if (16 * ks[2] * size > INT32_MAX || 16 * vs[2] * size > INT32_MAX) {
    return set_error(FATTN_ERANGE, "%s: 16 slots of the cache span more than 2 GiB", who);
  }
  return 0;
}

// Whether an operand's rows can be moved `vec` values at a time.
bool fits(int64_t vec, const void* p, int64_t size, const int64_t st[3], int64_t b, int64_t h, int64_t s) {
  return aligned(p, vec * size) && (b <= 1 || st[0] % vec == 0) && (h <= 1 || st[1] % vec == 0) &&
         (s <= 1 || st[2] % vec == 0);
}

int run_rotary(const char* who, fattn::RotaryArgs& a, int dtype, int cache_dtype, int64_t b, int64_t s,
               int64_t d, int64_t dim, void* stream) {
  const int64_t size = size_of(dtype);
  // (The most pairs: what the kernel's LDS holds for one token.)
  if (d <= 0 || d > 1024 || d % 2 != 0 || dim < 0 || dim % 2 != 0 || dim > d) {
    return set_error(FATTN_EINVAL, "%s: an even head_dim of at most 1024 and an even part of it to turn "
                     "expected, got %lld of %lld", who, static_cast<long long>(dim),
                     static_cast<long long>(d));
  }
  if (b > kMaxGrid || s > kMaxGrid || b * s > kMaxGrid) {
    return set_error(FATTN_ERANGE, "%s: more than %lld tokens", who, static_cast<long long>(kMaxGrid));
  }
  if (dim > 0 && !a.frequencies) return set_error(FATTN_EINVAL, "%s: null frequencies", who);
  a.B = static_cast<int>(b), a.S = static_cast<int>(s), a.D = static_cast<int>(d);
  a.pairs = static_cast<int>(dim / 2);
  int64_t vec = 16 / size;
  if (cache_dtype == FATTN_FP4) {
    // Sixteen values at a time, in two halves (of whole scales each in the half layout; of neighbours, eight values are
    // turned or not), or eight.
    bool pairs = d >= 64 && (a.interleaved ? dim % 8 == 0 : dim % 64 == 0 && (d - dim) % 64 == 0);
    for (int i = 0; i < 3; ++i) {
      const fattn::RotaryPart& p = a.part[i];
      if (p.heads == 0) continue;
      pairs = pairs && fits(vec, p.x, size, p.xs, b, p.heads, s);
      if (i == 0) pairs = pairs && fits(vec, p.y, size, p.ys, b, p.heads, s);
    }
    const int err = fattn::launch_rotary(a, dtype, cache_dtype, pairs ? 16 : 8, stream);
    if (err) return fattn::hip_error(err, who, "launch");
    return fattn::done();
  }
  auto allowed = [&](int64_t v) {
    if (d % v != 0 || (a.interleaved ? dim : dim / 2) % v != 0) return false;
    for (int i = 0; i < 3; ++i) {
      const fattn::RotaryPart& p = a.part[i];
      if (p.heads == 0) continue;
      if (!fits(v, p.x, size, p.xs, b, p.heads, s)) return false;
      if (a.table == nullptr || i == 0) {
        if (!fits(v, p.y, size, p.ys, b, p.heads, s)) return false;
      }  // (the pages' rows are 16-byte aligned)
    }
    return true;
  };
  while (vec >= 4 && !allowed(vec)) vec /= 2;
  if (vec < 4) vec = a.interleaved ? 2 : 1;
  const int err = fattn::launch_rotary(a, dtype, cache_dtype, static_cast<int>(vec), stream);
  if (err) return fattn::hip_error(err, who, "launch");
  return fattn::done();
}

int check_workspace(const char* who, const void* workspace, size_t bytes, size_t need) {
  if (need == 0 || (workspace && aligned(workspace, 16) && bytes >= need)) return 0;
  return set_error(FATTN_EWORKSPACE, "%s: a 16-byte aligned workspace of at least %zu bytes expected", who,
                   need);
}

// Shared by the paged and the cross attention: the plan, the workspace, the launch.
int run_split(const char* who, fattn::SplitArgs& a, int dtype, int cache_dtype, int64_t d,
              int64_t capacity, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t rows = static_cast<int64_t>(a.G) * a.SQ;
  const fattn::SplitPlan plan = fattn::split_plan(a.B, a.HK, rows, d, capacity, cache_dtype == fattn::kFP4);
  if (static_cast<int64_t>(a.B) * a.HK * plan.row_blocks > kMaxGrid ||
      static_cast<int64_t>(a.B) * a.H * a.SQ > kMaxGrid) {
    return set_error(FATTN_ERANGE, "%s: the grid exceeds the launch limit", who);
  }
  if (int rc = check_workspace(who, workspace, workspace_bytes, plan.bytes)) return rc;
  a.RB = plan.row_blocks, a.part_rows = plan.part_rows, a.wgs = plan.wgs, a.min_run = plan.min_run;
  a.begin = plan.begin;
  a.part = static_cast<float*>(workspace);
  a.before = reinterpret_cast<int64_t*>(static_cast<char*>(workspace) + plan.before);
  const int err = fattn::launch_split(a, dtype, cache_dtype, static_cast<int>(d), stream);
  if (err) return fattn::hip_error(err, who, "launch");
  return fattn::done();
}

// --- Cross attention's operands --------------------------------------------------------------------
constexpr const char* kCross = "fused_cross_attention";
struct Cross {
  fattn::View q, k, v;
};
// A [b, h, s, d] operand; false: strides that are negative or leave rows unaligned, or a base that is.
bool view(fattn::View& to, const float* p, const int64_t strides[3], int64_t b, int64_t h, int64_t s) {
  int64_t st[3];
  used3(st, strides, b, h, s);
  to = fattn::View{p, st[0], st[1], st[2]};
  return aligned(p, 16) && !negative(st, 3) && multiples(st, 4);
}
int bad_view(const char* who, const int64_t strides[3]) {
  if (negative(strides, 3)) return set_error(FATTN_EINVAL, "%s: negative strides", who);
  return set_error(FATTN_EALIGN, "%s: rows must be 16-byte aligned", who);
}
// The kernels address the rows of one (batch, head) with 32-bit byte offsets.
bool slice_fits(const fattn::View& v, int64_t s, int64_t d) {
  return s <= 1 || (s - 1) * v.ss * 4 + 4 * d <= int64_t{UINT32_MAX};
}
int cross_operands(Cross& c, const float* q, const int64_t q_strides[3], const float* k,
                   const int64_t k_strides[3], const float* v, const int64_t v_strides[3], int64_t b,
                   int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d, bool* none) {
  if (b < 0 || sq < 0 || sk < 0) return set_error(FATTN_EINVAL, "%s: negative size", kCross);
  if (heads == 0 && kv_heads == 0) b = 0;
  if (int rc = check_heads(kCross, heads, kv_heads, b == 0)) return rc;
  if (int rc = check_dim(kCross, d)) return rc;
  *none = b == 0;
  if (*none) return 0;
  const int64_t lim = INT32_MAX - 256;
  if (b > lim || sq > lim || sk > lim || b * heads > lim || b * heads * sq > lim ||
      b * kv_heads * sk > lim ||
      fattn::cross_query_blocks(b * kv_heads, heads / kv_heads, sq) + fattn::cross_blocks(b * kv_heads, sk) > kMaxGrid) {
    return set_error(FATTN_ERANGE, "%s: the sizes exceed 32-bit indexing or the launch limit", kCross);
  }
  if ((sq > 0 && (!q || !q_strides)) || (sk > 0 && (!k || !v || !k_strides || !v_strides))) {
    return set_error(FATTN_EINVAL, "%s: null operand", kCross);
  }
  if (sq > 0 && !view(c.q, q, q_strides, b, heads, sq)) return bad_view(kCross, q_strides);
  if (sk > 0 && !view(c.k, k, k_strides, b, kv_heads, sk)) return bad_view(kCross, k_strides);
  if (sk > 0 && !view(c.v, v, v_strides, b, kv_heads, sk)) return bad_view(kCross, v_strides);
  if (!slice_fits(c.k, sk, d) || !slice_fits(c.v, sk, d)) {
    return set_error(FATTN_ERANGE, "%s: the keys of one (batch, head) span more than 4 GiB", kCross);
  }
  return 0;
}

// --- Scored attention's operands --------------------------------------------------------------------
constexpr const char* kScored = "fused_scored_attention";
int scored_operands(fattn::ScoredArgs& a, const float* q, const int64_t q_strides[3], const float* k,
                    const int64_t k_strides[3], const float* v, const int64_t v_strides[3], int64_t b,
                    int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d, float scale, int causal,
                    float cap, const float* slopes, const int32_t* documents, int64_t document_stride,
                    const int32_t* prefix, bool* none) {
  if (b < 0 || sq < 0 || sk < 0) return set_error(FATTN_EINVAL, "%s: negative size", kScored);
  if (sq > sk) {
    return set_error(FATTN_EINVAL, "%s: %lld queries are more than the %lld positions", kScored,
                     static_cast<long long>(sq), static_cast<long long>(sk));
  }
  if (heads == 0 && kv_heads == 0) b = 0;
  if (int rc = check_heads(kScored, heads, kv_heads, b == 0)) return rc;
  if (int rc = check_dim(kScored, d)) return rc;
  if (int rc = check_cap(kScored, cap)) return rc;
  *none = b == 0 || sk == 0;
  if (*none) return 0;
  const int64_t lim = INT32_MAX - 256;
  if (b > lim || sk > lim || b * heads > lim || b * heads * sk > lim ||
      fattn::scored_blocks(b, heads, sq) + fattn::scored_blocks(b, kv_heads, sk) > kMaxGrid) {
    return set_error(FATTN_ERANGE, "%s: the sizes exceed 32-bit indexing or the launch limit", kScored);
  }
  if ((sq > 0 && (!q || !q_strides)) || !k || !v || !k_strides || !v_strides) {
    return set_error(FATTN_EINVAL, "%s: null operand", kScored);
  }
  if (documents && document_stride < 0) return set_error(FATTN_EINVAL, "%s: negative strides", kScored);
  if (sq > 0 && !view(a.q, q, q_strides, b, heads, sq)) return bad_view(kScored, q_strides);
  if (!view(a.k, k, k_strides, b, kv_heads, sk)) return bad_view(kScored, k_strides);
  if (!view(a.v, v, v_strides, b, kv_heads, sk)) return bad_view(kScored, v_strides);
  if (!slice_fits(a.k, sk, d) || !slice_fits(a.v, sk, d)) {
    return set_error(FATTN_ERANGE, "%s: the keys of one (batch, head) span more than 4 GiB", kScored);
  }
  a.B = static_cast<int>(b), a.H = static_cast<int>(heads), a.G = static_cast<int>(heads / kv_heads);
  a.SQ = static_cast<int>(sq), a.SK = static_cast<int>(sk);
  a.scale = scale, a.causal = causal ? 1 : 0;
  const float inverse = cap == 0.0f ? 1.0f : 1.0f / (cap * kLog2e);
  a.cap2 = cap * kLog2e, a.unit_rest = inverse > 0x1p40f ? 0x1p60f : inverse < 0x1p-40f ? 0x1p-60f : 1.0f;
  a.unit = inverse / a.unit_rest;
  a.slopes = slopes, a.documents = documents, a.document_stride = document_stride, a.prefix = prefix;
  return 0;
}

bool split_shape(int64_t b, int64_t heads, int64_t kv_heads, int64_t d) {
  return b >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && fattn::head_dim_supported(d);
}

}  // namespace

extern "C" {

int fattn_rotary(int dtype, int64_t b, int64_t s, int64_t d, const int64_t heads[3],
                 const void* const x[3], void* const y[3], const int64_t x_strides[9],
                 const int64_t y_strides[9], int rotated, const void* positions, int position_bits,
                 const int64_t position_strides[2], const double* frequencies, int64_t dim,
                 int interleaved, double magnitude, int inverse, void* stream) {
  const char* who = "fused_rotary";
  if (!known(dtype)) return set_error(FATTN_EINVAL, "%s: f32, f16 or bf16 only", who);
  if (b < 0 || s < 0 || !heads || !x || !y || !x_strides || !y_strides || !position_strides ||
      (position_bits != 32 && position_bits != 64)) {
    return set_error(FATTN_EINVAL, "%s: [b, heads, s, d] operands and positions of 32 or 64 bits expected",
                     who);
  }
  fattn::RotaryArgs a{};
  int64_t all = 0;
  for (int i = 0; i < 3; ++i) {
    if (heads[i] < 0 || heads[i] > kMaxHeads) {
      return set_error(FATTN_ERANGE, "%s: at most %lld heads", who, static_cast<long long>(kMaxHeads));
    }
    all += heads[i];
    fattn::RotaryPart& p = a.part[i];
    p.heads = static_cast<int>(heads[i]);
    p.rotate = (rotated >> i) & 1;
    if (heads[i] == 0) continue;
    p.x = x[i], p.y = y[i];
    copy3(p.xs, x_strides + 3 * i);
    copy3(p.ys, y_strides + 3 * i);
    if (negative(p.xs, 3) || negative(p.ys, 3)) return set_error(FATTN_EINVAL, "%s: negative strides", who);
  }
  if (b == 0 || s == 0 || all == 0) return fattn::done();
  for (int i = 0; i < 3; ++i) {
    if (heads[i] > 0 && (!x[i] || !y[i])) return set_error(FATTN_EINVAL, "%s: null operand", who);
  }
  if (!positions) return set_error(FATTN_EINVAL, "%s: null positions", who);
  a.positions = positions, a.pos64 = position_bits == 64;
  a.pos_strides[0] = position_strides[0], a.pos_strides[1] = position_strides[1];
  a.frequencies = frequencies, a.magnitude = magnitude;
  a.interleaved = interleaved ? 1 : 0, a.inverse = inverse ? 1 : 0;
  return run_rotary(who, a, dtype, dtype, b, s, d, dim, stream);
}

int fattn_paged_append(int dtype, int cache_dtype, int64_t b, int64_t heads, int64_t kv_heads,
                       int64_t s, int64_t d, const void* q, const int64_t q_strides[3], void* q_out,
                       const int64_t q_out_strides[3], const void* k, const int64_t k_strides[3],
                       const void* v, const int64_t v_strides[3], void* k_pages,
                       const int64_t k_page_strides[3], void* v_pages,
                       const int64_t v_page_strides[3], int64_t pages, int64_t page_size,
                       const int32_t* table, int64_t table_stride, int64_t table_width,
                       const int32_t* lengths, const int32_t* counts, const double* frequencies,
                       int64_t dim, int interleaved, double magnitude, void* stream) {
  const char* who = "paged_append";
  if (int rc = check_types(who, dtype, cache_dtype)) return rc;
  if (b < 0 || s < 0) return set_error(FATTN_EINVAL, "%s: negative size", who);
  if (int rc = check_heads(who, heads, kv_heads, kv_heads > 0)) return rc;
  if (int rc = check_dim(who, d)) return rc;
  if (b == 0 || s == 0) return fattn::done();
  fattn::RotaryArgs a{};
  if (int rc = check_cache(who, cache_dtype, k_pages, k_page_strides, v_pages, v_page_strides, pages,
                           kv_heads, page_size, table, table_stride, table_width, lengths,
                           a.page_strides, a.page_strides + 3)) {
    return rc;
  }
  if (!k || !v || !k_strides || !v_strides || (heads > 0 && (!q || !q_out || !q_strides || !q_out_strides))) {
    return set_error(FATTN_EINVAL, "%s: null operand", who);
  }
  if (cache_dtype == FATTN_FP4 && heads > 0 && q == q_out) {
    return set_error(FATTN_EINVAL, "%s: q_out must not be q with a 4-bit cache", who);
  }
  const int turned = frequencies != nullptr ? 1 : 0;
  a.part[0].heads = static_cast<int>(heads), a.part[0].rotate = turned;
  if (heads > 0) {
    a.part[0].x = q, a.part[0].y = q_out;
    copy3(a.part[0].xs, q_strides);
    copy3(a.part[0].ys, q_out_strides);
  }
  a.part[1] = fattn::RotaryPart{k, k_pages, {}, {}, static_cast<int>(kv_heads), turned};
  copy3(a.part[1].xs, k_strides);
  a.part[2] = fattn::RotaryPart{v, v_pages, {}, {}, static_cast<int>(kv_heads), 0};
  copy3(a.part[2].xs, v_strides);
  for (const fattn::RotaryPart& p : a.part) {
    if (negative(p.xs, 3) || negative(p.ys, 3)) return set_error(FATTN_EINVAL, "%s: negative strides", who);
  }
  a.frequencies = frequencies, a.magnitude = magnitude, a.interleaved = interleaved ? 1 : 0;
  a.table = table, a.lengths = lengths, a.counts = counts;
  a.table_stride = table_stride, a.table_width = table_width, a.pages = pages, a.page_size = page_size;
  return run_rotary(who, a, dtype, cache_dtype, b, s, d, turned ? dim : 0, stream);
}

size_t fattn_paged_attention_workspace_bytes(int64_t b, int64_t heads, int64_t kv_heads, int64_t d,
                                             int64_t capacity) {
  if (!split_shape(b, heads, kv_heads, d) || capacity < 0) return 0;
  return fattn::split_plan(b, kv_heads, heads / kv_heads, d, capacity).bytes;
}

int fattn_paged_attention(int dtype, int cache_dtype, int64_t b, int64_t heads, int64_t kv_heads,
                          int64_t d, const void* q, const int64_t q_strides[2], void* out,
                          const void* k_pages, const int64_t k_page_strides[3], const void* v_pages,
                          const int64_t v_page_strides[3], int64_t pages, int64_t page_size,
                          const int32_t* table, int64_t table_stride, int64_t table_width,
                          const int32_t* lengths, float scale, void* workspace,
                          size_t workspace_bytes, void* stream) {
  return fattn_paged_scored_attention(dtype, cache_dtype, b, heads, kv_heads, d, q, q_strides, out, k_pages,
                                      k_page_strides, v_pages, v_page_strides, pages, page_size, table,
                                      table_stride, table_width, lengths, scale, 0.0f, nullptr, workspace,
                                      workspace_bytes, stream);
}

int fattn_paged_scored_attention(int dtype, int cache_dtype, int64_t b, int64_t heads, int64_t kv_heads,
                                 int64_t d, const void* q, const int64_t q_strides[2], void* out,
                                 const void* k_pages, const int64_t k_page_strides[3],
                                 const void* v_pages, const int64_t v_page_strides[3], int64_t pages,
                                 int64_t page_size, const int32_t* table, int64_t table_stride,
                                 int64_t table_width, const int32_t* lengths, float scale, float cap,
                                 const float* slopes, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  const char* who = "paged_attention";
  if (int rc = check_types(who, dtype, cache_dtype)) return rc;
  if (b < 0) return set_error(FATTN_EINVAL, "%s: negative size", who);
  if (int rc = check_heads(who, heads, kv_heads, b == 0)) return rc;
  if (int rc = check_dim(who, d)) return rc;
  if (int rc = check_cap(who, cap)) return rc;
  if (b == 0) return fattn::done();
  fattn::SplitArgs a{};
  if (int rc = check_cache(who, cache_dtype, k_pages, k_page_strides, v_pages, v_page_strides, pages,
                           kv_heads, page_size, table, table_stride, table_width, lengths, a.ks, a.vs)) {
    return rc;
  }
  if (!q || !out || !q_strides) return set_error(FATTN_EINVAL, "%s: null operand", who);
  const int64_t q3[3] = {q_strides[0], q_strides[1], 0};
  used3(a.qs, q3, b, heads, 1);
  if (negative(a.qs, 2)) return set_error(FATTN_EINVAL, "%s: negative strides", who);
  if (!aligned(q, 16) || !aligned(out, 16) || !multiples(a.qs, 16 / size_of(dtype))) {
    return set_error(FATTN_EALIGN, "%s: rows must be 16-byte aligned", who);
  }
  const int64_t capacity = table_width * page_size;
  if (b > INT32_MAX || capacity > INT32_MAX - 64) {
    return set_error(FATTN_ERANGE, "%s: the cache exceeds 32-bit indexing", who);
  }
  a.q = q, a.o = out;
  a.k = k_pages, a.v = v_pages;
  a.table = table, a.table_stride = table_stride, a.lengths = lengths;
  a.page_size = static_cast<int>(page_size), a.pages = static_cast<int>(pages);
  a.by_page = fattn::divider(page_size / 16);
  a.B = static_cast<int>(b), a.H = static_cast<int>(heads), a.HK = static_cast<int>(kv_heads);
  a.G = static_cast<int>(heads / kv_heads), a.SQ = 1, a.SK = static_cast<int>(capacity);
  a.scale = scale;
  a.slopes = slopes, a.cap2 = cap * kLog2e, a.cap_inv = cap == 0.0f ? 0.0f : 1.0f / a.cap2;
  return run_split(who, a, dtype, cache_dtype, d, capacity, workspace, workspace_bytes, stream);
}

int fattn_paged_read(int cache_dtype, int dtype, int64_t b, int64_t kv_heads, int64_t s, int64_t d,
                     const void* k_pages, const int64_t k_page_strides[3], const void* v_pages,
                     const int64_t v_page_strides[3], int64_t pages, int64_t page_size,
                     const int32_t* table, int64_t table_stride, int64_t table_width,
                     const int32_t* lengths, const int32_t* starts, void* k, void* v, void* stream) {
  const char* who = "paged_read";
  if (!known(dtype) || !(known(cache_dtype) || cache_dtype == FATTN_FP4)) {
    return set_error(FATTN_EINVAL, "%s: f32, f16 or bf16 only", who);
  }
  if (b < 0 || s < 0) return set_error(FATTN_EINVAL, "%s: negative size", who);
  if (kv_heads < 0 || kv_heads > kMaxHeads) {
    return set_error(FATTN_ERANGE, "%s: at most %lld heads", who, static_cast<long long>(kMaxHeads));
  }
  if (int rc = check_dim(who, d)) return rc;
  if (b == 0 || s == 0 || kv_heads == 0) return fattn::done();
  fattn::PagedReadArgs a{};
  if (int rc = check_cache(who, cache_dtype, k_pages, k_page_strides, v_pages, v_page_strides, pages,
                           kv_heads, page_size, table, table_stride, table_width, lengths, a.ks, a.vs)) {
    return rc;
  }
  if (!k || !v) return set_error(FATTN_EINVAL, "%s: null operand", who);
  if (!aligned(k, 16) || !aligned(v, 16)) {
    return set_error(FATTN_EALIGN, "%s: rows must be 16-byte aligned", who);
  }
  if (b > kMaxGrid || s > (int64_t{1} << 26) ||
      b * kv_heads > kMaxGrid / fattn::paged_read_blocks(s, d)) {
    return set_error(FATTN_ERANGE, "%s: the sizes exceed 32-bit indexing or the launch limit", who);
  }
  a.k_pages = k_pages, a.v_pages = v_pages, a.k = k, a.v = v;
  a.table = table, a.lengths = lengths, a.starts = starts, a.table_stride = table_stride;
  a.table_width = static_cast<int>(table_width), a.pages = static_cast<int>(pages);
  a.page_size = static_cast<int>(page_size);
  a.B = static_cast<int>(b), a.HK = static_cast<int>(kv_heads), a.S = static_cast<int>(s);
  const int err = fattn::launch_paged_read(a, cache_dtype, dtype, static_cast<int>(d), stream);
  if (err) return fattn::hip_error(err, who, "launch");
  return fattn::done();
}

size_t fattn_cross_workspace_bytes(int64_t b, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk,
                                   int64_t d) {
  if (!split_shape(b, heads, kv_heads, d) || sq < 0 || sk < 0) return 0;
  return fattn::cross_forward_plan(b, heads, kv_heads, sq, sk, d).bytes;
}

size_t fattn_cross_backward_workspace_bytes(int64_t b, int64_t heads, int64_t kv_heads, int64_t sq,
                                            int64_t sk, int64_t d) {
  if (!split_shape(b, heads, kv_heads, d) || sq < 0 || sk < 0) return 0;
  return fattn::cross_backward_plan(b, heads, kv_heads, sq, sk, d).bytes;
}

int fattn_cross_forward(const float* q, const int64_t q_strides[3], const float* k,
                        const int64_t k_strides[3], const float* v, const int64_t v_strides[3],
                        int64_t b, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d,
                        const int32_t* key_lengths, float scale, float* out, float* lse,
                        void* workspace, size_t workspace_bytes, void* stream) {
  Cross c{};
  bool none = false;
  if (int rc = cross_operands(c, q, q_strides, k, k_strides, v, v_strides, b, heads, kv_heads, sq, sk, d,
                              &none)) {
    return rc;
  }
  if (none || sq == 0) return fattn::done();
  if (!out || !lse) return set_error(FATTN_EINVAL, "%s: null operand", kCross);
  if (!aligned(out, 16)) return set_error(FATTN_EALIGN, "%s: rows must be 16-byte aligned", kCross);
  const int B = static_cast<int>(b), H = static_cast<int>(heads), HK = static_cast<int>(kv_heads);
  const int SQ = static_cast<int>(sq), SK = static_cast<int>(sk);
  const fattn::CrossForwardPlan plan = fattn::cross_forward_plan(b, heads, kv_heads, sq, sk, d);
  if (int rc = check_workspace(kCross, workspace, workspace_bytes, plan.bytes)) return rc;
  if (plan.split) {
    fattn::SplitArgs a{};
    a.q = q, a.k = k, a.v = v, a.o = out, a.lse = lse;
    a.qs[0] = c.q.sb, a.qs[1] = c.q.sh, a.qs[2] = c.q.ss;
    a.ks[0] = c.k.sb, a.ks[1] = c.k.sh, a.ks[2] = c.k.ss;
    a.vs[0] = c.v.sb, a.vs[1] = c.v.sh, a.vs[2] = c.v.ss;
    a.lengths = key_lengths;
    a.B = B, a.H = H, a.HK = HK, a.G = H / HK, a.SQ = SQ, a.SK = SK, a.scale = scale;
    return run_split(kCross, a, FATTN_F32, FATTN_F32, d, sk, workspace, workspace_bytes, stream);
  }
  const int err = fattn::launch_cross_forward(c.q, c.k, c.v, out, lse, B, H, HK, SQ, SK,
                                              static_cast<int>(d), key_lengths, scale, plan, workspace,
                                              stream);
  if (err) return fattn::hip_error(err, kCross, "forward launch");
  return fattn::done();
}

int fattn_cross_backward(const float* q, const int64_t q_strides[3], const float* k,
                         const int64_t k_strides[3], const float* v, const int64_t v_strides[3],
                         int64_t b, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d,
                         const int32_t* key_lengths, float scale, const float* out, const float* lse,
                         const float* d_o, const int64_t do_strides[3], float* dq, float* dkv,
                         void* workspace, size_t workspace_bytes, void* stream) {
  Cross c{};
  bool none = false;
  if (int rc = cross_operands(c, q, q_strides, k, k_strides, v, v_strides, b, heads, kv_heads, sq, sk, d,
                              &none)) {
    return rc;
  }
  if (none || (sq == 0 && sk == 0)) return fattn::done();
  if ((sq > 0 && (!out || !lse || !d_o || !do_strides || !dq)) || (sk > 0 && !dkv)) {
    return set_error(FATTN_EINVAL, "%s: null operand", kCross);
  }
  fattn::View g{d_o, 0, 0, 0};
  if (sq > 0 && !view(g, d_o, do_strides, b, heads, sq)) return bad_view(kCross, do_strides);
  if (!aligned(out, 16) || !aligned(dq, 16) || !aligned(dkv, 16)) {
    return set_error(FATTN_EALIGN, "%s: rows must be 16-byte aligned", kCross);
  }
  if (!slice_fits(c.q, sq, d) || !slice_fits(g, sq, d) || sq * heads * d > int64_t{UINT32_MAX}) {
    return set_error(FATTN_ERANGE, "%s: the queries of one sample span more than 4 GiB", kCross);
  }
  const fattn::CrossBackwardPlan plan = fattn::cross_backward_plan(b, heads, kv_heads, sq, sk, d);
  if (int rc = check_workspace(kCross, workspace, workspace_bytes, plan.bytes)) return rc;
  const int err = fattn::launch_cross_backward(
      c.q, c.k, c.v, g, out, lse, dq, dkv, static_cast<int>(b), static_cast<int>(heads),
      static_cast<int>(kv_heads), static_cast<int>(sq), static_cast<int>(sk), static_cast<int>(d),
      key_lengths, scale, plan, workspace, stream);
  if (err) return fattn::hip_error(err, kCross, "backward launch");
  return fattn::done();
}

size_t fattn_scored_workspace_bytes(int64_t b, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk,
                                    int64_t d) {
  if (!split_shape(b, heads, kv_heads, d) || sq < 0 || sk < sq) return 0;
  return fattn::scored_plan(b, heads, sq, sk, d).bytes;
}

size_t fattn_scored_backward_workspace_bytes(int64_t b, int64_t heads, int64_t kv_heads, int64_t sq,
                                             int64_t sk, int64_t d, int causal) {
  if (!split_shape(b, heads, kv_heads, d) || sq < 0 || sk < sq) return 0;
  return fattn::scored_backward_plan(b, heads, kv_heads, sq, sk, d, causal).bytes;
}

int fattn_scored_forward(const float* q, const int64_t q_strides[3], const float* k,
                         const int64_t k_strides[3], const float* v, const int64_t v_strides[3],
                         int64_t b, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d,
                         float scale, int causal, float cap, const float* slopes,
                         const int32_t* documents, int64_t document_stride, const int32_t* prefix,
                         float* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  fattn::ScoredArgs a{};
  bool none = false;
  if (int rc = scored_operands(a, q, q_strides, k, k_strides, v, v_strides, b, heads, kv_heads, sq, sk, d, scale,
                               causal, cap, slopes, documents, document_stride, prefix, &none)) {
    return rc;
  }
  if (none || sq == 0) return fattn::done();
  if (!out || !lse) return set_error(FATTN_EINVAL, "%s: null operand", kScored);
  if (!aligned(out, 16)) return set_error(FATTN_EALIGN, "%s: rows must be 16-byte aligned", kScored);
  const fattn::ScoredPlan plan = fattn::scored_plan(b, heads, sq, sk, d);
  if (fattn::scored_blocks(b, heads, sq) * plan.nc > kMaxGrid) {
    return set_error(FATTN_ERANGE, "%s: the grid exceeds the launch limit", kScored);
  }
  if (int rc = check_workspace(kScored, workspace, workspace_bytes, plan.bytes)) return rc;
  a.out = out, a.lse = lse;
  const int err = fattn::launch_scored_forward(a, static_cast<int>(d), plan, workspace, stream);
  if (err) return fattn::hip_error(err, kScored, "forward launch");
  return fattn::done();
}

int fattn_scored_backward(const float* q, const int64_t q_strides[3], const float* k,
                          const int64_t k_strides[3], const float* v, const int64_t v_strides[3],
                          int64_t b, int64_t heads, int64_t kv_heads, int64_t sq, int64_t sk, int64_t d,
                          float scale, int causal, float cap, const float* slopes,
                          const int32_t* documents, int64_t document_stride, const int32_t* prefix,
                          const float* out, const float* lse, const float* d_o,
                          const int64_t do_strides[3], float* dq, float* dkv, void* workspace,
                          size_t workspace_bytes, void* stream) {
  fattn::ScoredArgs a{};
  bool none = false;
  if (int rc = scored_operands(a, q, q_strides, k, k_strides, v, v_strides, b, heads, kv_heads, sq, sk, d, scale,
                               causal, cap, slopes, documents, document_stride, prefix, &none)) {
    return rc;
  }
  if (none) return fattn::done();
  if ((sq > 0 && (!out || !lse || !d_o || !do_strides || !dq)) || !dkv) {
    return set_error(FATTN_EINVAL, "%s: null operand", kScored);
  }
  if (sq > 0 && !view(a.d_o, d_o, do_strides, b, heads, sq)) return bad_view(kScored, do_strides);
  if (!aligned(out, 16) || !aligned(dq, 16) || !aligned(dkv, 16)) {
    return set_error(FATTN_EALIGN, "%s: rows must be 16-byte aligned", kScored);
  }
  if (!slice_fits(a.q, sq, d) || !slice_fits(a.d_o, sq, d) || sq * heads * d > int64_t{UINT32_MAX}) {
    return set_error(FATTN_ERANGE, "%s: the queries of one sample span more than 4 GiB", kScored);
  }
  const fattn::ScoredBackwardPlan plan = fattn::scored_backward_plan(b, heads, kv_heads, sq, sk, d, causal);
  if (fattn::scored_blocks(b, heads, sq) * plan.ncq + fattn::scored_blocks(b, kv_heads, sk) * plan.nck > kMaxGrid) {
    return set_error(FATTN_ERANGE, "%s: the grid exceeds the launch limit", kScored);
  }
  if (int rc = check_workspace(kScored, workspace, workspace_bytes, plan.bytes)) return rc;
  a.o = out, a.lse = const_cast<float*>(lse), a.dq = dq, a.dkv = dkv;
  const int err = fattn::launch_scored_backward(a, static_cast<int>(d), plan, workspace, stream);
  if (err) return fattn::hip_error(err, kScored, "backward launch");
  return fattn::done();
}

}  // extern "C"
