// Appending a batch's keys and values to the paged cache for gfx950, the keys
// rotated to their positions on the way, in the cache's own type or in 4 bits
// (int4_rows.hpp), and the queries rotated beside them; and reading rows of
// 4-bit pages back as values. The counterpart of paged_copy.hip's scatter and
// gather (cacheblend_vllm/kv_layout.py:90-161) for rows that are not copied
// as they are.
//
// A pair of dims (x, y), dim + rotary_dim / 2 apart (neox) or next to each
// other, at position p becomes (x c - y s, y c + x s), c and s from row p of
// the table; products and differences in float32, each rounded, then once to
// the type (4-bit keys: in 64 bits).
//
// Bound by HBM: every row is read once and written once (8192 tokens of 32 + 2 x
// 8 heads x 128 bf16: 37 us, 5.6 TB/s). A thread takes 16 dims of one head as
// two 16-byte pieces, the two halves of 8 pairs, so that no pair is read twice
// and in-place outputs are safe; the threads of a wave cover whole heads of one
// token after another.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "int4_rows.hpp"

namespace cbk {
namespace {

constexpr int kThreads = 256;
constexpr int kPairs = 8;  // per thread of the pieces' kernel

struct Rows {  // [tokens, heads, head_dim], strides in elements
  const void* base;
  int64_t token_stride, head_stride;
};

// field by field: a choice of addresses would put the kernel's arguments into scratch memory
__device__ __forceinline__ Rows choose(bool first, const Rows& a, const Rows& b) {
  return Rows{first ? a.base : b.base, first ? a.token_stride : b.token_stride, first ? a.head_stride : b.head_stride};
}

struct AppendArgs {
  Rows query, key, value;
  Rows query_out, key_out;  // base NULL: none
  char* k_base;
  char* v_base;
  const int64_t* slots;
  const int64_t* positions;  // NULL: no rotation
  const void* table;         // [table_rows, rotary_dim]: cosines, then sines
  int64_t table_stride;      // elements
  int64_t table_rows;
  int64_t block_stride, token_stride;  // pages, bytes
  uint32_t num_tokens, num_slots;
  uint32_t q_heads, heads, head_dim, rotary_dim;
  int32_t table_dtype;
  bool neox;
  FastDiv block_div;   // by the page's tokens
  FastDiv heads_div;   // by q_heads + 2 heads
  FastDiv unit_div;    // by the threads of a head
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// element conversions of the three types, one at a time (the general kernel)
// and eight at a time
template <int DT> struct Elem;
template <> struct Elem<CBK_DTYPE_F32> {
  typedef float T;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Elem<CBK_DTYPE_BF16> {
  typedef __bf16 T;
  static __device__ __forceinline__ float get(__bf16 x) { return float(x); }
  static __device__ __forceinline__ __bf16 put(float x) { return __bf16(x); }
};
template <> struct Elem<CBK_DTYPE_F16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(_Float16 x) { return float(x); }
  static __device__ __forceinline__ _Float16 put(float x) { return _Float16(x); }
};

template <int DT>
__device__ __forceinline__ f32x8 load8(const void* base, int64_t at) {
  typedef typename Elem<DT>::T T8 __attribute__((ext_vector_type(8)));
  const typename Elem<DT>::T* p = static_cast<const typename Elem<DT>::T*>(base) + at;
  T8 v;
  if constexpr (DT == CBK_DTYPE_F32) {
    const f32x4* w = reinterpret_cast<const f32x4*>(p);
    v = __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return v;
  } else {
    v = __builtin_bit_cast(T8, *reinterpret_cast<const u32x4*>(p));
    return __builtin_convertvector(v, f32x8);
  }
}

template <int DT, bool STREAM = false>
__device__ __forceinline__ void store8(void* base, int64_t at, const f32x8& x) {
  typedef typename Elem<DT>::T T8 __attribute__((ext_vector_type(8)));
  typename Elem<DT>::T* p = static_cast<typename Elem<DT>::T*>(base) + at;
  if constexpr (DT == CBK_DTYPE_F32) {
    f32x4* w = reinterpret_cast<f32x4*>(p);
    const f32x4 lo = __builtin_shufflevector(x, x, 0, 1, 2, 3), hi = __builtin_shufflevector(x, x, 4, 5, 6, 7);
    if constexpr (STREAM) {
      __builtin_nontemporal_store(lo, w);
      __builtin_nontemporal_store(hi, w + 1);
    } else {
      w[0] = lo;
      w[1] = hi;
    }
  } else {
    const u32x4 bits = __builtin_bit_cast(u32x4, __builtin_convertvector(x, T8));
    if constexpr (STREAM) __builtin_nontemporal_store(bits, reinterpret_cast<u32x4*>(p));
    else *reinterpret_cast<u32x4*>(p) = bits;
  }
}

__device__ __forceinline__ f32x8 table8(const void* table, int32_t dtype, int64_t at) {
  if (dtype == CBK_DTYPE_F32) return load8<CBK_DTYPE_F32>(table, at);
  if (dtype == CBK_DTYPE_BF16) return load8<CBK_DTYPE_BF16>(table, at);
  return load8<CBK_DTYPE_F16>(table, at);
}

__device__ __forceinline__ float table1(const void* table, int32_t dtype, int64_t at) {
  if (dtype == CBK_DTYPE_F32) return static_cast<const float*>(table)[at];
  if (dtype == CBK_DTYPE_BF16) return float(static_cast<const __bf16*>(table)[at]);
  return float(static_cast<const _Float16*>(table)[at]);
}

// (x, y) turned: each product and difference rounded (no fused multiply-add),
// so that the result is that of the separate operations
template <typename V>
__device__ __forceinline__ void turn(V& x, V& y, const V& c, const V& s) {
#pragma clang fp contract(off)
  const V a = x * c - y * s;
  y = y * c + x * s;
  x = a;
}

// What a token's rows do: the page row's offset from the planes' bases (-1:
// none, a slot or position out of range) and whether its position is in the
// table.
struct Token {
  int64_t page;
  int64_t position;
  bool placed;
};

__device__ __forceinline__ Token token_of(const AppendArgs& a, uint32_t t) {
  Token r;
  const int64_t slot = a.slots[t];
  r.position = a.positions ? a.positions[t] : 0;
  r.placed = r.position >= 0 && r.position < a.table_rows;
  r.page = -1;
  if (slot >= 0 && slot < int64_t(a.num_slots) && (r.placed || !a.positions)) {
    const uint32_t blk = a.block_div.div(uint32_t(slot));
    r.page = int64_t(blk) * a.block_stride + int64_t(uint32_t(slot) - blk * a.block_div.d) * a.token_stride;
  }
  return r;
}

// Over the lanes whose index differs in the bits of LANES - 1.
template <int LANES>
__device__ __forceinline__ void group_extremes(double& low, double& high, bool& finite) {
#pragma unroll
  for (int off = 1; off < LANES; off <<= 1) {
    low = fmin(low, __shfl_xor(low, off));
    high = fmax(high, __shfl_xor(high, off));
    finite = __shfl_xor(int(finite), off) && finite;
  }
}

struct Extremes {
  double low, high;
  bool finite;
  __device__ __forceinline__ void add(double v) {
    low = fmin(low, v);
    high = fmax(high, v);
    finite = finite && fabs(v) < __builtin_inf();
  }
  __device__ __forceinline__ void join(const Extremes& o) {
    low = fmin(low, o.low);
    high = fmax(high, o.high);
    finite = finite && o.finite;
  }
  // of a group in 4 lanes (quarters) or in 2
  __device__ __forceinline__ Int4Scale scale(bool quarters) {
    group_extremes<2>(low, high, finite);
    const Extremes other{__shfl_xor(low, 2), __shfl_xor(high, 2), __shfl_xor(int(finite), 2) != 0};
    if (quarters) join(other);
    return int4_scale(low, high, finite);
  }
};

// A thread's 8 pairs (x, y), turned by (c, s) if TURN, to 4 bits. With `halves`
// the x are [d0, d0 + 8), a quarter of a group of their own (the rest in the
// neighbouring lanes), the y [d1, d1 + 8); otherwise x and y alternate over the
// 16 dims from d0, half a group. The 64-bit values are computed twice, for the
// extremes and for the codes, and never held: 96 registers instead of 148, so
// that the queries' rows of the launch, bound by HBM, have five waves per SIMD
// instead of three (8192 tokens of 32 + 2 x 8 heads x 128 bf16: 64.9 -> 51.7 us;
// at six waves registers spill). `row` NULL: nothing is written.
template <bool TURN>
__device__ __forceinline__ void store_codes(char* row, uint32_t head_dim, bool halves, uint32_t d0, uint32_t d1, f32x8 xv,
                                            f32x8 yv, f32x8 cv, f32x8 sv) {
#pragma clang fp contract(off)
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = xv[i];
    y[i] = yv[i];
  }
#define CBK_FIRST(i) (TURN ? double(x[i]) * double(cv[i]) - double(y[i]) * double(sv[i]) : double(x[i]))
#define CBK_SECOND(i) (TURN ? double(y[i]) * double(cv[i]) + double(x[i]) * double(sv[i]) : double(y[i]))
  Extremes ex{__builtin_inf(), -__builtin_inf(), true}, ey = ex;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ex.add(CBK_FIRST(i));
    ey.add(CBK_SECOND(i));
  }
  if (!halves) {
    ex.join(ey);
    ey = ex;
  }
  const Int4Scale sx = ex.scale(halves), sy = ey.scale(halves);
  // (the values are not to be kept until here)
#pragma unroll
  for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(x[i]), "+v"(y[i]));
  uint32_t even = 0, odd = 0;  // codes of the x, of the y
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    even |= int4_code(CBK_FIRST(i), sx) << (4 * i);
    odd |= int4_code(CBK_SECOND(i), sy) << (4 * i);
  }
#undef CBK_FIRST
#undef CBK_SECOND
  if (row == nullptr) return;
  if (!halves) {  // x and y in turn: each half's four pairs of codes are a word
    auto spread = [](uint32_t w) {  // 4 codes to the low halves of 4 bytes
      w = (w | (w << 8)) & 0x00ff00ffu;
      return (w | (w << 4)) & 0x0f0f0f0fu;
    };
    const uint32_t lo = spread(even & 0xffffu) | spread(odd & 0xffffu) << 4;
    const uint32_t hi = spread(even >> 16) | spread(odd >> 16) << 4;
    even = lo;
    odd = hi;
  }
  *reinterpret_cast<uint32_t*>(row + d0 / 2) = even;
  *reinterpret_cast<uint32_t*>(row + d1 / 2) = odd;
  uint32_t* const words = reinterpret_cast<uint32_t*>(row + head_dim / 2);
  if (d0 % kInt4Group == 0) words[d0 / kInt4Group] = int4_scale_word(sx);
  if (halves && d1 % kInt4Group == 0) words[d1 / kInt4Group] = int4_scale_word(sy);
}

// One thread per 16 dims of a (token, head): rotary_dim is head_dim or 0,
// everything 16-byte aligned, head_dim a multiple of 16 (4-bit pages: 64).
template <int DT, bool INT4>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(INT4 ? 5 : 8))) void append_pieces_kernel(const AppendArgs a) {
  const uint32_t units = a.unit_div.d, per = kThreads / units;  // threads of a head, heads of a block
  const uint32_t local = a.unit_div.div(threadIdx.x), u = threadIdx.x - local * units;
  if (local >= per) return;
  const uint32_t row = blockIdx.x * per + local;
  const uint32_t t = a.heads_div.div(row);
  if (t >= a.num_tokens) return;
  uint32_t h = row - t * a.heads_div.d;
  const Token tok = token_of(a, t);
  // queries, then keys, then values
  const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.heads;
  if (!is_q) h -= a.q_heads;
  if (is_v) h -= a.heads;
  const Rows in = choose(is_q, a.query, choose(is_v, a.value, a.key));
  const bool rotate = a.positions != nullptr && !is_v;
  // neox pairs lie half a head apart; the others, and rows not rotated, side by side
  const bool halves = a.neox && a.positions != nullptr;
  const uint32_t d0 = halves ? kPairs * u : 2 * kPairs * u, d1 = halves ? d0 + a.head_dim / 2 : d0 + kPairs;
  const int64_t at = int64_t(t) * in.token_stride + int64_t(h) * in.head_stride;
  f32x8 x[2] = {load8<DT>(in.base, at + d0), load8<DT>(in.base, at + d1)};
  f32x8 c = f32x8(1.f), s = f32x8(0.f);
  if (rotate && tok.placed) {
    const int64_t tab = tok.position * a.table_stride + kPairs * u;
    c = table8(a.table, a.table_dtype, tab);
    s = table8(a.table, a.table_dtype, tab + a.head_dim / 2);
  }
  // as pairs: the pieces themselves, or their even and odd dims
  if (!halves) {
    const f32x8 even = __builtin_shufflevector(x[0], x[1], 0, 2, 4, 6, 8, 10, 12, 14);
    x[1] = __builtin_shufflevector(x[0], x[1], 1, 3, 5, 7, 9, 11, 13, 15);
    x[0] = even;
  }
  char* const page = tok.page < 0 ? nullptr : (is_v ? a.v_base : a.k_base) + tok.page;
  if constexpr (INT4) {
    if (!is_q) {  // whole heads: the lanes of a group are here together
      char* const row = page ? page + int64_t(h) * int4_row_bytes(a.head_dim) : nullptr;
      if (rotate) store_codes<true>(row, a.head_dim, halves, d0, d1, x[0], x[1], c, s);
      else store_codes<false>(row, a.head_dim, halves, d0, d1, x[0], x[1], c, s);
    }
  }
  const Rows out = choose(is_q, a.query_out, a.key_out);
  const bool copy = !is_v && out.base != nullptr;
  if (INT4 && !copy) return;
  if (rotate) turn(x[0], x[1], c, s);
  if (!halves) {
    const f32x8 front = __builtin_shufflevector(x[0], x[1], 0, 8, 1, 9, 2, 10, 3, 11);
    x[1] = __builtin_shufflevector(x[0], x[1], 4, 12, 5, 13, 6, 14, 7, 15);
    x[0] = front;
  }
  if constexpr (!INT4) {
    if (!is_q && page) {
      store8<DT>(page, int64_t(h) * a.head_dim + d0, x[0]);
      store8<DT>(page, int64_t(h) * a.head_dim + d1, x[1]);
    }
  }
  if (copy) {
    if (rotate && !tok.placed) x[0] = x[1] = f32x8(0.f);
    const int64_t to = int64_t(t) * out.token_stride + int64_t(h) * out.head_stride;
    store8<DT>(const_cast<void*>(out.base), to + d0, x[0]);
    store8<DT>(const_cast<void*>(out.base), to + d1, x[1]);
  }
}

// One wave per (token, head), lane l its dims l + 64 i: any head_dim up to
// 512, rotary_dim, stride and alignment. All dims are read before one is
// written (in-place outputs).
constexpr int kLaneDims = 8;

template <int DT, bool INT4>
__global__ __launch_bounds__(kThreads) void append_rows_kernel(const AppendArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t row = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const uint32_t t = a.heads_div.div(row);
  if (t >= a.num_tokens) return;
  uint32_t h = row - t * a.heads_div.d;
  const Token tok = token_of(a, t);
  const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.heads;
  if (!is_q) h -= a.q_heads;
  if (is_v) h -= a.heads;
  const Rows in = choose(is_q, a.query, choose(is_v, a.value, a.key));
  const bool rotate = a.positions != nullptr && !is_v;
  const T* src = static_cast<const T*>(in.base) + int64_t(t) * in.token_stride + int64_t(h) * in.head_stride;
  const uint32_t half = a.rotary_dim / 2;
  float x[kLaneDims];
  double y[kLaneDims];
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i) {
#pragma clang fp contract(off)
    const uint32_t d = lane + 64 * i;
    x[i] = 0.f;
    y[i] = 0.0;
    if (d >= a.head_dim) continue;
    x[i] = E::get(src[d]);
    y[i] = double(x[i]);
    if (rotate && tok.placed && d < a.rotary_dim) {
      const uint32_t j = a.neox ? (d < half ? d : d - half) : d / 2;  // the pair
      const bool second = a.neox ? d >= half : (d & 1);
      const uint32_t other = a.neox ? (second ? d - half : d + half) : (d ^ 1u);
      const float o = E::get(src[other]);
      const int64_t tab = tok.position * a.table_stride + j;
      const float c = table1(a.table, a.table_dtype, tab), s = table1(a.table, a.table_dtype, tab + half);
      const float xc = x[i] * c, os = o * s;
      x[i] = second ? xc + os : xc - os;
      const double yc = y[i] * double(c), ys = double(o) * double(s);
      y[i] = second ? yc + ys : yc - ys;
    }
  }
  char* const page = tok.page < 0 ? nullptr : (is_v ? a.v_base : a.k_base) + tok.page;
  if (!is_q && page) {
    if constexpr (INT4) {
      char* dst = page + int64_t(h) * int4_row_bytes(a.head_dim);
#pragma unroll
      for (int i = 0; i < kLaneDims; ++i) {
        if (uint32_t(64 * i) >= a.head_dim) break;  // uniform
        const uint32_t d = lane + 64 * i;
        double low = y[i], high = y[i];
        bool finite = fabs(y[i]) < __builtin_inf();
        group_extremes<32>(low, high, finite);
        const Int4Scale s = int4_scale(low, high, finite);
        // 8 codes of neighbouring lanes to a word
        uint32_t word = int4_code(y[i], s) << (4 * (lane & 7));
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) word |= uint32_t(__shfl_xor(int(word), off));
        if (d < a.head_dim && (lane & 7) == 0) *reinterpret_cast<uint32_t*>(dst + d / 2) = word;
        if (d < a.head_dim && (lane & 31) == 0)
          *reinterpret_cast<uint32_t*>(dst + a.head_dim / 2 + d / kInt4Group * 4) = int4_scale_word(s);
      }
    } else {
      T* dst = reinterpret_cast<T*>(page) + int64_t(h) * a.head_dim;
#pragma unroll
      for (int i = 0; i < kLaneDims; ++i)
        if (lane + 64 * i < a.head_dim) dst[lane + 64 * i] = E::put(x[i]);
    }
  }
  const Rows out = choose(is_q, a.query_out, a.key_out);
  if (is_v || out.base == nullptr) return;
  T* dst = static_cast<T*>(const_cast<void*>(out.base)) + int64_t(t) * out.token_stride + int64_t(h) * out.head_stride;
  const bool zero = rotate && !tok.placed;
#pragma unroll
  for (int i = 0; i < kLaneDims; ++i)
    if (lane + 64 * i < a.head_dim) dst[lane + 64 * i] = E::put(zero ? 0.f : x[i]);
}

// Rows of 4-bit pages as values: a thread reads one word of codes and its
// group's scale word and writes 8 values, past the caches (65,531 tokens of 4 x
// 128 bf16: 28.7 us, 6.1 TB/s; 40.3 through them). Bound by HBM, mostly the
// values written; a slot out of range gives a zero row.
struct GatherArgs {
  const char* k_base;
  const char* v_base;
  const int64_t* slots;
  char* out_k;
  int64_t out_plane, out_token;        // bytes: V minus K, token to token
  int64_t block_stride, token_stride;  // pages, bytes
  uint32_t num_tokens, num_slots, head_dim;
  FastDiv block_div;
  FastDiv row_div;   // by the words of a row
  FastDiv head_div;  // by the words of a head
};

template <int DT>
__global__ __launch_bounds__(kThreads) void gather_int4_kernel(const GatherArgs a) {
  const uint32_t f = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t row = a.row_div.div(f);
  if (row >= 2 * a.num_tokens) return;
  const uint32_t w = f - row * a.row_div.d;  // the word of the row
  const bool is_v = row >= a.num_tokens;
  const uint32_t t = is_v ? row - a.num_tokens : row;
  const int64_t slot = a.slots[t];
  f32x8 x = f32x8(0.f);
  if (slot >= 0 && slot < int64_t(a.num_slots)) {
    const uint32_t blk = a.block_div.div(uint32_t(slot));
    const uint32_t h = a.head_div.div(w), j = w - h * a.head_div.d;
    const char* src = (is_v ? a.v_base : a.k_base) + int64_t(blk) * a.block_stride +
                      int64_t(uint32_t(slot) - blk * a.block_div.d) * a.token_stride +
                      int64_t(h) * int4_row_bytes(a.head_dim);
    const uint32_t word = reinterpret_cast<const uint32_t*>(src)[j];
    const uint32_t sw = reinterpret_cast<const uint32_t*>(src + a.head_dim / 2)[j / 4];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = int4_value((word >> (4 * e)) & 15u, sw);
  }
  store8<DT, true>(a.out_k + (is_v ? a.out_plane : 0) + int64_t(t) * a.out_token, int64_t(w) * 8, x);
}

template <bool INT4>
int launch_append(const AppendArgs& a, int32_t dtype, bool pieces, hipStream_t stream) {
  const uint64_t rows = uint64_t(a.num_tokens) * a.heads_div.d;
  const uint64_t per = pieces ? kThreads / a.unit_div.d : kThreads / 64;
  const uint64_t grid = (rows + per - 1) / per;
  CBK_REQUIRE(grid * kThreads < (uint64_t(1) << 32) && rows + per < (uint64_t(1) << 32),
              "append: %llu workgroups exceed one launch", (unsigned long long)grid);
#define CBK_APPEND(DT)                                                                                           \
  case DT:                                                                                                       \
    if (pieces) hipLaunchKernelGGL((append_pieces_kernel<DT, INT4>), dim3(uint32_t(grid)), dim3(kThreads), 0, stream, a); \
    else hipLaunchKernelGGL((append_rows_kernel<DT, INT4>), dim3(uint32_t(grid)), dim3(kThreads), 0, stream, a); \
    break;
  switch (dtype) {
    CBK_APPEND(CBK_DTYPE_F32)
    CBK_APPEND(CBK_DTYPE_BF16)
    CBK_APPEND(CBK_DTYPE_F16)
  }
#undef CBK_APPEND
  return launch_status("paged append");
}

int64_t address(const void* p) { return int64_t(reinterpret_cast<uintptr_t>(p)); }

}  // namespace
}  // namespace cbk

extern "C" {

int cbk_paged_append(const cbk_kv_desc* kv, const int64_t* slots_dev, int64_t num_tokens, const void* key_dev,
                     int64_t key_token_stride, int64_t key_head_stride, const void* value_dev,
                     int64_t value_token_stride, int64_t value_head_stride, const void* query_dev,
                     int64_t query_token_stride, int64_t query_head_stride, int64_t q_heads, int64_t heads,
                     int64_t head_dim, int32_t dtype, int32_t int4, const int64_t* positions_dev,
                     const void* cos_sin_dev, int64_t cos_sin_row_stride_elems, int64_t cos_sin_rows,
                     int32_t cos_sin_dtype, int64_t rotary_dim, int32_t neox, void* query_out_dev,
                     int64_t query_out_token_stride, int64_t query_out_head_stride, void* key_out_dev,
                     int64_t key_out_token_stride, int64_t key_out_head_stride, cbk_stream_t stream) {
  using namespace cbk;
  clear_error();
  if (int rc = validate_desc(kv)) return rc;
  CBK_REQUIRE(num_tokens >= 0, "num_tokens must be >= 0");
  CBK_REQUIRE(dtype == CBK_DTYPE_F32 || dtype == CBK_DTYPE_BF16 || dtype == CBK_DTYPE_F16, "dtype %d", int(dtype));
  CBK_REQUIRE(heads > 0 && q_heads >= 0 && heads < (1 << 20) && q_heads < (1 << 20), "heads out of range");
  CBK_REQUIRE(head_dim > 0 && head_dim <= 64 * kLaneDims, "head_dim %lld: 1 to %d supported", (long long)head_dim,
              64 * kLaneDims);
  const int64_t es = dtype == CBK_DTYPE_F32 ? 4 : 2;
  if (int4) {
    CBK_REQUIRE(head_dim % kInt4Group == 0, "4-bit rows need a head_dim that is a multiple of %d", kInt4Group);
    CBK_REQUIRE(kv->row_bytes == heads * int4_row_bytes(head_dim), "a 4-bit row of %lld x %lld is %lld bytes, not %lld",
                (long long)heads, (long long)head_dim, (long long)(heads * int4_row_bytes(head_dim)),
                (long long)kv->row_bytes);
    const int64_t words[4] = {address(kv->k_base), address(kv->v_base), kv->block_stride, kv->token_stride};
    CBK_REQUIRE(common_vec_bytes(words, 4) >= 4, "4-bit pages must be 4-byte aligned");
  } else {
    CBK_REQUIRE(kv->row_bytes == heads * head_dim * es, "the pages' rows are %lld bytes, the keys' %lld",
                (long long)kv->row_bytes, (long long)(heads * head_dim * es));
    const int64_t elems[4] = {address(kv->k_base), address(kv->v_base), kv->block_stride, kv->token_stride};
    CBK_REQUIRE(common_vec_bytes(elems, 4) >= es, "the pages must be aligned to their elements");
  }
  if (num_tokens == 0) return CBK_OK;
  CBK_REQUIRE(num_tokens < (int64_t(1) << 31), "num_tokens out of range");
  CBK_REQUIRE(slots_dev && key_dev && value_dev, "NULL pointer");
  CBK_REQUIRE((query_dev != nullptr) == (q_heads > 0) && (query_out_dev != nullptr) == (q_heads > 0),
              "query heads need a query and its output");
  if (positions_dev != nullptr) {
    CBK_REQUIRE(cos_sin_dev != nullptr && cos_sin_rows > 0, "rotation needs a table");
    CBK_REQUIRE(rotary_dim > 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0, "rotary_dim %lld of head_dim %lld",
                (long long)rotary_dim, (long long)head_dim);
    CBK_REQUIRE(cos_sin_row_stride_elems >= rotary_dim, "table row stride smaller than a row");
    CBK_REQUIRE(cos_sin_dtype == CBK_DTYPE_F32 || cos_sin_dtype == CBK_DTYPE_BF16 || cos_sin_dtype == CBK_DTYPE_F16,
                "table dtype %d", int(cos_sin_dtype));
  }
  AppendArgs a;
  a.query = Rows{query_dev, query_token_stride, query_head_stride};
  a.key = Rows{key_dev, key_token_stride, key_head_stride};
  a.value = Rows{value_dev, value_token_stride, value_head_stride};
  a.query_out = Rows{query_out_dev, query_out_token_stride, query_out_head_stride};
  a.key_out = Rows{key_out_dev, key_out_token_stride, key_out_head_stride};
  a.k_base = static_cast<char*>(kv->k_base);
  a.v_base = static_cast<char*>(kv->v_base);
  a.slots = slots_dev;
  a.positions = positions_dev;
  a.table = cos_sin_dev;
  a.table_stride = cos_sin_row_stride_elems;
  a.table_rows = positions_dev ? cos_sin_rows : 0;
  a.block_stride = kv->block_stride;
  a.token_stride = kv->token_stride;
  a.num_tokens = uint32_t(num_tokens);
  a.num_slots = uint32_t(kv->num_blocks * kv->block_size);
  a.q_heads = uint32_t(q_heads);
  a.heads = uint32_t(heads);
  a.head_dim = uint32_t(head_dim);
  a.rotary_dim = positions_dev ? uint32_t(rotary_dim) : 0;
  a.table_dtype = cos_sin_dtype;
  a.neox = neox != 0;
  a.block_div = FastDiv::make(uint32_t(kv->block_size));
  a.heads_div = FastDiv::make(uint32_t(q_heads + 2 * heads));
  a.unit_div = FastDiv::make(uint32_t(head_dim >= 16 ? head_dim / 16 : 1));
  // the pieces' kernel: whole 16-byte pieces of pairs, and of a table row; for
  // 4 bits a group's lanes side by side within aligned lanes
  int64_t bytes[20] = {address(key_dev), key_token_stride * es, key_head_stride * es, address(value_dev),
                       value_token_stride * es, value_head_stride * es, address(query_dev), query_token_stride * es,
                       query_head_stride * es, address(query_out_dev), query_out_token_stride * es,
                       query_out_head_stride * es, address(key_out_dev), key_out_token_stride * es,
                       key_out_head_stride * es, 0, 0, 0, 0, 0};
  if (!int4) {
    bytes[15] = address(kv->k_base);
    bytes[16] = address(kv->v_base);
    bytes[17] = kv->block_stride;
    bytes[18] = kv->token_stride;
  }
  bool pieces = common_vec_bytes(bytes, 20) == 16 && head_dim % (int4 ? 64 : 16) == 0;
  if (positions_dev != nullptr) {
    const int64_t te = cos_sin_dtype == CBK_DTYPE_F32 ? 4 : 2;
    const int64_t table[3] = {address(cos_sin_dev), cos_sin_row_stride_elems * te, head_dim / 2 * te};
    pieces = pieces && rotary_dim == head_dim && common_vec_bytes(table, 3) == 16;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return int4 ? launch_append<true>(a, dtype, pieces, s) : launch_append<false>(a, dtype, pieces, s);
}

int cbk_paged_gather_int4(const cbk_kv_desc* kv, const int64_t* slots_dev, int64_t num_tokens, int64_t heads,
                          int64_t head_dim, int32_t dtype, void* out_k_dev, void* out_v_dev, int64_t out_token_stride,
                          cbk_stream_t stream) {
  using namespace cbk;
  clear_error();
  if (int rc = validate_desc(kv)) return rc;
  CBK_REQUIRE(num_tokens >= 0, "num_tokens must be >= 0");
  CBK_REQUIRE(dtype == CBK_DTYPE_F32 || dtype == CBK_DTYPE_BF16 || dtype == CBK_DTYPE_F16, "dtype %d", int(dtype));
  CBK_REQUIRE(heads > 0 && heads < (1 << 20) && head_dim > 0 && head_dim % kInt4Group == 0 && head_dim < (1 << 20),
              "4-bit rows need a head_dim that is a multiple of %d", kInt4Group);
  CBK_REQUIRE(kv->row_bytes == heads * int4_row_bytes(head_dim), "a 4-bit row of %lld x %lld is %lld bytes, not %lld",
              (long long)heads, (long long)head_dim, (long long)(heads * int4_row_bytes(head_dim)),
              (long long)kv->row_bytes);
  if (num_tokens == 0) return CBK_OK;
  CBK_REQUIRE(slots_dev && out_k_dev && out_v_dev, "NULL pointer");
  const int64_t es = dtype == CBK_DTYPE_F32 ? 4 : 2;
  CBK_REQUIRE(out_token_stride >= heads * head_dim * es, "output token stride smaller than a row");
  const int64_t words[4] = {address(kv->k_base), address(kv->v_base), kv->block_stride, kv->token_stride};
  CBK_REQUIRE(common_vec_bytes(words, 4) >= 4, "4-bit pages must be 4-byte aligned");
  const int64_t outs[3] = {address(out_k_dev), address(out_v_dev), out_token_stride};
  CBK_REQUIRE(common_vec_bytes(outs, 3) == 16, "the output must be 16-byte aligned");
  GatherArgs a;
  a.k_base = static_cast<const char*>(kv->k_base);
  a.v_base = static_cast<const char*>(kv->v_base);
  a.slots = slots_dev;
  a.out_k = static_cast<char*>(out_k_dev);
  a.out_plane = address(out_v_dev) - address(out_k_dev);
  a.out_token = out_token_stride;
  a.block_stride = kv->block_stride;
  a.token_stride = kv->token_stride;
  const uint64_t row_words = uint64_t(heads) * uint64_t(head_dim) / 8;
  const uint64_t total = 2 * uint64_t(num_tokens) * row_words;
  CBK_REQUIRE(total + kThreads < (uint64_t(1) << 32), "too many rows in one launch (%lld tokens)",
              (long long)num_tokens);
  a.num_tokens = uint32_t(num_tokens);
  a.num_slots = uint32_t(kv->num_blocks * kv->block_size);
  a.head_dim = uint32_t(head_dim);
  a.block_div = FastDiv::make(uint32_t(kv->block_size));
  a.row_div = FastDiv::make(uint32_t(row_words));
  a.head_div = FastDiv::make(uint32_t(head_dim / 8));
  const dim3 grid(uint32_t((total + kThreads - 1) / kThreads)), block(kThreads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case CBK_DTYPE_F32: hipLaunchKernelGGL((gather_int4_kernel<CBK_DTYPE_F32>), grid, block, 0, s, a); break;
    case CBK_DTYPE_BF16: hipLaunchKernelGGL((gather_int4_kernel<CBK_DTYPE_BF16>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((gather_int4_kernel<CBK_DTYPE_F16>), grid, block, 0, s, a); break;
  }
  return launch_status("paged int4 gather");
}

}  // extern "C"
