// Attention of a sequence's latest tokens over its context in 4-bit pages
// (int4_rows.hpp) for gfx950:
//
//   out[b, r, h] = sum_k softmax_k( scale q[b, r, h] . key[k, h / G] ) value[k, h / G]
//
// over keys k <= len_b - R + r of sequence b (row r of its R rows is the
// token at that place), G = Hq / Hkv.
//
// Bound by HBM: 0.625 bytes a key or value element, each read once for all
// heads of a group. The codes go to the matrix cores as they are. With key
// element offset + step * n, n the 4-bit code, and 32 dims g sharing both,
//
//   q . key   = sum_g step_g (sum_{d in g} q_d n_d) + offset_g (sum_{d in g} q_d)
//   out_d     = sum_k (p_k step_g) n_d + sum_k p_k offset_g
//
// so the inner sums are products of small whole numbers on the matrix cores, the
// codes in a form that takes little work:
//  - beside q (16 bits) a halfword 000n or 00n0 (hex) is the float16 subnormal
//    number n 2^-24 or n 2^-20: four masks and a shift make 8 codes an operand. q,
//    times a power of two of its row that brings its largest element to 2^15 ..
//    2^16 (its exponent is put back last, the range of q and of keys is float32's),
//    and every second element times 2^-4 more, is a float16 operand: float16
//    and bf16 elements as they are, down to where float16 ends, 2^-36 of the row's
//    largest. (One product a code word. e4m3 parts of q, two or three products, held
//    it to 2^-17 of that element only.)
//  - beside p step a halfword 0x4300 | n is the bf16 value 128 + n, one and-or
//    for two codes; a product with -128 follows, so that the running sums stay
//    small.
//  - float32 converts the codes, to n - 8 for the values: the two sums of out_d
//    then do not cancel; q is three bf16 parts.
// sum_g offset_g (sum q_d) is one more product: a row's steps and offsets, as
// they are stored, with the sums of q in three bf16 parts. p step is cut into
// two bf16 parts (float32: three), the last rounded to nearest (2^-16, 2^-23 of
// it; cut off instead it would be a bias, which a long context's sums of both
// signs do not forgive).
//
// A wave takes 32 keys of one KV head at a time, their rows staged in its own
// LDS by DMA two steps ahead (no barrier in the loop): a step's buffer holds V
// of its tile and K of the next, for it takes S^T of the next tile beside P . V
// of its own, two chains of dependent work in turns. And a wave takes 16 columns of
// S^T = K . Q^T: VT column groups of 16 / VT rows each, for the rows of the
// group are often fewer than 16. The Q operand of a 16-key half is zero outside
// the half's column group, so VT 2 gives both halves one accumulator, and the
// softmax's work on the VALU half the columns. Half t's row m is key 8 (m / 4) +
// 4 t + m % 4 of the 32, so that lane (j = lane / 16, c) holds, over the two
// halves, keys 8 j .. 8 j + 7: those of lane group j in the second product, whose
// codes a ds_read_tr4_b64 hands out, of 16 dims in its first word (from the
// rows that lanes 0 to 7 address) and of the next 16 in its second (lanes 8 to
// 15, the same rows, 8 bytes on).
//
// The sequences' 32-key tiles, one after another, are cut into as many equal
// ranges as fill the GPU, whatever sequences they belong to; a workgroup takes
// one range and up to 8 KV heads (of one row tile), a wave a head: neighbouring
// heads' rows share cache lines, and side by side the waves ask for them at the
// same time. (With a workgroup a head, on one XCD, the heads drifted apart, L2
// fetched 1.6 GB for 0.83 of pages, and 64 sequences of up to 16K keys took 255
// us whatever the work per key; now 209 to 215, 3.9 TB/s. Without the work 187,
// without the transfers 171: what is left is their dependences, at the two waves
// a SIMD that the registers allow.) With fewer heads several waves of a head take
// its tiles in turn. A sequence that one range holds whole is written at once,
// the others' partial results are merged by a second launch.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "int4_rows.hpp"

namespace cbk {
namespace {

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;   // keys of a wave's step
constexpr int kStages = 3;  // tiles in a wave's LDS
// waves of a workgroup, at most (float32 takes the registers of 8 with 4)
constexpr int max_waves(int32_t dtype) { return dtype == CBK_DTYPE_F32 ? 4 : 8; }
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
// Logits are held in units of 4 times log 2: float32's largest logit times log2 e
// is past its range, a quarter of that is not.
constexpr float kUnit = 4.f;
constexpr float kRescale = 8.f / kUnit;  // headroom before the reference maximum is raised
// The weights before they are divided by their sum are 2^-18 at the reference maximum, so
// 2^-10 at most: a tile's products with 128 + n (32 keys' 143 steps, of a 15th of
// float32's whole range each: 2e38) stay within the range, and so do, beside them, the
// sums of 256 keys of the largest values, of more keys if the values are smaller in
// proportion. At the other end products are rounded to bf16's smallest number, 2^-133,
// which over 2^-18 and for 15 steps is an absolute 2e-34.
constexpr float kWeights = -18.f;

struct Int4AttnArgs {
  const void* q;
  void* out;
  int64_t q_batch, q_row, q_head;        // elements
  int64_t out_batch, out_row, out_head;
  const char* k_base;
  const char* v_base;
  int64_t block_stride, token_stride;    // bytes
  const int32_t* tables;
  int64_t table_stride;                  // entries
  const int32_t* lens;
  uint32_t batch, rows, hq, hkv, group;  // rows: of a sequence
  uint32_t num_blocks, max_len;
  uint32_t row_tiles;                    // of 16 / VT (row, head of the group) pairs
  uint32_t ranges;
  uint32_t heads, turns;                 // of a workgroup: KV heads, and waves that share one's tiles
  float scale;
  bool q_pieces;                         // 16-byte pieces of q are aligned
  FastDiv block_div;
  // partial results of range r's first (0) and last (1) unfinished sequence:
  // entry ((2 r + which) hkv + kv head) * rows * group + row * group + head
  float2* ml;
  float* o;
};

// The tiles [first, end) of range r of `total` tiles.
struct Ranges {
  uint32_t each, more;  // tiles of a range; ranges that have one more
  __device__ __forceinline__ Ranges(uint32_t total, uint32_t ranges) : each(total / ranges), more(total % ranges) {}
  __device__ __forceinline__ uint32_t first(uint32_t r) const { return r * each + min(r, more); }
  __device__ __forceinline__ uint32_t of(uint32_t tile) const {
    const uint32_t big = more * (each + 1);
    return tile < big ? tile / (each + 1) : more + (tile - big) / each;
  }
};

__device__ __forceinline__ uint32_t context_of(const Int4AttnArgs& a, uint32_t b) {
  return uint32_t(min(max(a.lens[b], 0), int32_t(a.max_len)));
}

__device__ __forceinline__ uint32_t tiles_of(uint32_t len) { return (len + kTile - 1) / kTile; }

__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  return uint32_t(__builtin_amdgcn_readlane(int(wave_inclusive_scan(v)), 63));
}

// LDS DMA from a 64-bit address per lane (the rows of pages anywhere): lane
// l's 16 or 4 bytes land at lds + l * size, N requests' one after another. M0
// and its waits as CBK_LDS_DMA's; lds wave-uniform.
#define CBK_LDS_FIRST(op, addr) "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\t" op " " addr ", off\n\t"
#define CBK_LDS_NEXT(op, step, addr) "s_nop 0\n\ts_add_u32 m0, m0, " step "\n\ts_nop 0\n\t" op " " addr ", off\n\t"
#define CBK_LDS_LAST "s_nop 0\n\ts_mov_b32 m0, %0"
template <int PIECE, int N>
__device__ __forceinline__ void lds_dma(const char* base, const uint64_t (&off)[N], uint32_t lds) {
  static_assert(N % 5 == 0, "requests in fives");
#pragma unroll
  for (int n = 0; n < N; n += 5) {
    uint32_t saved;
    const char* const p[5] = {base + off[n], base + off[n + 1], base + off[n + 2], base + off[n + 3], base + off[n + 4]};
    const uint32_t to = __builtin_amdgcn_readfirstlane(int(lds + n * 64 * PIECE));
    if constexpr (PIECE == 16) {
      asm volatile(CBK_LDS_FIRST("global_load_lds_dwordx4", "%2") CBK_LDS_NEXT("global_load_lds_dwordx4", "0x400", "%3")
                       CBK_LDS_NEXT("global_load_lds_dwordx4", "0x400", "%4") CBK_LDS_NEXT("global_load_lds_dwordx4", "0x400", "%5")
                           CBK_LDS_NEXT("global_load_lds_dwordx4", "0x400", "%6") CBK_LDS_LAST
                   : "=&s"(saved) : "s"(to), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]) : "memory", "scc");
    } else {
      asm volatile(CBK_LDS_FIRST("global_load_lds_dword", "%2") CBK_LDS_NEXT("global_load_lds_dword", "0x100", "%3")
                       CBK_LDS_NEXT("global_load_lds_dword", "0x100", "%4") CBK_LDS_NEXT("global_load_lds_dword", "0x100", "%5")
                           CBK_LDS_NEXT("global_load_lds_dword", "0x100", "%6") CBK_LDS_LAST
                   : "=&s"(saved) : "s"(to), "v"(p[0]), "v"(p[1]), "v"(p[2]), "v"(p[3]), "v"(p[4]) : "memory", "scc");
    }
  }
}
__device__ __forceinline__ void lds_dma_word(const void* addr, uint32_t lds) {
  uint32_t saved;
  asm volatile(CBK_LDS_FIRST("global_load_lds_dword", "%2") CBK_LDS_LAST
               : "=&s"(saved) : "s"(__builtin_amdgcn_readfirstlane(int(lds))), "v"(addr) : "memory");
}

// How codes n become an MFMA operand: as bf16 128 + n, or converted to bf16 n -
// LESS (beside q of 16 bits: as float16 n 2^-24 and n 2^-20 in turns).
enum class Form { kBf16, kExact, kHalf };

// 8 codes of a word as 8 operand elements, in the order 0 4 1 5 2 6 3 7.
template <Form F, int LESS = 0>
__device__ __forceinline__ s16x8 operand(uint32_t w) {
  u32x4 r;
  if constexpr (F == Form::kExact) {
    const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;  // codes 0 2 4 6, 1 3 5 7
    auto f = [](uint32_t x, int byte) { return __float_as_uint(float((x >> (8 * byte)) & 0xffu) - float(LESS)); };
    auto pair = [](uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); };
    r[0] = pair(f(even, 0), f(even, 2));
    r[1] = pair(f(odd, 0), f(odd, 2));
    r[2] = pair(f(even, 1), f(even, 3));
    r[3] = pair(f(odd, 1), f(odd, 3));
  } else {
    const uint32_t mask = 0x000f000fu, one = 0x43004300u;
    // (and, or in one instruction: the compiler takes two for two constants.
    // No inline assembly: the hazards between what it writes and what a matrix
    // instruction still reads would go unseen)
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_bitop3_b32(w >> (4 * i), mask, one, 0xea);
  }
  return __builtin_bit_cast(s16x8, r);
}

__device__ __forceinline__ f32x4 mma(const s16x8& a, const s16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The operands of q . n: parts of q, and the codes' words.
template <Form F> struct QOperand;
template <> struct QOperand<Form::kExact> {
  typedef s16x8 Q;
  static __device__ __forceinline__ s16x8 codes(uint32_t w) { return operand<Form::kExact>(w); }
  static __device__ __forceinline__ f32x4 mul(const s16x8& k, const Q& q, const f32x4& c) { return mma(k, q, c); }
  // 8 elements' upper 8 bits, in the codes' order; x: what is left
  static __device__ __forceinline__ Q cut(float (&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(__float_as_uint(x[i + 4]), __float_as_uint(x[i]), 0x07060302u);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] -= __uint_as_float(__float_as_uint(x[e]) & 0xffff0000u);
    return __builtin_bit_cast(s16x8, w);
  }
};
template <> struct QOperand<Form::kHalf> {
  typedef h16x8 Q;
  static __device__ __forceinline__ h16x8 codes(uint32_t w) {
    const uint32_t low = 0x000f000fu, high = 0x00f000f0u;
    return __builtin_bit_cast(h16x8, u32x4{w & low, w & high, (w >> 8) & low, (w >> 8) & high});
  }
  static __device__ __forceinline__ f32x4 mul(const h16x8& k, const Q& q, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q, c, 0, 0, 0);
  }
  // 8 elements in the codes' order, those beside n 2^-20 times 2^-4
  static __device__ __forceinline__ Q cut(float (&x)[8]) {
    constexpr float less = 1.f / 16.f;
    return Q{_Float16(x[0]), _Float16(x[4]), _Float16(x[1] * less), _Float16(x[5] * less),
             _Float16(x[2]), _Float16(x[6]), _Float16(x[3] * less), _Float16(x[7] * less)};
  }
};

// two floats rounded to bf16, x in the low half
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, b2));
}

template <int DT> __device__ __forceinline__ float load_elem(const void* p, int64_t at);
template <> __device__ __forceinline__ float load_elem<CBK_DTYPE_F32>(const void* p, int64_t at) {
  return static_cast<const float*>(p)[at];
}
template <> __device__ __forceinline__ float load_elem<CBK_DTYPE_BF16>(const void* p, int64_t at) {
  return bf16_bits_to_float(static_cast<const uint16_t*>(p)[at]);
}
template <> __device__ __forceinline__ float load_elem<CBK_DTYPE_F16>(const void* p, int64_t at) {
  return float(static_cast<const _Float16*>(p)[at]);
}
// 8 neighbouring elements, in 16-byte pieces where they are aligned; zeros if not `live`
template <int DT>
__device__ __forceinline__ void load_elems(const void* p, int64_t at, bool pieces, bool live, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  if (!live) return;
  if (!pieces) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = load_elem<DT>(p, at + e);
  } else if constexpr (DT == CBK_DTYPE_F32) {
    const f32x4* w = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const f32x4 lo = w[0], hi = w[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = lo[e];
      x[e + 4] = hi[e];
    }
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t bits = uint16_t(w[e / 2] >> (16 * (e & 1)));
      x[e] = DT == CBK_DTYPE_BF16 ? bf16_bits_to_float(bits) : float(__builtin_bit_cast(_Float16, bits));
    }
  }
}
template <int DT> __device__ __forceinline__ void store_elem(void* p, int64_t at, float x) {
  if constexpr (DT == CBK_DTYPE_F32) static_cast<float*>(p)[at] = x;
  else if constexpr (DT == CBK_DTYPE_BF16) static_cast<__bf16*>(p)[at] = __bf16(x);
  else static_cast<_Float16*>(p)[at] = _Float16(x);
}

// The operands' parts, the form of the codes beside q and beside p step.
template <int DT> struct Parts;
template <> struct Parts<CBK_DTYPE_BF16> { static constexpr int q = 1, p = 2; static constexpr Form k = Form::kHalf, v = Form::kBf16; };
template <> struct Parts<CBK_DTYPE_F16> { static constexpr int q = 1, p = 2; static constexpr Form k = Form::kHalf, v = Form::kBf16; };
template <> struct Parts<CBK_DTYPE_F32> { static constexpr int q = 3, p = 3; static constexpr Form k = Form::kExact, v = Form::kExact; };

template <int DT, int NG, int VT, int PIECE>
__global__ __launch_bounds__(64 * max_waves(DT), 1) void int4_attn_kernel(const Int4AttnArgs a) {
  constexpr int kMax = max_waves(DT);
  constexpr int QP = Parts<DT>::q, PP = Parts<DT>::p;
  constexpr Form KF = Parts<DT>::k, VF = Parts<DT>::v;
  using QO = QOperand<KF>;
  constexpr int D = 32 * NG, RB = kInt4GroupBytes * NG;  // dims and bytes of a head's row
  constexpr int U = 2 / VT, COLS = 16 / VT;
  constexpr uint32_t kBuf = kTile * RB;                      // K or V rows of a tile
  constexpr uint32_t kPieces = RB / PIECE, kInsts = 2 * kTile * kPieces / 64;
  constexpr uint32_t kWaveLds = kStages * 2 * kBuf;
  static_assert(2 * kTile * kPieces % 64 == 0 && 16 * D * 4 + 128 <= int(kWaveLds), "whole requests; the wave's results fit its buffers");
  // per wave: tiles of K rows, then V rows; then the results of a sequence
  __shared__ __attribute__((aligned(16))) char lds[kMax][kWaveLds];
  __shared__ uint32_t s_pages[kMax][2][64];  // block table entries of two tiles' keys

  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t j = lane >> 4, c = lane & 15;
  // workgroups of one range on one XCD, one after another: a token's row is
  // one piece of memory for all heads
  const uint32_t units = a.hkv / a.heads * a.row_tiles;
  const uint32_t place_in = blockIdx.x >> 3;
  const uint32_t range = __builtin_amdgcn_readfirstlane((place_in / units) * 8 + (blockIdx.x & 7));
  if (range >= a.ranges) return;
  const uint32_t unit = __builtin_amdgcn_readfirstlane(place_in % units);
  const uint32_t head0 = unit / a.row_tiles * a.heads, row_tile = unit % a.row_tiles;  // the workgroup's
  const uint32_t turn = __builtin_amdgcn_readfirstlane(wave / a.heads), turns = a.turns;
  const uint32_t kvh = head0 + (wave - turn * a.heads);

  // the tiles of 64 sequences, a lane each (the first 64 are read once), and of all
  const uint32_t tiles0 = lane < a.batch ? tiles_of(context_of(a, lane)) : 0u;
  uint32_t all = tiles0;
  for (uint32_t b = lane + 64; b < a.batch; b += 64) all += tiles_of(context_of(a, b));
  const Ranges cut(wave_total(all), a.ranges);
  uint32_t at = cut.first(range);
  const uint32_t end = cut.first(range + 1);
  if (at == end) return;
  // the sequence that holds tile `at`, and the tiles before it
  uint32_t seq = 0, before = 0;
  for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
    uint32_t n = tiles0;
    if (b0 > 0) n = b0 + lane < a.batch ? tiles_of(context_of(a, b0 + lane)) : 0u;
    const uint32_t upto = before + wave_inclusive_scan(n);
    const uint64_t past = __ballot(upto > at);
    if (past) {
      const int first = __builtin_ctzll(past);
      seq = b0 + uint32_t(first);
      before = uint32_t(__builtin_amdgcn_readlane(int(upto - n), first));
      break;
    }
    before = uint32_t(__builtin_amdgcn_readlane(int(upto), 63));
  }
  seq = __builtin_amdgcn_readfirstlane(seq);

  // this lane's row (row, head of the group) and its column group
  const uint32_t v = c / COLS, n_row = row_tile * COLS + c % COLS;
  const bool live = n_row < a.rows * a.group;
  const uint32_t qr = live ? n_row / a.group : 0, qh = kvh * a.group + (live ? n_row % a.group : 0);
  // a negative scale goes into the queries
  const float sign = a.scale < 0.f ? -1.f : 1.f;
  int c2_exponent;
  const float c2 = frexpf(fabsf(a.scale) * kLog2e, &c2_exponent);  // 0.5 .. 1, its exponent in the rows' units
  const uint32_t lds0 = lds_address(&lds[wave][0]), pages0 = lds_address(&s_pages[wave][0][0]);
  // the selector that puts a float's upper half into the low (first 16 keys) or high half of a word
  const uint32_t place = v ? 0x03020c0cu : 0x0c0c0302u, half = v ? 0xffff0000u : 0x0000ffffu;

  for (bool first_seq = true; at < end; first_seq = false) {
    uint32_t len = context_of(a, seq);
    while (before + tiles_of(len) <= at) {  // empty sequences, and on to the next
      before += tiles_of(len);
      len = context_of(a, ++seq);
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    len = __builtin_amdgcn_readfirstlane(len);
    before = __builtin_amdgcn_readfirstlane(before);
    const uint32_t seq_end = before + tiles_of(len);
    const uint32_t stop = min(end, seq_end);
    const bool whole = at == before && stop == seq_end;
    const int32_t tile0 = int32_t(at - before + turn);           // the wave's first tile of the sequence
    const int32_t count = int32_t((stop - at + turns - 1 - turn) / turns);
    const int32_t* table = a.tables + int64_t(seq) * a.table_stride;
    const int32_t last_key = live ? int32_t(len) - int32_t(a.rows) + int32_t(qr) : -1;  // the row sees keys up to it

    float x_q[NG][8];  // the row's elements 32 g + 8 j ..
#pragma unroll
    for (int g = 0; g < NG; ++g)
      load_elems<DT>(a.q, int64_t(seq) * a.q_batch + int64_t(qr) * a.q_row + int64_t(qh) * a.q_head + 32 * g + 8 * j,
                     a.q_pieces, live, x_q[g]);

    // The block table's entries of step i's rows -- K of tile i + 1, lanes 0 to
    // 31, and V of tile i, the others -- by DMA; and, from them, the rows, by DMA.
    // Keys past the context, or in a page out of range, are read from the first
    // page and masked: their bits of the result, K's, are clear.
    auto key_of = [&](int32_t i) __attribute__((always_inline)) {  // of this lane; < 0 before the first tile
      return int32_t(tile0 + turns * (i + (lane < 32u ? 1 : 0))) * kTile + int32_t(lane & 31u);
    };
    auto entries = [&](int32_t i) __attribute__((always_inline)) {
      const uint32_t key = uint32_t(min(max(key_of(i), 0), int32_t(len) - 1));
      lds_dma_word(table + a.block_div.div(key), pages0 + uint32_t(i & 1) * 256);
    };
    const char* const k_base = a.k_base + int64_t(kvh) * RB;
    const int64_t v_minus_k = a.v_base - a.k_base;
    auto request = [&](int32_t i, uint32_t buf) __attribute__((always_inline)) {
      const int32_t key = key_of(i);
      const uint32_t page = s_pages[wave][i & 1][lane];
      const bool held = key >= 0 && key < int32_t(len) && page < a.num_blocks;
      uint64_t row = 0;
      if (held) {
        const uint32_t blk = a.block_div.div(uint32_t(key));
        row = uint64_t(page) * uint64_t(a.block_stride) +
              uint64_t(uint32_t(key) - blk * a.block_div.d) * uint64_t(a.token_stride);
      }
      if (lane >= 32u) row += uint64_t(v_minus_k);
      uint64_t off[kInsts];
#pragma unroll
      for (uint32_t n = 0; n < kInsts; ++n) {
        // piece 64 n + lane of the buffer: of row R of the K rows, then the V
        // rows; that is key 8 (R % 16 / 4) + 4 (R / 16) + R % 4
        const uint32_t piece = 64 * n + lane, line = piece / kPieces, part = piece - line * kPieces, R = line % kTile;
        const int from = int((line & 32u) + 8 * ((R >> 2) & 3) + 4 * (R >> 4) + (R & 3));
        off[n] = (uint64_t(uint32_t(__shfl(int(uint32_t(row)), from))) |
                  (uint64_t(uint32_t(__shfl(int(uint32_t(row >> 32)), from))) << 32)) + part * PIECE;
      }
      lds_dma<PIECE>(k_base, off, lds0 + buf * 2 * kBuf);
      return uint32_t(__ballot(held));
    };

    uint32_t held = 0, held_next = 0;  // of the K rows of steps i and i + 1
    if (count > 0) {
      entries(-1);
      entries(0);
    }
    CBK_WAIT_VM_LGKM0(0);  // nothing of the compiler's own in flight from here on
    if (count > 0) {
      held = request(-1, 2);
      if (count > 1) entries(1);
      held_next = request(0, 0);
    }

    // Q operands (zero outside a half's column group), and the sums of their
    // groups as the operand beside the steps and offsets: lane group j has part j;
    // made while the first rows are on their way
    typename QO::Q qf[QP][VT][NG];
    s16x8 qsum;
    int unit;  // the exponent of S^T's unit
    {
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x_q[g][e]));
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      // the row's largest element to 2^15 .. 2^16 (float32, whose codes have no 2^-24: 2^-9 .. 2^-8),
      // whatever its exponent: S^T holds for keys up to the end of the range
      const int e = int(__float_as_uint(top) >> 23) - 127, down = (KF == Form::kHalf ? 15 : -9) - e;
      unit = c2_exponent - 2 + 24 - 15 + e;  // of kUnit
      uint32_t part[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x_q[g][e] = __builtin_ldexpf(x_q[g][e] * sign, down);
          sum += x_q[g][e];
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if constexpr (KF == Form::kHalf) sum *= 0x1p-24f;
        const uint32_t hi = __float_as_uint(sum) & 0xffff0000u;
        const float rest = sum - __uint_as_float(hi);
        const uint32_t mid = __float_as_uint(rest) & 0xffff0000u;
        const uint32_t low = __float_as_uint(rest - __uint_as_float(mid)) & 0xffff0000u;
        part[g] = j == 0 ? hi : j == 1 ? mid : j == 2 ? low : 0u;
#pragma unroll
        for (int p = 0; p < QP; ++p) {
          const typename QO::Q w = QO::cut(x_q[g]);
#pragma unroll
          for (int t = 0; t < VT; ++t) qf[p][t][g] = VT == 1 || v == uint32_t(t) ? w : typename QO::Q(0);
        }
      }
      u32x4 w = u32x4(0u);
#pragma unroll
      for (int g = 0; g < NG; ++g) w[g] = part[g];
      qsum = __builtin_bit_cast(s16x8, w);
    }

    float m = kNegInf, l = 0.f, zsum[NG];
    f32x4 o[2 * NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      zsum[g] = 0.f;
      o[2 * g] = o[2 * g + 1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    f32x4 x[U];  // logits, then weights, of key 8 j + 4 (u VT + v) + r and column c's row
    uint32_t seen = 0xffu;  // which of the lane's keys its row sees: bit 4 t + r
    bool masked = false;    // uniform: not all keys of the tile, for all rows

    // S^T of a tile
    auto logits = [&](const char* kb, f32x4 (&s)[U]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // the offsets' part: of each half by itself, for a masked key's offset may
        // be NaN, which the other half's zeros would not keep out
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          const uint32_t* sw = reinterpret_cast<const uint32_t*>(kb + (16 * (u * VT + t) + c) * RB + 16 * NG);
          u32x4 w = u32x4(0u);
#pragma unroll
          for (int g = 0; g < NG; ++g) w[g] = sw[g];
          const f32x4 part = mma(__builtin_bit_cast(s16x8, w), qsum, f32x4{0.f, 0.f, 0.f, 0.f});
          s[u] = t == 0 || v == uint32_t(t) ? part : s[u];
        }
        f32x4 acc[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          acc[g] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < VT; ++t) {
            const auto kf = QO::codes(*reinterpret_cast<const uint32_t*>(kb + (16 * (u * VT + t) + c) * RB + 16 * g + 4 * j));
#pragma unroll
            for (int p = 0; p < QP; ++p) acc[g] = QO::mul(kf, qf[p][t][g], acc[g]);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t* sw = reinterpret_cast<const uint32_t*>(kb + (16 * (u * VT + v) + 4 * j + r) * RB + 16 * NG);
          float sum = s[u][r];
#pragma unroll
          for (int g = 0; g < NG; ++g) sum = fmaf(__uint_as_float(sw[g] << 16), acc[g][r], sum);
          s[u][r] = __builtin_ldexpf(sum * c2, unit);
        }
      }
    };
    // the tile's mask, from its keys' bits, and the reference maximum
    auto settle = [&](int32_t key0, uint32_t here) __attribute__((always_inline)) {
      masked = here != ~0u || key0 + kTile > int32_t(len - a.rows + 1);
      seen = 0xffu;
      if (masked) {
        const int32_t left = last_key - key0 - int32_t(8 * j) + 1;  // of the lane's 8 keys
        seen = (here >> (8 * j)) & 0xffu;
        seen &= left <= 0 ? 0u : left >= 8 ? 0xffu : (1u << left) - 1u;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!((seen >> (4 * (u * VT + v) + r)) & 1u)) x[u][r] = kNegInf;
      }
      float lm = x[0][0];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) lm = fmaxf(lm, x[u][r]);
      if (__any(lm > m + kRescale)) {  // rare: raise the reference of the columns that need it
        float bm = fmaxf(lm, __shfl_xor(lm, 16));
        bm = fmaxf(bm, __shfl_xor(bm, 32));
        const float mn = fmaxf(m, bm);
        const float alpha = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f((m - mn) * kUnit);
        m = mn;
        l *= alpha;
        float ao[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) ao[r] = __shfl(alpha, int(4 * j + r));
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          zsum[g] *= alpha;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            o[2 * g][r] *= ao[r];
            o[2 * g + 1][r] *= ao[r];
          }
        }
      }
    };
    // O += P . V of the settled tile
    auto sums = [&](const char* vb, auto mask) __attribute__((always_inline)) {
      constexpr bool MASK = decltype(mask)::value;
      const float ms = m == kNegInf ? 0.f : m;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[u][r] = __builtin_amdgcn_exp2f(fmaf(x[u][r] - ms, kUnit, kWeights));
          l += x[u][r];
        }
      // p step in bf16 parts, operand word r key r of the first half in its low
      // half, of the second in its high half
      u32x4 pw[NG][PP];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y[NG][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t* sw = reinterpret_cast<const uint32_t*>(vb + (16 * (u * VT + v) + 4 * j + r) * RB + 16 * NG);
          const bool sees = !MASK || ((seen >> (4 * (u * VT + v) + r)) & 1u);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const uint32_t word = sees ? sw[g] : 0u;  // a masked key's step and offset may be anything
            y[g][u] = x[u][r] * __uint_as_float(word << 16);
            float z = __uint_as_float(word & 0xffff0000u);
            if constexpr (VF == Form::kExact) z = fmaf(8.f, __uint_as_float(word << 16), z);
            zsum[g] = fmaf(x[u][r], z, zsum[g]);
          }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int q = 0; q < PP; ++q) {
            if (q + 1 < PP) {  // the upper halves, and what is left
              pw[g][q][r] = VT == 1 ? __builtin_amdgcn_perm(__float_as_uint(y[g][U - 1]), __float_as_uint(y[g][0]), 0x07060302u)
                                    : __builtin_amdgcn_perm(0u, __float_as_uint(y[g][0]), place);
#pragma unroll
              for (int u = 0; u < U; ++u) y[g][u] -= __uint_as_float(__float_as_uint(y[g][u]) & 0xffff0000u);
            } else {
              pw[g][q][r] = pack_bf16(y[g][0], y[g][U - 1]) & (VT == 1 ? 0xffffffffu : half);
            }
          }
      }
      const uint32_t from = (16 * ((c >> 2) & 1) + 4 * j + (c & 3)) * RB + (c >> 3) * 8;  // the row of key 8 j + c % 8
      const s16x8 less = __builtin_bit_cast(s16x8, u32x4(0xc300c300u));  // -128
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const i32x2 w = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)((__attribute__((address_space(3))) const void*)(vb + from + 16 * g)));
        const s16x8 vf[2] = {operand<VF, 8>(uint32_t(w[0])), operand<VF, 8>(uint32_t(w[1]))};
#pragma unroll
        for (int q = 0; q < PP; ++q) {
          const s16x8 pf = __builtin_bit_cast(s16x8, pw[g][q]);
#pragma unroll
          for (int d = 0; d < 2; ++d) o[2 * g + d] = mma(pf, vf[d], o[2 * g + d]);
          if constexpr (VF != Form::kExact)
#pragma unroll
            for (int d = 0; d < 2; ++d) o[2 * g + d] = mma(pf, less, o[2 * g + d]);
        }
      }
    };

    if (count > 0) {  // step -1: S^T of tile 0 alone
      CBK_WAIT_VM_LGKM0(kInsts);
      asm volatile("" ::: "memory");
      const uint32_t here = held;
      held = held_next;
      if (count > 2) entries(2);
      if (count > 1) held_next = request(1, 1);
      logits(&lds[wave][2 * 2 * kBuf], x);
      settle(int32_t(tile0) * kTile, here);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    uint32_t buf = 0;  // of step i: i % kStages
    for (int32_t i = 0; i < count; ++i) {
      // requested in this order: step i, the entries of step i + 2, step i + 1;
      // all but the last have landed
      if (i + 1 < count) CBK_WAIT_VM_LGKM0(kInsts);
      else CBK_WAIT_VM_LGKM0(0);
      asm volatile("" ::: "memory");
      const uint32_t here = held;
      held = held_next;
      if (i + 3 < count) entries(i + 3);
      if (i + 2 < count) held_next = request(i + 2, buf == 0 ? 2 : buf - 1);  // the buffer of step i - 1
      const char* kb = &lds[wave][buf * 2 * kBuf];
      const char* vb = kb + kBuf;
      buf = buf == kStages - 1 ? 0 : buf + 1;
      if (i + 1 < count) {
        f32x4 next[U];
        if (masked) {
          logits(kb, next);
          sums(vb, std::true_type());
        } else {
          logits(kb, next);
          sums(vb, std::false_type());
        }
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = next[u];
        settle(int32_t(tile0 + turns * (i + 1)) * kTile, here);
      } else {
        sums(vb, std::true_type());
      }
      // the reads of this step's buffer are done before the next requests into it
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }

    // the wave's results, then all waves' and column groups' together
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      zsum[g] += __shfl_xor(zsum[g], 16);
      zsum[g] += __shfl_xor(zsum[g], 32);
    }
    float* mine = reinterpret_cast<float*>(&lds[wave][0]);  // [16 columns][D], then m and l of each
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float z = __shfl(zsum[g], int(4 * j + r));
#pragma unroll
        for (int d = 0; d < 2; ++d) mine[(4 * j + r) * D + 32 * g + 16 * d + c] = o[2 * g + d][r] + z;
      }
    if (j == 0) {
      mine[16 * D + 2 * c] = m;
      mine[16 * D + 2 * c + 1] = l;
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.heads * uint32_t(COLS * D); e += blockDim.x) {
      const uint32_t line = e / D, dim = e - line * D, head = line / COLS, row = line - head * COLS;
      const uint32_t n = row_tile * COLS + row;
      if (n >= a.rows * a.group) continue;
      float top = kNegInf, sum = 0.f, acc = 0.f;
      for (uint32_t w = head; w < a.heads * turns; w += a.heads)
#pragma unroll
        for (int t = 0; t < VT; ++t) top = fmaxf(top, reinterpret_cast<const float*>(&lds[w][0])[16 * D + 2 * (t * COLS + row)]);
      const float ts = top == kNegInf ? 0.f : top;
      for (uint32_t w = head; w < a.heads * turns; w += a.heads)
#pragma unroll
        for (int t = 0; t < VT; ++t) {
          const float* res = reinterpret_cast<const float*>(&lds[w][0]);
          const uint32_t col = t * COLS + row;
          const float f = __builtin_amdgcn_exp2f((res[16 * D + 2 * col] - ts) * kUnit);
          sum = fmaf(f, res[16 * D + 2 * col + 1], sum);
          acc = fmaf(f, res[col * D + dim], acc);
        }
      const uint32_t r = n / a.group, h = (head0 + head) * a.group + n % a.group;
      if (whole) {
        store_elem<DT>(a.out, int64_t(seq) * a.out_batch + int64_t(r) * a.out_row + int64_t(h) * a.out_head + dim,
                       sum == 0.f ? 0.f : acc / sum);
      } else {
        const int64_t id = (int64_t(2 * range + (first_seq ? 0 : 1)) * a.hkv + head0 + head) * (a.rows * a.group) + n;
        a.o[id * D + dim] = acc;
        if (dim == 0) a.ml[id] = make_float2(top, sum);
      }
    }
    __syncthreads();  // the buffers are free for the next sequence
    at = stop;
  }
}

// The sequences that more than one range holds, and those without keys: a
// workgroup per row, every 32 lanes each SUBS-th range of it, each lane D / 32
// dims. 256 ranges of 32 rows: 46 us with one 32 lanes a row, 14 with 8, 6.9
// with 32.
template <int DT, int D, int SUBS>
__global__ __launch_bounds__(32 * SUBS) void int4_attn_merge_kernel(const Int4AttnArgs a) {
  constexpr int N = D / 32;
  typedef float VecN __attribute__((ext_vector_type(N)));
  __shared__ float s_o[SUBS][D], s_l[SUBS], s_m[SUBS];
  const uint32_t seq = blockIdx.y;
  const uint32_t lane = threadIdx.x & 63, dim = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const uint32_t tiles = tiles_of(context_of(a, seq));
  const uint32_t per_head = a.rows * a.group;
  const uint32_t kvh = blockIdx.x / per_head, n = blockIdx.x - kvh * per_head;
  float top = kNegInf, sum = 0.f;
  VecN acc = VecN(0.f);
  if (tiles != 0) {
    // tiles before the sequence, and of all
    uint32_t before = 0, total = 0;
    for (uint32_t b = lane; b < a.batch; b += 64) {
      const uint32_t t = tiles_of(context_of(a, b));
      total += t;
      before += b < seq ? t : 0u;
    }
    total = wave_total(total);
    before = wave_total(before);
    const Ranges cut(total, a.ranges);
    const uint32_t r0 = cut.of(before), r1 = cut.of(before + tiles - 1);
    if (r0 == r1) return;  // written by its range
    // range r0 may end with this sequence after others; the rest begin in it
    const uint32_t which0 = cut.first(r0) < before ? 1u : 0u;
#pragma unroll 4
    for (uint32_t r = r0 + sub; r <= r1; r += SUBS) {
      const int64_t id = (int64_t(2 * r + (r == r0 ? which0 : 0u)) * a.hkv + kvh) * per_head + n;
      const float2 ml = a.ml[id];
      const VecN part = *reinterpret_cast<const VecN*>(a.o + id * D + N * dim);
      const float mn = fmaxf(top, ml.x), ms = mn == kNegInf ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f((top - ms) * kUnit), w = __builtin_amdgcn_exp2f((ml.x - ms) * kUnit);
      sum = f * sum + w * ml.y;
      acc = f * acc + w * part;
      top = mn;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) s_o[sub][N * dim + e] = acc[e];
  if (dim == 0) {
    s_m[sub] = top;
    s_l[sub] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= uint32_t(D)) return;
  float all = kNegInf, l = 0.f, o = 0.f;
#pragma unroll
  for (int i = 0; i < SUBS; ++i) all = fmaxf(all, s_m[i]);
  const float ms = all == kNegInf ? 0.f : all;
#pragma unroll
  for (int i = 0; i < SUBS; ++i) {
    const float w = __builtin_amdgcn_exp2f((s_m[i] - ms) * kUnit);
    l = fmaf(w, s_l[i], l);
    o = fmaf(w, s_o[i][threadIdx.x], o);
  }
  const uint32_t r = n / a.group, h = kvh * a.group + n % a.group;
  store_elem<DT>(a.out, int64_t(seq) * a.out_batch + int64_t(r) * a.out_row + int64_t(h) * a.out_head + threadIdx.x,
                 l == 0.f ? 0.f : o / l);
}

// Column groups for the rows of a KV head.
constexpr int column_groups(uint64_t rows) { return rows <= 8 ? 2 : 1; }

struct Plan {
  uint32_t row_tiles, ranges, heads, turns;
};

int plan_of(int64_t batch, int64_t rows, int64_t hq, int64_t hkv, int64_t max_len, int32_t dtype, Plan* p) {
  CBK_REQUIRE(batch >= 0 && batch < (1 << 16), "batch out of range");
  CBK_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "query heads must be divisible by KV heads");
  CBK_REQUIRE(rows > 0 && hq < (1 << 16) && rows < (1 << 16), "rows or heads out of range");
  CBK_REQUIRE(max_len >= 0 && max_len < (int64_t(1) << 31) - kTile, "context out of range");
  const int64_t n = rows * (hq / hkv);
  p->row_tiles = uint32_t((n + 15) / 16);
  const uint32_t waves = uint32_t(max_waves(dtype));
  for (p->heads = waves; hkv % p->heads != 0;) --p->heads;
  p->turns = waves / p->heads;
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  // a workgroup of each CU (LDS, registers); fewer where its waves would have
  // less than a tile or two each
  const int64_t most = batch * ((max_len + kTile - 1) / kTile);
  CBK_REQUIRE(most < (int64_t(1) << 31), "context tiles out of range");
  const int64_t units = hkv / p->heads * int64_t(p->row_tiles);
  int64_t ranges = (int64_t(cus) + units - 1) / units;
  ranges = std::min(ranges, (most + p->turns - 1) / p->turns);
  p->ranges = uint32_t(ranges > 1 ? ranges : 1);
  return CBK_OK;
}

size_t ml_bytes(const Plan& p, int64_t rows, int64_t hq) {
  return (size_t(2) * p.ranges * size_t(rows) * size_t(hq) * sizeof(float2) + 255) & ~size_t(255);
}

size_t plan_bytes(const Plan& p, int64_t rows, int64_t hq, int64_t d) {
  return ml_bytes(p, rows, hq) + size_t(2) * p.ranges * size_t(rows) * size_t(hq) * size_t(d) * sizeof(float);
}

template <int DT, int NG, int P>
int launch_pieces(const Int4AttnArgs& a, hipStream_t s) {
  const uint64_t groups = uint64_t(a.hkv / a.heads) * a.row_tiles * ((a.ranges + 7) / 8 * 8);
  const uint32_t threads = 64 * a.heads * a.turns;
  CBK_REQUIRE(groups * threads < (uint64_t(1) << 32), "int4 attention: %llu workgroups exceed one launch",
              (unsigned long long)groups);
  const dim3 grid(uint32_t(groups), 1, 1), block(threads);
  if (column_groups(uint64_t(a.rows) * a.group) == 2)
    hipLaunchKernelGGL((int4_attn_kernel<DT, NG, 2, P>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((int4_attn_kernel<DT, NG, 1, P>), grid, block, 0, s, a);
  return launch_status("int4 attention");
}

template <int DT, int NG>
int launch(const Int4AttnArgs& a, bool pieces16, hipStream_t s) {
  // 16-byte pieces of a row: whole ones, where the pages are aligned to them. In
  // 4-byte pieces a tile of 128 dims takes four times the requests, and the addresses
  // spill 40 to 50 registers: 64 sequences of up to 16K keys 369 us, 217 in 16 bytes.
  constexpr int P = kInt4GroupBytes * NG % 16 == 0 ? 16 : 4;
  if (int rc = pieces16 ? launch_pieces<DT, NG, P>(a, s) : launch_pieces<DT, NG, 4>(a, s)) return rc;
  // a sequence of many ranges: more lanes for each of its rows (a call in us with
  // 8 / 32 sets of them, 32 over 8 heads x 128: 256 ranges a sequence 32.3 /
  // 25.1, 64 35.4 / 34.0, 16 42.1 / 42.3, 8 62.1 / 65.1)
  const dim3 grid(a.rows * a.hq, a.batch);
  if (a.ranges > 16 * a.batch) hipLaunchKernelGGL((int4_attn_merge_kernel<DT, 32 * NG, 32>), grid, dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((int4_attn_merge_kernel<DT, 32 * NG, 8>), grid, dim3(256), 0, s, a);
  return launch_status("int4 attention merge");
}

}  // namespace
}  // namespace cbk

extern "C" {

size_t cbk_paged_attention_int4_workspace_bytes(int64_t batch, int64_t rows, int64_t hq, int64_t hkv, int64_t head_dim,
                                                int64_t max_len, int32_t dtype) {
  using namespace cbk;
  Plan p;
  if (batch <= 0 || head_dim <= 0 || plan_of(batch, rows, hq, hkv, max_len, dtype, &p)) return 0;
  return plan_bytes(p, rows, hq, head_dim);
}

int cbk_paged_attention_int4(const void* q_dev, int64_t q_batch_stride, int64_t q_row_stride, int64_t q_head_stride,
                             int64_t batch, int64_t rows, int64_t hq, const cbk_kv_desc* kv, int64_t hkv,
                             int64_t head_dim, const int32_t* tables_dev, int64_t table_stride, int64_t table_width,
                             const int32_t* lens_dev, float scale, int32_t dtype, void* out_dev,
                             int64_t out_batch_stride, int64_t out_row_stride, int64_t out_head_stride,
                             void* workspace_dev, size_t workspace_bytes, cbk_stream_t stream) {
  using namespace cbk;
  clear_error();
  if (int rc = validate_desc(kv)) return rc;
  CBK_REQUIRE(dtype == CBK_DTYPE_F32 || dtype == CBK_DTYPE_BF16 || dtype == CBK_DTYPE_F16, "dtype %d", int(dtype));
  CBK_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim %lld: 64 or 128 supported", (long long)head_dim);
  CBK_REQUIRE(hkv > 0 && kv->row_bytes == hkv * int4_row_bytes(head_dim), "a 4-bit row of %lld x %lld is not %lld bytes",
              (long long)hkv, (long long)head_dim, (long long)kv->row_bytes);
  CBK_REQUIRE(std::isfinite(scale), "scale must be finite");
  CBK_REQUIRE(table_width >= 0 && table_width < (int64_t(1) << 31) && table_stride >= 0,
              "block table width out of range");
  CBK_REQUIRE(kv->num_blocks < (int64_t(1) << 31), "num_blocks out of range");
  int64_t max_len = table_width * kv->block_size;
  Plan p;
  if (int rc = plan_of(batch, rows, hq, hkv, max_len, dtype, &p)) return rc;
  if (batch == 0) return CBK_OK;
  CBK_REQUIRE(q_dev && out_dev && lens_dev && (tables_dev || table_width == 0), "NULL pointer");
  const int64_t words[4] = {int64_t(reinterpret_cast<uintptr_t>(kv->k_base)),
                            int64_t(reinterpret_cast<uintptr_t>(kv->v_base)), kv->block_stride, kv->token_stride};
  const int vec = common_vec_bytes(words, 4);
  CBK_REQUIRE(vec >= 4, "4-bit pages must be 4-byte aligned");
  const size_t need = plan_bytes(p, rows, hq, head_dim);
  if (workspace_dev == nullptr || workspace_bytes < need)
    return set_error(CBK_ERR_WORKSPACE, "int4 attention workspace %zu < %zu bytes", workspace_bytes, need);
  CBK_REQUIRE((reinterpret_cast<uintptr_t>(workspace_dev) & 255) == 0, "workspace must be 256-byte aligned");
  Int4AttnArgs a;
  a.q = q_dev;
  a.out = out_dev;
  a.q_batch = q_batch_stride;
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.out_batch = out_batch_stride;
  a.out_row = out_row_stride;
  a.out_head = out_head_stride;
  a.k_base = static_cast<const char*>(kv->k_base);
  a.v_base = static_cast<const char*>(kv->v_base);
  a.block_stride = kv->block_stride;
  a.token_stride = kv->token_stride;
  a.tables = tables_dev;
  a.table_stride = table_stride;
  a.lens = lens_dev;
  a.batch = uint32_t(batch);
  a.rows = uint32_t(rows);
  a.hq = uint32_t(hq);
  a.hkv = uint32_t(hkv);
  a.group = uint32_t(hq / hkv);
  a.num_blocks = uint32_t(kv->num_blocks);
  a.max_len = uint32_t(max_len);
  a.row_tiles = p.row_tiles;
  a.ranges = p.ranges;
  a.heads = p.heads;
  a.turns = p.turns;
  a.scale = scale;
  const int64_t es = dtype == CBK_DTYPE_F32 ? 4 : 2;
  const int64_t pieces[4] = {int64_t(reinterpret_cast<uintptr_t>(q_dev)), q_batch_stride * es, q_row_stride * es, q_head_stride * es};
  a.q_pieces = common_vec_bytes(pieces, 4) == 16;
  a.block_div = FastDiv::make(uint32_t(kv->block_size));
  a.ml = static_cast<float2*>(workspace_dev);
  a.o = reinterpret_cast<float*>(static_cast<char*>(workspace_dev) + ml_bytes(p, rows, hq));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool p16 = vec == 16;
#define CBK_INT4_ATTN(DT) return head_dim == 128 ? launch<DT, 4>(a, p16, s) : launch<DT, 2>(a, p16, s);
  switch (dtype) {
    case CBK_DTYPE_F32: CBK_INT4_ATTN(CBK_DTYPE_F32)
    case CBK_DTYPE_BF16: CBK_INT4_ATTN(CBK_DTYPE_BF16)
    default: CBK_INT4_ATTN(CBK_DTYPE_F16)
  }
#undef CBK_INT4_ATTN
}

}  // extern "C"
