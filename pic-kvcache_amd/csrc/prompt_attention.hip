// Causal attention of packed prompts for gfx950: sequences of different
// lengths side by side in one [tokens, heads, head_dim] tensor each of
// queries, keys and values,
//
//   out[i, h] = sum_{k <= pos_i} softmax_k( scale q[i, h] . key[k, h / G] ) value[k, h / G]
//
// with k over the query's own sequence and pos_i its place in it: a sequence's
// last query is its last key (with more keys than queries the first keys are
// context from before; with fewer the first queries see nothing). Logits and
// softmax in float32, G = Hq / Hkv.
//
// Bound by the matrix cores' rate and, beside it, by the VALU work per logit
// (a fused multiply-add, an exp2, half a conversion). The tiling, the LDS
// blocks and the software pipeline are those of the side-forward attention
// (attention.hip): one workgroup of 4 waves per 128 rows of (query, group
// head) of one sequence and KV head, K/V blocks of 32 keys by DMA through
// rings of four LDS buffers, S^T = K . Q^T of block b + 1 and P . V of block b
// - 1 issued beside the softmax of block b, exponents against a fixed
// reference. It differs in what it does not do: no logit is rounded to the
// inputs' type, positions and sequences follow from the lengths.
// The weights, as the second product's operand, are rounded to the inputs' type
// (half a step each, as the output itself); their sums are of the rounded ones,
// in float32, so that equal values come out as they are. float16 weights of less
// than 2^-14 of the reference's are rounded to 2^-25 of that: the reference, from the
// first block, is at 1, for later weights may be up to 2^16 times it before the
// tile is computed again.
//
// float32 inputs: prompt_attention_f32.hip.
//
// Which sequence and tile a workgroup has is found on the device (the lengths
// stay there).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention_mfma.hpp"
#include "prompt_attention.hpp"

namespace cbk {
namespace {

constexpr int kWaves = 4;
constexpr int kRowTiles = 2;  // 16-row tiles per wave
constexpr int kRows = kWaves * 16 * kRowTiles;
constexpr int kKeyBlock = kAttnKeyBlock;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
// The lazy rescaling's logits are in units of 2 log 2: float32's largest logit
// times log2 e is past its range, half of that is not. Its headroom: 2^8.
constexpr float kUnit = 2.f;
constexpr float kRescale = 8.f / kUnit;
constexpr float kLargest = 0x1p26f;  // to there a reference is rounded by 4 at most: a common factor of 2^4 in the weights

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// p = 2^(S c2 - m) (MASK: 0 past each row's position), rounded to the dtype: the A
// operand of P . V; nms = -m (0 while m is -inf). In one multiply-add, which leaves
// m's rounding error in the exponent, harmless up to kLargest; LAZY, for any m: in
// units of kUnit, the product rounded as m was.
template <bool F16, int RT, bool MASK, bool LAZY>
__device__ __forceinline__ void probs_block(const f32x4 (&s)[RT][2], int32_t k0, float c2, const int32_t (&rpos)[RT],
                                            const float (&nms)[RT], uint32_t grp, typename Ops<F16>::A8 (&pa)[RT]) {
  using O = Ops<F16>;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    typename O::A4 ph[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y;
        if constexpr (LAZY) {
#pragma clang fp contract(off)
          const float x = s[t][h][i] * c2;
          y = (x + nms[t]) * kUnit;
        } else {
          y = fmaf(s[t][h][i], c2, nms[t]);
        }
        if constexpr (MASK) y = k0 + 16 * h + int32_t(4 * grp) + i > rpos[t] ? kNegInf : y;
        p[i] = __builtin_amdgcn_exp2f(y);
      }
      ph[h] = __builtin_bit_cast(typename O::A4, u32x2{O::pack(p[0], p[1]), O::pack(p[2], p[3])});
    }
    pa[t] = __builtin_shufflevector(ph[0], ph[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// This lane's largest logit of each row tile (in c2's units; -inf: none visible).
template <int RT>
__device__ __forceinline__ void logits_max(const f32x4 (&s)[RT][2], int32_t k0, float c2, const int32_t (&rpos)[RT],
                                           uint32_t grp, float (&lm)[RT]) {
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    lm[t] = kNegInf;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k0 + 16 * h + int32_t(4 * grp) + i <= rpos[t]) lm[t] = fmaxf(lm[t], s[t][h][i] * c2);
  }
}

// K and V blocks through rings of four LDS buffers, requested three steps
// ahead of the one that reads them.
template <bool F16, int D, int RT>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2, D == 64 ? 3 : 2))) void prompt_kernel(
    const PromptArgs a) {
  constexpr int W = kWaves;
  constexpr uint32_t P = D / 8;                        // 16-byte pieces per key row
  constexpr uint32_t kInsts = kKeyBlock * P / 64 / W;  // requests per wave per block, each of K and V
  constexpr uint32_t kRowsPerInst = 64 / P;
  constexpr int kBuffers = 4;
  static_assert(kInsts >= 1 && W * 16 * D <= 2 * kBuffers * kKeyBlock * D, "wave count vs block and staging");
  // K blocks, then V blocks; the output staging reuses the whole region
  __shared__ __attribute__((aligned(16))) uint16_t kvbuf[2][kBuffers][kKeyBlock * D];
  auto& kbuf = kvbuf[0];
  auto& vbuf = kvbuf[1];
  using O = Ops<F16>;
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row = lane & 15, grp = lane >> 4;
  // workgroup -> (tile, key range, KV head), the KV head fastest
  const uint32_t S = a.parts.splits;
  const uint32_t kvh = __builtin_amdgcn_readfirstlane(blockIdx.x % a.hkv);
  const uint32_t rest = __builtin_amdgcn_readfirstlane(blockIdx.x / a.hkv);
  const uint32_t rank = S == 1 ? rest : __builtin_amdgcn_readfirstlane(rest / S);
  const uint32_t split = rest - rank * S;
  const PromptTile tl = prompt_tile<kRows>(a, rank, lane);
  if (tl.beyond) {  // no tile: rows that belong to no sequence
    if (S == 1) prompt_outside(a, tl, kvh, D * 2);
    return;
  }
  if (tl.none) return;
  const uint32_t nrows = tl.nq * a.group;
  const uint32_t r_wave = tl.tile * kRows + wave * 16 * RT;
  const int32_t shift = int32_t(tl.nk) - int32_t(tl.nq);  // a query's position minus its index
  const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;  // a negative scale goes into the queries
  const float c2 = fabsf(a.scale) * kLog2e, c2_lazy = fabsf(a.scale) * (kLog2e / kUnit);

  // this lane's rows (one per row tile): (query, head) and their Q fragments
  typename O::A8 qf[RT][D / 32];
  int32_t rpos[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const uint32_t r = r_wave + 16 * t + row;
    const bool valid = r < nrows;
    const uint32_t qi = valid ? a.group_div.div(r) : 0;
    const uint32_t qh = kvh * a.group + (valid ? r - qi * a.group : 0);
    rpos[t] = valid ? int32_t(qi) + shift : -1;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + int64_t(tl.q0 + qi) * a.q_token + int64_t(qh) * a.q_head;
#pragma unroll
    for (int st = 0; st < D / 32; ++st) {
      u32x4 w = u32x4(0u);
      if (valid) w = *reinterpret_cast<const u32x4*>(src + 32 * st + 8 * grp) ^ u32x4(sign);
      qf[t][st] = __builtin_bit_cast(typename O::A8, w);
    }
  }
  // the wave's earliest and latest positions, the workgroup's blocks: this
  // workgroup's range of them
  const uint32_t last_row = min(nrows, r_wave + 16 * RT);
  int32_t wmax = r_wave < nrows ? int32_t(a.group_div.div(last_row - 1)) + shift : -1;
  int32_t wmin = r_wave < nrows ? int32_t(a.group_div.div(r_wave)) + shift : 0x7fffffff;
  const int32_t gmax = int32_t(a.group_div.div(min(nrows, (tl.tile + 1) * kRows) - 1)) + shift;
  const int32_t tile_blocks = gmax < 0 ? 0 : gmax / kKeyBlock + 1;
  int32_t b_lo = 0, nblocks = __builtin_amdgcn_readfirstlane(tile_blocks);
  if (S > 1) {
    b_lo = __builtin_amdgcn_readfirstlane(int32_t(uint32_t(tile_blocks) * split / S));
    nblocks = __builtin_amdgcn_readfirstlane(int32_t(uint32_t(tile_blocks) * (split + 1) / S)) - b_lo;
  }
  const int32_t key0 = b_lo * kKeyBlock;
  const int32_t nk = int32_t(tl.nk) - key0;
  const uint16_t* const k_seq = static_cast<const uint16_t*>(a.k) + int64_t(tl.k0) * a.k_token + int64_t(kvh) * a.k_head;
  const uint16_t* const k_range = k_seq + int64_t(key0) * a.k_token;
  const uint16_t* const v_range =
      static_cast<const uint16_t*>(a.v) + int64_t(tl.k0 + key0) * a.v_token + int64_t(kvh) * a.v_head;
#pragma unroll
  for (int t = 0; t < RT; ++t) rpos[t] -= key0;
  wmax -= key0;
  wmin -= key0;

  // per row tile: the reference m (log2 units, or kUnit of them where it is lazy) and
  // -m for the exponents (0 while m is -inf)
  float m[RT], nms[RT];
  f32x4 o[RT][D / 16], ol[RT];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      m[t] = kNegInf;
      nms[t] = 0.f;
      ol[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < D / 16; ++c) o[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  clear();
  // nothing of the compiler's own in flight once the requests start
  CBK_WAIT_VM_LGKM0(0);

  // per-lane request offsets (key row of the block, swizzled piece), bytes
  uint32_t krow[kInsts], koff[kInsts], voff[kInsts];
#pragma unroll
  for (uint32_t j = 0; j < kInsts; ++j) {
    krow[j] = (wave * kInsts + j) * kRowsPerInst + lane / P;
    const uint32_t piece = (lane % P) ^ lds_swizzle<D>(krow[j]);
    koff[j] = uint32_t((krow[j] * a.k_token + piece * 8) * 2);
    voff[j] = uint32_t((krow[j] * a.v_token + piece * 8) * 2);
  }
  // one block's requests from its base to its buffer; rows past the
  // sequence's end repeat its last key (masked)
  auto request_rows = [&](const void* base, int32_t left, int64_t stride, const uint32_t (&offs)[kInsts],
                          uint32_t l) __attribute__((always_inline)) {
    if (left >= kKeyBlock) {
      lds_dma16n<kInsts>(base, offs, l + wave * kInsts * 1024);
    } else {
      const uint32_t last = uint32_t(left - 1);
#pragma unroll
      for (uint32_t j = 0; j < kInsts; ++j) {
        const uint32_t back = krow[j] - min(krow[j], last);  // rows to step back
        lds_dma16(base, offs[j] - uint32_t(back * stride * 2), l + (wave * kInsts + j) * 1024);
      }
    }
  };
  // block b (clamped: past the end repeats the last) into buffer b % kBuffers
  auto request = [&](int32_t b, const uint16_t* src, int64_t stride, const uint32_t (&offs)[kInsts],
                     uint16_t (&bufs)[kBuffers][kKeyBlock * D]) {
    const uint32_t l = lds_address(bufs[b % kBuffers]);
    b = min(b, nblocks - 1);
    request_rows(src + int64_t(b) * kKeyBlock * stride, nk - b * kKeyBlock, stride, offs, l);
  };
  const BlockOffsets<D> off(lane);
  // this wave's blocks: [0, b_m) are visible to all of its rows, [b_m, b_w)
  // masked, [b_w, nblocks) past its latest position (skipped; the wave still
  // takes its part in the requests and barriers).
  const int32_t b_w = wmax < 0 ? 0 : min(wmax / kKeyBlock + 1, nblocks);
  const int32_t b_m = wmax < 0 ? 0 : min(int32_t((int64_t(max(wmin, -1)) + 1) / kKeyBlock), b_w);
  // Lazy rescaling (the first step, and the rare second pass): exponents stay
  // relative to a reference that is raised -- and O rescaled, one step later,
  // between P . V of the block before and its own -- when some lane sees a
  // logit above it by more than kRescale.
  bool pending = false;  // O still to be rescaled by alpha
  float alpha[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) alpha[t] = 1.f;
  auto rescale_o = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float ao[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ao[i] = __shfl(alpha[t], int(4 * grp + i));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[t][c][i] *= ao[i];
        ol[t][i] *= ao[i];
      }
    }
  };
  // The steps' request streams: K kBuffers blocks ahead of the step, V two
  // fewer, clamped at the last block (every block before it is whole).
  constexpr uint32_t kSlot = kKeyBlock * D * 2, kVOffset = kBuffers * kSlot;
  const int64_t kstep = int64_t(kKeyBlock) * a.k_token * 2, vstep = int64_t(kKeyBlock) * a.v_token * 2;
  const int32_t last_left = nk - (nblocks - 1) * kKeyBlock;  // keys from the last block on
  const char* const kg0 = reinterpret_cast<const char*>(k_range) + int64_t(min(kBuffers, nblocks - 1)) * kstep;
  const char* const vg0 = reinterpret_cast<const char*>(v_range) + int64_t(min(kBuffers - 2, nblocks - 1)) * vstep;
  const char* kg = kg0;
  const char* vg = vg0;
  auto stream = [&](int32_t j, const char*& g, int64_t stride_bytes, int64_t stride, const uint32_t (&offs)[kInsts],
                    uint32_t l) __attribute__((always_inline)) {
    const bool inner = j < nblocks - 1;
    request_rows(g, inner ? kKeyBlock : last_left, stride, offs, l);
    if (inner) g += stride_bytes;
  };
  // P . V of a block some of whose keys some rows do not see, one key at a
  // time and without the products of zero: what such a row's unseen value rows
  // hold, infinities and NaN among it, does not reach it.
  auto pv_careful = [&](const uint16_t* vs, const typename O::A8 (&pa)[RT]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const u32x4 pw = __builtin_bit_cast(u32x4, pa[t]);
#pragma nounroll
      for (int key = 0; key < kKeyBlock; ++key) {
        // lane (row, g) holds keys 4 g + e (words 0, 1) and 16 + 4 g + e (words 2, 3)
        const int half = key >> 4, g = (key >> 2) & 3, e = key & 3;
        const uint32_t w = half ? (e >> 1 ? pw[3] : pw[2]) : (e >> 1 ? pw[1] : pw[0]);
        const float mine = e & 1 ? O::hi(w) : O::lo(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __shfl(mine, int(16 * g + 4 * grp + i));
          if (p == 0.f) continue;
          ol[t][i] += p;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const uint32_t dim = 16 * c + row;
            const uint16_t bits = vs[key * D + ((dim / 8) ^ lds_swizzle<D>(key)) * 8 + dim % 8];
            o[t][c][i] = fmaf(p, O::lo(bits), o[t][c][i]);
          }
        }
      }
    }
  };
  // KIND: 0 visible, 1 masked, 2 P . V of the wave's last block only, 3 no
  // work; FIRST: no block before; PHASE: b % kPhases when known at compile time
  // (then every LDS address is a lane's offset plus a constant), or -1; FIX:
  // exponents against the fixed reference. sc holds S^T of block b, pp P of
  // block b - 1; the step leaves S^T of block b + 1 in sn and P of block b in
  // pc (two register sets taken in turn: no copies between steps).
  auto step = [&](auto kind, auto first, auto phase, auto fix, int32_t b, f32x4 (&sc)[RT][2],
                  f32x4 (&sn)[RT][2], typename O::A8 (&pp)[RT], typename O::A8 (&pc)[RT])
                  __attribute__((always_inline)) {
    constexpr int KIND = decltype(kind)::value;
    constexpr bool FIRST = decltype(first)::value;
    constexpr int PHASE = decltype(phase)::value;
    constexpr bool FIX = decltype(fix)::value;
    // K(b + 1) and V(b - 1) have landed: all but the requests of the last kBuffers - 2 steps
    CBK_WAIT_VM_LGKM0(2 * (kBuffers - 2) * kInsts);
    asm volatile("s_barrier" ::: "memory");
    uint32_t kb_addr, vb_addr, kw_addr, vw_addr;
    if constexpr (PHASE >= 0) {
      kw_addr = lds_address(kbuf[PHASE % kBuffers]);
      vw_addr = lds_address(vbuf[(PHASE + kBuffers - 2) % kBuffers]);
      kb_addr = lds_address(kbuf[(PHASE + 1) % kBuffers]);
      vb_addr = lds_address(vbuf[(PHASE + kBuffers - 1) % kBuffers]);
    } else {
      const uint32_t k0 = lds_address(kbuf[0]);
      kw_addr = k0 + (uint32_t(b) % kBuffers) * kSlot;
      kb_addr = k0 + (uint32_t(b + 1) % kBuffers) * kSlot;
      vw_addr = k0 + (uint32_t(b + kBuffers - 2) % kBuffers) * kSlot + kVOffset;
      vb_addr = k0 + (uint32_t(b + kBuffers - 1) % kBuffers) * kSlot + kVOffset;
      asm volatile("" : "+s"(kb_addr), "+s"(vb_addr));
    }
    stream(b + kBuffers, kg, kstep, a.k_token, koff, kw_addr);      // into the K buffer block b used
    stream(b + kBuffers - 2, vg, vstep, a.v_token, voff, vw_addr);  // into the V buffer block b - 2 used
    if constexpr (KIND < 3) {
      const uint16_t* ks = (const uint16_t*)(__attribute__((address_space(3))) const uint16_t*)(size_t)kb_addr;
      const uint16_t* vs = (const uint16_t*)(__attribute__((address_space(3))) const uint16_t*)(size_t)vb_addr;
      auto pv = [&]() __attribute__((always_inline)) {
        if (!FIX && b - 1 >= b_m) pv_careful(vs, pp);
        else pv_block<F16, D, RT>(vs, off, pp, o, ol);
      };
      if constexpr (KIND < 2) {
        qk_block<F16, D, RT>(ks, off, qf, sn);
        if constexpr (!FIX) {
          float lm[RT];
          logits_max<RT>(sc, b * kKeyBlock, c2_lazy, rpos, grp, lm);
          uint64_t over = 0;
#pragma unroll
          for (int t = 0; t < RT; ++t) over |= __ballot(lm[t] > m[t] + kRescale);
          if (pending || over != 0) {
            if (pending) rescale_o();
            pending = false;
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              alpha[t] = 1.f;
              if (__any(lm[t] > m[t] + kRescale)) {
                const float bm = fmaxf(lm[t], __shfl_xor(lm[t], 16));
                const float mn = fmaxf(m[t], fmaxf(bm, __shfl_xor(bm, 32)));
                alpha[t] = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f((m[t] - mn) * kUnit);
                m[t] = mn;
                nms[t] = mn == kNegInf ? 0.f : -mn;  // a row that sees no key of the range yet
                pending = true;
              }
            }
          }
        }
        probs_block<F16, RT, KIND == 1, !FIX>(sc, b * kKeyBlock, FIX ? c2 : c2_lazy, rpos, nms, grp, pc);
        if constexpr (!FIRST) pv();
        // P of block b is computed here, beside P . V of block b - 1 (the
        // compiler would otherwise sink it to its use in the next step)
#pragma unroll
        for (int t = 0; t < RT; ++t) asm volatile("" : "+v"(pc[t]));
      } else if constexpr (!FIRST) {
        if constexpr (!FIX) {
          if (pending) rescale_o();
          pending = false;
        }
        pv();
      }
    }
  };
  using visible = std::integral_constant<int, 0>;
  using masked = std::integral_constant<int, 1>;
  using last = std::integral_constant<int, 2>;
  using none = std::integral_constant<int, 3>;
  using yes = std::true_type;
  using no = std::false_type;
  f32x4 sa[RT][2], sb[RT][2];
  typename O::A8 pa[RT], pb[RT];
  using any = std::integral_constant<int, -1>;
  // one step with its buffers chosen at run time, S^T of block b in sa and P
  // of block b - 1 in pa before and after
  auto single = [&](auto kind, auto first, auto fix, int32_t& b) __attribute__((always_inline)) {
    step(kind, first, any(), fix, b++, sa, sb, pa, pb);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      sa[t][0] = sb[t][0];
      sa[t][1] = sb[t][1];
      pa[t] = pb[t];
    }
  };
  // steps [b, end) of one kind: kPhases at a time from a multiple of kPhases
  // (the rings and the two register sets back where they started), single
  // steps at the edges; the rare second pass takes single steps only
  constexpr int kPhases = 4;
  static_assert(kPhases % kBuffers == 0 && kPhases % 2 == 0, "whole turns of the rings and register sets");
  auto run = [&](auto kind, auto fix, int32_t& b, int32_t end) __attribute__((always_inline)) {
    if constexpr (decltype(fix)::value && decltype(kind)::value == 0) {
      while (b < end && b % kPhases != 0) single(kind, no(), fix, b);
      for (; b + kPhases <= end; b += kPhases) {
        step(kind, no(), std::integral_constant<int, 0>(), fix, b, sa, sb, pa, pb);
        step(kind, no(), std::integral_constant<int, 1>(), fix, b + 1, sb, sa, pb, pa);
        step(kind, no(), std::integral_constant<int, 2>(), fix, b + 2, sa, sb, pa, pb);
        step(kind, no(), std::integral_constant<int, 3>(), fix, b + 3, sb, sa, pb, pa);
      }
    }
    while (b < end) single(kind, no(), fix, b);
  };
  auto lds_at = [](uint32_t l) { return (const uint16_t*)(__attribute__((address_space(3))) const uint16_t*)(size_t)l; };
  // one pass over the blocks; the first step always takes the lazy path (it
  // sets the references that are not set yet from the range's first block)
  auto pass = [&](auto fix) __attribute__((always_inline)) {
    // the first kBuffers blocks of K and two fewer of V ahead of step 0, in
    // the order the steps wait for them; then every wave takes steps 0 ..
    // nblocks. A range past the first also reads the sequence's block 0, into
    // the V buffer that step 1 fills first.
    const bool first_ref = decltype(fix)::value && b_lo > 0;
    if (first_ref) lds_dma16n<kInsts>(k_seq, koff, lds_address(vbuf[kBuffers - 1]) + wave * kInsts * 1024);
    request(0, k_range, a.k_token, koff, kbuf);
    request(1, k_range, a.k_token, koff, kbuf);
#pragma unroll
    for (int j = 0; j < kBuffers - 2; ++j) {
      request(2 + j, k_range, a.k_token, koff, kbuf);
      request(j, v_range, a.v_token, voff, vbuf);
    }
    CBK_WAIT_VM_LGKM0((2 * (kBuffers - 2) + 1) * kInsts);  // K(0), and the sequence's block 0, have landed
    asm volatile("s_barrier" ::: "memory");
    if (first_ref && b_w > 0) {
      qk_block<F16, D, RT>(lds_at(lds_address(vbuf[kBuffers - 1])), off, qf, sa);
      float lm[RT];
      logits_max<RT>(sa, -key0, c2, rpos, grp, lm);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float bm = fmaxf(lm[t], __shfl_xor(lm[t], 16));
        m[t] = fmaxf(bm, __shfl_xor(bm, 32));
        nms[t] = m[t] == kNegInf ? 0.f : -m[t];
      }
    }
    int32_t b = 0;
    if (b_w > 0) {
      qk_block<F16, D, RT>(lds_at(lds_address(kbuf[0])), off, qf, sa);
      // the masked form, whatever the block: one copy of the step fewer
      if (first_ref) {
        single(masked(), yes(), fix, b);
      } else {
        single(masked(), yes(), no(), b);
        if constexpr (decltype(fix)::value) {  // the references in log2 units
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            m[t] *= kUnit;
            nms[t] *= kUnit;
          }
        }
      }
    }
    run(visible(), fix, b, b_m);
    run(masked(), fix, b, b_w);
    if (b_w > 0)
      step(last(), no(), any(), fix, b++, sa, sb, pa, pb);
    else
      step(none(), yes(), any(), fix, b++, sa, sb, pa, pb);
    for (; b <= nblocks; ++b) step(none(), no(), any(), fix, b, sa, sb, pa, pb);
    CBK_WAIT_VM_LGKM0(0);  // no LDS write in flight past this point
  };
  // Fixed reference: every row keeps the maximum of the sequence's block 0,
  // where a row that sees anything sees key 0 (a logit of the row, so no term
  // exceeds 2^(max - m)): no per-logit maximum. The key ranges share it. A row
  // whose terms outgrew it (its sum past 2^100, or a term past float16), that
  // has no reference although it sees keys, or one past kLargest, or whose output
  // is not finite is recomputed, workgroup-wide, with the lazy rescaling and with
  // the masked blocks' P . V key by key.
  __shared__ uint32_t s_redo;
  float to_unit = 1.f / kUnit;  // of m
  if (nblocks > 0) {
    pass(yes());
    bool bad = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      bad |= !(fabsf(m[t]) < kLargest) && rpos[t] >= 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bad |= !finite_bits(ol[t][i]) || ol[t][i] >= 0x1p100f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) bad |= !finite_bits(o[t][c][i]);
      }
    }
    if (threadIdx.x == 0) s_redo = 0;
    __syncthreads();
    if (bad) s_redo = 1;
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(s_redo)) {  // uniform: the pass's loops stay scalar
      pending = false;
      clear();
      kg = kg0;
      vg = vg0;
      pass(no());
      to_unit = 1.f;
    }
  }
  __syncthreads();  // every wave is done with the K buffers the output staging reuses

  if (S > 1) {  // this range's partial results (attention_split.hpp)
    const uint64_t rows_all = uint64_t(a.total_q) * a.hq;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float rm = __shfl(m[t], int(4 * grp + i));
        const uint32_t rr = r_wave + 16 * t + 4 * grp + i;
        if (rr >= nrows) continue;
        const uint32_t qi = a.group_div.div(rr);
        const uint64_t id = split * rows_all + uint64_t(tl.q0 + qi) * a.hq + kvh * a.group + rr - qi * a.group;
        // (a row that sees no key of the range may have the sequence's first reference, infinite perhaps)
        if (row == 0) a.parts.ml[id] = make_float2(ol[t][i] == 0.f ? kNegInf : rm * to_unit, ol[t][i]);
        float* po = a.parts.o + id * D + row;
        if (nblocks > 0)
#pragma unroll
          for (int c = 0; c < D / 16; ++c) po[16 * c] = o[t][c][i];
      }
    return;
  }
  // normalize and write, one row tile at a time through the wave's LDS
  // staging area (the K buffers are free now): whole 16-byte pieces per row
  uint16_t* os = &kvbuf[0][0][0] + wave * 16 * D;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    // row sums of the rounded probabilities, already in O's layout
    float lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = ol[t][i] == 0.f ? 0.f : 1.f / ol[t][i];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const uint32_t u01 = O::pack(o[t][c][0] * lo[0], o[t][c][1] * lo[1]);
      const uint32_t u23 = O::pack(o[t][c][2] * lo[2], o[t][c][3] * lo[3]);
      const uint32_t col = 16 * c + row;
      os[(4 * grp + 0) * D + col] = uint16_t(u01 & 0xffffu);
      os[(4 * grp + 1) * D + col] = uint16_t(u01 >> 16);
      os[(4 * grp + 2) * D + col] = uint16_t(u23 & 0xffffu);
      os[(4 * grp + 3) * D + col] = uint16_t(u23 >> 16);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 16 * (D / 8) / 64; ++c) {
      const uint32_t idx = lane + 64 * c;
      const uint32_t orow = idx / (D / 8), chunk = idx % (D / 8);
      const uint32_t rr = r_wave + 16 * t + orow;
      if (rr < nrows) {
        const uint32_t qi = a.group_div.div(rr), oh = kvh * a.group + rr - qi * a.group;
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) + int64_t(tl.q0 + qi) * a.out_token +
                                  int64_t(oh) * a.out_head + chunk * 8) =
            *reinterpret_cast<const u32x4*>(&os[orow * D + chunk * 8]);
      }
    }
    __syncthreads();
  }
}

template <bool F16>
int launch_16(const PromptArgs& a, uint32_t d, hipStream_t s) {
  const uint64_t groups = prompt_tiles(a, kRows) * a.hkv * a.parts.splits;
  CBK_REQUIRE(groups * 64 * kWaves < (uint64_t(1) << 32), "prompt attention: %llu workgroups exceed one launch",
              (unsigned long long)groups);
  const dim3 grid(static_cast<uint32_t>(groups)), block(64 * kWaves);
  if (d == 128) hipLaunchKernelGGL((prompt_kernel<F16, 128, kRowTiles>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((prompt_kernel<F16, 64, kRowTiles>), grid, block, 0, s, a);
  return launch_status("prompt attention");
}

int check_sizes(int64_t total_q, int64_t total_k, int64_t batch, int64_t hq, int64_t hkv, int64_t head_dim,
                int32_t dtype) {
  CBK_REQUIRE(dtype == CBK_DTYPE_F32 || dtype == CBK_DTYPE_BF16 || dtype == CBK_DTYPE_F16, "dtype %d", int(dtype));
  CBK_REQUIRE(total_q >= 0 && total_k >= 0 && total_q < (int64_t(1) << 30) && total_k < (int64_t(1) << 30),
              "tokens out of range");
  CBK_REQUIRE(batch >= 0 && batch < (int64_t(1) << 24), "batch out of range");
  CBK_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "query heads must be divisible by KV heads");
  CBK_REQUIRE(total_q * hq < (int64_t(1) << 31), "tokens * heads too large");
  CBK_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim %lld: 64 or 128 supported", (long long)head_dim);
  return CBK_OK;
}

// The ranges of the side attention's rules (attention_split.hpp), with the average
// sequence's keys, for the lengths stay on the device; a causal tile sees half of them
// in the mean. us a call without ranges / with those taken (their number):
//  16 bits, 32 heads over 8 x 128: one prompt of up to 4000, several of 100 to 1000
//    none; 64 queries of 2000 keys 46.3 / 21.8 (8), 256 of 16000 310 / 91.5 (11), 1024 of
//    32768 631 / 482 (4), four of 128 of 4000 84.7 / 50.0 (4). Over all sizes tried,
//    16 over 8 x 128 and 16 over 4 x 64 among them, at most 4% longer than without
//    (a prompt of 4000, 16 over 4 x 64: 60.7 / 63.1 (2)).
//  float32, 16 over 8 x 128: 64 queries of 2000 keys 172 / 30.2 (15), 256 of 16000
//    1410 / 211 (12); one prompt of 300 32.5 / 25.4 (2), 1000 89.5 / 50.2 (3), 2000
//    188 / 128 (3); two of 1000 99.1 / 81.6 (3); of 1024, 333, 777 and 256 101 / 74.1 (2).
//    Equal prompts whose tiles are most of a round lose: four of 700 74.6 / 81.6 (2), six of
//    500 58.9 / 72.1 (2), eight of 300 39.3 / 53.7 (2), and 16 over 4 x 64 23.0 / 35.3 (2);
//    nothing that the host knows tells them from uneven ones, which gain.
uint32_t splits_of(int64_t total_q, int64_t total_k, int64_t batch, int64_t hq, int64_t hkv, int64_t head_dim,
                   int32_t dtype) {
  const uint64_t group = uint64_t(hq / hkv);
  const uint64_t per = dtype == CBK_DTYPE_F32 ? prompt_f32_rows(uint64_t(total_q) * group, uint64_t(hkv)) : kRows;
  const uint64_t tiles = (uint64_t(total_q) * group / uint64_t(batch) + per - 1) / per * uint64_t(batch);
  const int64_t nk = (total_k + batch - 1) / batch;
  if (dtype == CBK_DTYPE_F32) return attn_f32_splits(tiles * uint64_t(hkv), nk);
  return attn_splits(tiles * uint64_t(hkv), uint64_t(total_q) * uint64_t(hq), nk, head_dim);
}

}  // namespace
}  // namespace cbk

extern "C" {

size_t cbk_prompt_attention_workspace_bytes(int64_t total_q, int64_t total_k, int64_t batch, int64_t hq, int64_t hkv,
                                            int64_t head_dim, int32_t dtype) {
  using namespace cbk;
  if (check_sizes(total_q, total_k, batch, hq, hkv, head_dim, dtype) || total_q == 0 || batch == 0) return 0;
  return attn_parts_bytes(splits_of(total_q, total_k, batch, hq, hkv, head_dim, dtype), uint64_t(total_q) * uint64_t(hq),
                          head_dim);
}

int cbk_prompt_attention(const void* q_dev, int64_t q_token_stride, int64_t q_head_stride, const void* k_dev,
                         int64_t k_token_stride, int64_t k_head_stride, const void* v_dev, int64_t v_token_stride,
                         int64_t v_head_stride, const int32_t* ends_q_dev, const int32_t* ends_k_dev, int64_t batch,
                         int64_t total_q, int64_t total_k, int64_t hq, int64_t hkv, int64_t head_dim, float scale,
                         int32_t dtype, void* out_dev, int64_t out_token_stride, int64_t out_head_stride,
                         int32_t zero_outside, void* workspace_dev, size_t workspace_bytes, cbk_stream_t stream) {
  using namespace cbk;
  clear_error();
  if (int rc = check_sizes(total_q, total_k, batch, hq, hkv, head_dim, dtype)) return rc;
  if (total_q == 0) return CBK_OK;
  CBK_REQUIRE(batch > 0, "queries without a sequence");
  CBK_REQUIRE(q_dev && out_dev && ends_q_dev && ends_k_dev && (total_k == 0 || (k_dev && v_dev)), "NULL pointer");
  CBK_REQUIRE(std::isfinite(scale), "scale must be finite");
  const int64_t es = dtype == CBK_DTYPE_F32 ? 4 : 2;
  const int64_t align[12] = {q_token_stride * es, q_head_stride * es, k_token_stride * es, k_head_stride * es,
                             v_token_stride * es, v_head_stride * es, out_token_stride * es, out_head_stride * es,
                             int64_t(reinterpret_cast<uintptr_t>(q_dev)), int64_t(reinterpret_cast<uintptr_t>(k_dev)),
                             int64_t(reinterpret_cast<uintptr_t>(v_dev)), int64_t(reinterpret_cast<uintptr_t>(out_dev))};
  CBK_REQUIRE(common_vec_bytes(align, 12) == 16, "q/k/v/out pointers and strides must be 16-byte aligned");
  // the requests' per-lane 32-bit byte offsets span a 32-key block
  CBK_REQUIRE(k_token_stride >= 0 && k_token_stride < (int64_t(1) << 24) && v_token_stride >= 0 &&
                  v_token_stride < (int64_t(1) << 24),
              "K/V token strides must stay below 2^24 elements");
  PromptArgs a;
  a.q = q_dev;
  a.k = k_dev;
  a.v = v_dev;
  a.out = out_dev;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k_token = k_token_stride;
  a.k_head = k_head_stride;
  a.v_token = v_token_stride;
  a.v_head = v_head_stride;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.ends_q = ends_q_dev;
  a.ends_k = ends_k_dev;
  a.batch = uint32_t(batch);
  a.total_q = uint32_t(total_q);
  a.total_k = uint32_t(total_k);
  a.element = uint32_t(es);
  a.hq = uint32_t(hq);
  a.hkv = uint32_t(hkv);
  a.group = uint32_t(hq / hkv);
  a.group_div = FastDiv::make(a.group);
  a.scale = scale;
  a.zero_outside = zero_outside != 0;
  // without a workspace one range: every tile's keys in one workgroup
  uint32_t splits = 1;
  const uint64_t rows = uint64_t(total_q) * uint64_t(hq);
  if (workspace_dev != nullptr) {
    splits = splits_of(total_q, total_k, batch, hq, hkv, head_dim, dtype);
    const size_t need = attn_parts_bytes(splits, rows, head_dim);
    if (workspace_bytes < need)
      return set_error(CBK_ERR_WORKSPACE, "prompt attention workspace %zu < %zu bytes", workspace_bytes, need);
    CBK_REQUIRE((reinterpret_cast<uintptr_t>(workspace_dev) & 255) == 0, "workspace must be 256-byte aligned");
  }
  a.parts = attn_parts(splits, rows, workspace_dev);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc;
  switch (dtype) {
    case CBK_DTYPE_F32: rc = launch_prompt_f32(a, uint32_t(head_dim), s); break;
    case CBK_DTYPE_BF16: rc = launch_16<false>(a, uint32_t(head_dim), s); break;
    default: rc = launch_16<true>(a, uint32_t(head_dim), s);
  }
  if (rc || splits == 1) return rc;
  const AttnSpan span{ends_q_dev, uint32_t(batch), a.zero_outside};
  return launch_attn_merge(a.parts, a.total_q, a.hq, uint32_t(head_dim), nullptr, out_dev, out_token_stride, dtype, false,
                           s, out_head_stride, span);
}

}  // extern "C"
