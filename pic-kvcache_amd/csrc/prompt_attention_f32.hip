// float32 attention of packed prompts for gfx950 (prompt_attention.hip): the
// products on the bf16 matrix cores.
//
// A float32 value is three bf16, rounded one after another (8 + 8 + 8 bits
// hold all 24), and a product of two such values six of the nine products of
// their parts; the three left out are below 2^-24 of it. Six
// v_mfma_f32_16x16x32_bf16 take 96 cycles a wave where the float32
// instructions, eight v_mfma_f32_16x16x4_f32, take 256.
//
// One workgroup (4 waves of 16 or 32 rows, prompt_f32_rows) per 64 or 128 rows
// of (query, group head) of one sequence, key range and KV head. The next 32-key
// block's rows are loaded into registers while a block is computed, then cut
// into parts and stored to LDS, in the layout of the 16-bit kernels, three times.
// S^T = K . Q^T, online softmax and O += P . V as there, P cut like the inputs.
// Three workgroups of 64 rows per CU (48 KiB of LDS each; two of 128 at head_dim
// 128, which take the registers) take turns at the matrix cores, the VALU and
// the LDS, each busy for a third to two thirds of the time: 8000 tokens of 32 / 8
// heads x 128 2.51 ms, 209 TFLOP/s, 1.25 PFLOP/s of bf16 products.
//
// Rows with a term that is not finite are computed again one by one, over
// their visible keys only: the blocks multiply a masked key's probability of
// zero with its value row, which may hold anything.
#include <cmath>

#include "attention_mfma.hpp"
#include "prompt_attention.hpp"

namespace cbk {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kKeys = kAttnKeyBlock;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

using O16 = Ops<false>;

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Two floats as three words of bf16 pairs.
__device__ __forceinline__ void cut(float x, float y, uint32_t (&w)[3]) {
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    w[p] = O16::pack(x, y);
    x -= O16::lo(w[p]);
    y -= O16::hi(w[p]);
  }
}

// acc += a . b, the parts' products from the smallest on
__device__ __forceinline__ f32x4 mma6(const s16x8 (&a)[3], const s16x8 (&b)[3], f32x4 acc) {
  acc = O16::mma32(a[2], b[0], acc);
  acc = O16::mma32(a[0], b[2], acc);
  acc = O16::mma32(a[1], b[1], acc);
  acc = O16::mma32(a[1], b[0], acc);
  acc = O16::mma32(a[0], b[1], acc);
  return O16::mma32(a[0], b[0], acc);
}

// One row's keys [lo, hi] by the whole wave: every lane two dims. The sum l
// and the maximum m (natural units) of the keys, o the lane's outputs.
template <int D>
__device__ void attend_row(const float* q, const float* k, const float* v, int64_t k_token, int64_t v_token, float scale,
                           int32_t lo, int32_t hi, uint32_t lane, float& m, float& l, float& o0, float& o1) {
#pragma clang fp contract(off)  // x - ms of two rounded logits: 0 for equal ones, however large
  const float q0 = q[lane], q1 = D > 64 ? q[lane + 64] : 0.f;
  m = kNegInf;
  l = o0 = o1 = 0.f;
  for (int32_t j = lo; j <= hi; ++j) {
    const float* kr = k + int64_t(j) * k_token;
    const float* vr = v + int64_t(j) * v_token;
    float dot = q0 * kr[lane] + (D > 64 ? q1 * kr[lane + 64] : 0.f);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) dot += __shfl_xor(dot, off);
    const float x = dot * scale;
    const float mn = fmaxf(m, x);
    const float ms = mn == kNegInf ? 0.f : mn;
    const float alpha = expf(m - ms);
    const float p = expf(x - ms);
    l = l * alpha + p;
    o0 = o0 * alpha + p * vr[lane];
    o1 = o1 * alpha + p * (D > 64 ? vr[lane + 64] : 0.f);
    m = mn;
    if (l != l) {  // NaN from here on in every lane (uniform): a bad key that many rows see early
      o0 = o1 = l;
      return;
    }
  }
}

constexpr int waves_per_simd(int d, int row_tiles) { return d == 64 || row_tiles == 1 ? 3 : 2; }

// RT: 16-row tiles of a wave.
template <int D, int RT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(waves_per_simd(D, RT), waves_per_simd(D, RT)))) void prompt_f32_kernel(const PromptArgs a) {
  constexpr uint32_t kRows = 16 * RT * kWaves;
  constexpr uint32_t P4 = D / 4;             // 16-byte pieces of a row
  constexpr int N = kKeys * int(P4) / kThreads;  // pieces per thread and block, each of K and V
  constexpr uint32_t kStep = kThreads / P4;  // rows the workgroup loads at a time
  constexpr uint32_t kPart = kKeys * D;      // elements of a block's part
  __shared__ __attribute__((aligned(16))) uint16_t kbuf[3 * kPart], vbuf[3 * kPart];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row = lane & 15, grp = lane >> 4;
  const uint32_t S = a.parts.splits;
  const uint32_t kvh = __builtin_amdgcn_readfirstlane(blockIdx.x % a.hkv);
  const uint32_t rest = __builtin_amdgcn_readfirstlane(blockIdx.x / a.hkv);
  const uint32_t rank = __builtin_amdgcn_readfirstlane(rest / S);
  const uint32_t split = rest - rank * S;
  const PromptTile tl = prompt_tile<kRows>(a, rank, lane);
  if (tl.beyond) {
    if (S == 1) prompt_outside(a, tl, kvh, D * 4);
    return;
  }
  if (tl.none) return;
  const uint32_t nrows = tl.nq * a.group;
  const uint32_t r0 = tl.tile * kRows + wave * 16 * RT;  // the wave's first row
  const int32_t shift = int32_t(tl.nk) - int32_t(tl.nq);  // a query's position minus its index
  const float* k_seq = static_cast<const float*>(a.k) + int64_t(tl.k0) * a.k_token + int64_t(kvh) * a.k_head;
  const float* v_seq = static_cast<const float*>(a.v) + int64_t(tl.k0) * a.v_token + int64_t(kvh) * a.v_head;

  int32_t rpos[RT];
  s16x8 qf[RT][D / 32][3];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const uint32_t r = r0 + 16 * t + row;
    const bool valid = r < nrows;
    const uint32_t qi = valid ? a.group_div.div(r) : 0, qh = kvh * a.group + (valid ? r - qi * a.group : 0);
    rpos[t] = valid ? int32_t(qi) + shift : -1;
    const float* q_row = static_cast<const float*>(a.q) + int64_t(tl.q0 + qi) * a.q_token + int64_t(qh) * a.q_head;
#pragma unroll
    for (int st = 0; st < D / 32; ++st) {
      u32x4 w[3] = {u32x4(0u), u32x4(0u), u32x4(0u)};
      if (valid) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(q_row + 32 * st + 8 * grp + 4 * h);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t c[3];
            cut(x[2 * i], x[2 * i + 1], c);
#pragma unroll
            for (int p = 0; p < 3; ++p) w[p][2 * h + i] = c[p];
          }
        }
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) qf[t][st][p] = __builtin_bit_cast(s16x8, w[p]);
    }
  }
  // the wave's earliest and latest positions; the workgroup's blocks: its
  // share of the tile's
  const int32_t wmax = r0 < nrows ? int32_t(a.group_div.div(min(nrows, r0 + 16 * RT) - 1)) + shift : -1;
  const int32_t wmin = r0 < nrows ? int32_t(a.group_div.div(r0)) + shift : 0x7fffffff;
  const int32_t gmax = int32_t(a.group_div.div(min(nrows, (tl.tile + 1) * kRows) - 1)) + shift;
  const uint32_t nblocks = gmax < 0 ? 0u : uint32_t(gmax) / kKeys + 1;
  const int32_t b_lo = __builtin_amdgcn_readfirstlane(int32_t(nblocks * split / S));
  const int32_t b_hi = __builtin_amdgcn_readfirstlane(int32_t(nblocks * (split + 1) / S));

  const uint32_t lr = threadIdx.x / P4, lp = threadIdx.x % P4;
  f32x4 kreg[N], vreg[N];
  auto load = [&](int32_t b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int32_t key = b * kKeys + int32_t(lr + kStep * i);
      kreg[i] = vreg[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (key < int32_t(tl.nk)) {
        kreg[i] = *reinterpret_cast<const f32x4*>(k_seq + int64_t(key) * a.k_token + 4 * lp);
        vreg[i] = *reinterpret_cast<const f32x4*>(v_seq + int64_t(key) * a.v_token + 4 * lp);
      }
    }
  };
  auto store = [&](uint16_t* buf, const f32x4 (&reg)[N]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t key = lr + kStep * i;
      uint32_t c0[3], c1[3];
      cut(reg[i][0], reg[i][1], c0);
      cut(reg[i][2], reg[i][3], c1);
#pragma unroll
      for (int p = 0; p < 3; ++p)
        *reinterpret_cast<u32x2*>(buf + p * kPart + key * D + ((lp / 2) ^ lds_swizzle<D>(key)) * 8 + (lp & 1) * 4) =
            u32x2{c0[p], c1[p]};
    }
  };
  const BlockOffsets<D> off(lane);
  f32x4 o[RT][D / 16];
  float m[RT], l[RT];  // log2 units; l of this lane's keys only
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = kNegInf;
    l[t] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float c2 = a.scale * kLog2e;
  if (b_lo < b_hi) load(b_lo);
  for (int32_t b = b_lo; b < b_hi; ++b) {
    __syncthreads();  // every wave is done with the block before
    store(kbuf, kreg);
    store(vbuf, vreg);
    __syncthreads();
    if (b + 1 < b_hi) load(b + 1);
    if (wmax < b * kKeys) continue;  // no row of the wave sees the block
    f32x4 s[RT][2];
    const char* kp = reinterpret_cast<const char*>(kbuf);
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s16x8 kf[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) kf[p] = *reinterpret_cast<const s16x8*>(kp + off.k[st] + h * (16 * D * 2) + p * (kPart * 2));
#pragma unroll
        for (int t = 0; t < RT; ++t) s[t][h] = mma6(kf, qf[t][st], st == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : s[t][h]);
      }
    s16x8 pf[RT][3];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float bm = kNegInf;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[t][h][i] * c2;
          if (wmin < b * kKeys + kKeys - 1 && b * kKeys + 16 * h + int32_t(4 * grp) + i > rpos[t]) x = kNegInf;
          s[t][h][i] = x;
          bm = fmaxf(bm, x);
        }
      bm = fmaxf(bm, __shfl_xor(bm, 16));
      bm = fmaxf(bm, __shfl_xor(bm, 32));
      if (__any(bm > m[t])) {  // some row's maximum rose
        const float mn = fmaxf(m[t], bm);
        const float alpha = mn == m[t] ? 1.f : __builtin_amdgcn_exp2f(m[t] - mn);
        m[t] = mn;
        l[t] *= alpha;
        float ao[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ao[i] = __shfl(alpha, int(4 * grp + i));
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][c][i] *= ao[i];
      }
      const float ms = m[t] == kNegInf ? 0.f : m[t];
      // the two halves' S^T registers, concatenated, are P's operand
      u32x4 w[3];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(s[t][h][i] - ms);
        l[t] += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t c[3];
          cut(p[2 * i], p[2 * i + 1], c);
#pragma unroll
          for (int n = 0; n < 3; ++n) w[n][2 * h + i] = c[n];
        }
      }
#pragma unroll
      for (int n = 0; n < 3; ++n) pf[t][n] = __builtin_bit_cast(s16x8, w[n]);
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      typedef short s16x4v __attribute__((ext_vector_type(4)));
      s16x8 vf[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        s16x4v w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4v*)((__attribute__((address_space(3))) const void*)(
                  reinterpret_cast<const char*>(vbuf) + off.v[c] + h * (16 * D * 2) + p * (kPart * 2))));
        vf[p] = __builtin_shufflevector(w[0], w[1], 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) o[t][c] = mma6(pf[t], vf, o[t][c]);
    }
  }

  // the wave's rows with a term that is not finite, or with keys but no sum
  // (logits that are finite by themselves, -inf times log2 e): redone below
  uint32_t bad = 0;  // bit 16 t + row
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l[t] += __shfl_xor(l[t], 16);
    l[t] += __shfl_xor(l[t], 32);
    const uint64_t lb = __ballot(!finite_bits(l[t]) || (l[t] == 0.f && b_lo < b_hi && rpos[t] >= b_lo * kKeys));
    uint32_t here = uint32_t((lb | (lb >> 16) | (lb >> 32) | (lb >> 48)) & 0xffffu);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bool f = true;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) f = f && finite_bits(o[t][c][i]);
      const uint64_t ob = __ballot(!f);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if ((ob >> (16 * g)) & 0xffffu) here |= 1u << (4 * g + i);
    }
    // lanes 0..15 hold rows 0..15
    bad |= (here & uint32_t(__ballot(r0 + 16 * t + row < nrows)) & 0xffffu) << (16 * t);
  }
  const uint64_t rows_all = uint64_t(a.total_q) * a.hq;
  // where row rr's results go: the output, or the range's partial results
  auto place = [&](uint32_t rr, uint64_t& id) __attribute__((always_inline)) {
    const uint32_t gr = r0 + rr, oq = a.group_div.div(gr), oh = kvh * a.group + gr - oq * a.group;
    id = split * rows_all + uint64_t(tl.q0 + oq) * a.hq + oh;
    return S == 1 ? static_cast<float*>(a.out) + int64_t(tl.q0 + oq) * a.out_token + int64_t(oh) * a.out_head
                  : a.parts.o + id * D;
  };
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t rr = 16 * t + 4 * grp + i;
      const float rl = __shfl(l[t], int(4 * grp + i)), rm = __shfl(m[t], int(4 * grp + i));
      if (r0 + rr >= nrows || ((bad >> rr) & 1u)) continue;
      uint64_t id;
      float* dst = place(rr, id);
      const float f = S > 1 ? 1.f : rl > 0.f ? 1.f / rl : 0.f;
      if (S > 1 && row == 0) a.parts.ml[id] = make_float2(0.5f * rm, rl);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) dst[16 * c + row] = o[t][c][i] * f;
    }
  while (bad) {  // uniform
    const uint32_t rr = uint32_t(__builtin_ctz(bad));
    bad &= bad - 1;
    const uint32_t oq = a.group_div.div(r0 + rr);
    const int32_t last = min(__builtin_amdgcn_readfirstlane(int32_t(oq) + shift), b_hi * kKeys - 1);
    const uint32_t oh = kvh * a.group + r0 + rr - oq * a.group;
    const float* q = static_cast<const float*>(a.q) + int64_t(tl.q0 + oq) * a.q_token + int64_t(oh) * a.q_head;
    float fm, fl, o0, o1;
    attend_row<D>(q, k_seq, v_seq, a.k_token, a.v_token, a.scale, b_lo * kKeys, last, lane, fm, fl, o0, o1);
    uint64_t id;
    float* dst = place(rr, id);
    const float f = S > 1 ? 1.f : fl == 0.f ? 0.f : 1.f / fl;
    if (S > 1 && lane == 0) a.parts.ml[id] = make_float2(fm * (0.5f * kLog2e), fl);
    dst[lane] = o0 * f;
    if constexpr (D > 64) dst[lane + 64] = o1 * f;
  }
}

}  // namespace

int launch_prompt_f32(const PromptArgs& a, uint32_t d, hipStream_t stream) {
  const uint32_t rows = prompt_f32_rows(uint64_t(a.total_q) * a.group, a.hkv);
  const uint64_t groups = prompt_tiles(a, rows) * a.hkv * a.parts.splits;
  CBK_REQUIRE(groups * kThreads < (uint64_t(1) << 32), "prompt attention f32: %llu workgroups exceed one launch",
              (unsigned long long)groups);
  const dim3 grid(static_cast<uint32_t>(groups)), block(kThreads);
  if (rows == 128) {
    if (d == 128) hipLaunchKernelGGL((prompt_f32_kernel<128, 2>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((prompt_f32_kernel<64, 2>), grid, block, 0, stream, a);
  } else {
    if (d == 128) hipLaunchKernelGGL((prompt_f32_kernel<128, 1>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((prompt_f32_kernel<64, 1>), grid, block, 0, stream, a);
  }
  return launch_status("prompt attention f32");
}

}  // namespace cbk
