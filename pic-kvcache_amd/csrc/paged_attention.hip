// The plan and entry points of paged_attention.hpp, and its bf16 kernels.
#include <algorithm>
#include <cmath>

#include "paged_attention.hpp"

namespace cbk {

int launch_paged_attention_bf16(const PagedAttnArgs& a, int64_t head_dim, hipStream_t s) {
  return launch_type<CBK_DTYPE_BF16>(a, head_dim, s);
}

namespace {

// All rules go by what the block tables have room for, which the host knows, not by the
// lengths, which it does not read (64 sequences of up to 1 K, tables of 128 K: 42.3 us, 41.4 with tables of
// their own, weighed 66.5 and 51.4; 24 of 8 K 87.2 and 86.8, 109 and 103).
//
// Sequences stay whole where that gives a wave few more tiles than equal ranges (a merge
// is as long as two or three), and few altogether (they may differ in length, and the
// longest counts). us a call, ranges / whole, bf16, 32 heads over 8 x 128: 1 sequence of
// 600 12.6 / 12.0, of 1000 (weights summed, 4 tiles instead of 1) 15.6 / 21.0; 64 of 256 to 1024
// 38.5 / 35.9; 256 of 128 to 512 88 / 77; 64 of 4 K to 16 K (512 tiles both) 451 / 534.
constexpr int64_t kMergeTiles = 2, kWholeTiles = 16;

// A sequence in more ranges than this: more waves for a head and fewer heads for a workgroup
// (neighbouring heads' rows are then not read at the same time, but there is less to merge). us
// a call with 8 / 4 / 2 / 1 heads, 32 heads over 8 x 128 and 256 ranges with 8 of them: 1
// sequence of 3000 14.8 / 15.1 / 13.8 / 13.6, of 8 K 17.9 / 16.8 / 15.3 / 14.8, of 32 K 31.7 / 31.0 /
// 29.8 / 29.9, of 128 K 102 / 101 / 101 / 106; 8 of 4 K 23.2 / 25.7 / 24.9 / 25.4; 64 of 16 K 394 /
// 392 / 410 / 459.
constexpr int64_t kMostRanges = 64;

// Pages of more bytes than this in the tables (twice the last cache level) are read past the caches; of
// what fits there a part may be found again. us a call, kept / past, bf16, 32 heads over
// 8 x 128: up to 67 MB (1 x 32 K) 24.6 / 25.1, 168 (64 x 1 K) 35.6 / 43.9, 460 (24 x 8 K)
// 91 / 81, 2600 (64 x 16 K) 445 / 397.
constexpr int64_t kStreamBytes = int64_t(512) << 20;

// Key weights by a second product instead of by logits in scratch: in 16 bits (float32's
// products take longer), from so many rows of a KV head and of a set on, where workgroups of 64
// keys of a set fill three quarters of the CUs. us a call, logits / second product, bf16, 128,
// 32 heads over 8, one set: 1 prompt of 4 K, 32 rows, 38 / 43, of 8 K 43.7 / 46.7, of 16 K 62.8 /
// 56.1; 24 of 2 K to 8 K 385 / 325, 16 rows 223 / 237; a set for each KV head (128 rows) 8 of
// 2 K to 8 K, 32 rows, 138 / 168.
constexpr int64_t kWindowRows = 128, kWindowSetRows = 512;

struct Plan {
  uint32_t rt, row_tiles, ranges, heads, turns, max_tiles;
  bool whole;
  size_t ml, o, stats, logits;  // bytes of the scratch's parts
  size_t bytes() const { return ml + o + stats + logits; }
};

size_t padded(size_t n) { return (n + 255) & ~size_t(255); }

int plan_of(int64_t batch, int64_t rows, int64_t hq, int64_t hkv, int64_t d, int64_t max_len, int32_t dtype, int64_t sets,
            Plan* p) {
  CBK_REQUIRE(batch >= 0 && batch < (1 << 16), "batch out of range");
  CBK_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "query heads must be divisible by KV heads");
  CBK_REQUIRE(rows > 0 && hq < (1 << 16) && rows < (1 << 16) && rows * hq < (int64_t(1) << 31), "rows or heads out of range");
  CBK_REQUIRE(max_len >= 0 && max_len < (int64_t(1) << 31) - 32, "context out of range");
  const int64_t n = rows * (hq / hkv), keys = dtype == CBK_DTYPE_F32 ? 16 : 32;
  // (two row tiles a wave take the registers of two waves: half as many read at a time, but
  // each tile once for both: 32 sequences of up to 8 K, 5 rows of 32 heads over 8, 112 us, one
  // row tile a wave 142; 9 of 3 K, 4 rows of 40 over 8, 24.3 and 25.4; four spill)
  p->rt = n <= 16 ? 1 : 2;
  p->row_tiles = uint32_t((n + 16 * p->rt - 1) / (16 * p->rt));
  const uint32_t waves = uint32_t(max_waves(int(p->rt)));
  for (p->heads = waves; hkv % p->heads != 0;) --p->heads;
  int cus = 0;
  if (int rc = device_cus(&cus)) return rc;
  p->max_tiles = uint32_t((max_len + keys - 1) / keys);
  const int64_t most = batch * int64_t(p->max_tiles);
  CBK_REQUIRE(most + batch * int64_t(kHead) < (int64_t(1) << 31), "context tiles out of range");
  // Short sequences: a range each, no second launch, the waves of a workgroup
  // taking a head's tiles in turns while that leaves no CU two workgroups.
  uint32_t heads = p->heads;
  for (uint32_t h = p->heads; h > 0; --h)
    if (hkv % h == 0 && batch * (hkv / h) * int64_t(p->row_tiles) <= cus) heads = h;
  const int64_t groups = batch * (hkv / heads) * int64_t(p->row_tiles), turns = waves / heads;
  const int64_t alone = (p->max_tiles + turns - 1) / turns * ((groups + cus - 1) / cus);  // a wave's tiles
  const int64_t cut = (most * hkv * p->row_tiles + int64_t(cus) * waves - 1) / (int64_t(cus) * waves);
  p->whole = alone <= std::min(cut + kMergeTiles, kWholeTiles);
  if (p->whole) {
    p->heads = heads;
    p->turns = uint32_t(turns);
    p->ranges = uint32_t(std::max<int64_t>(batch, 1));
  } else {
    // a workgroup of each CU (registers); fewer where its waves would have less
    // than a tile each
    for (;;) {
      p->turns = waves / p->heads;
      const int64_t units = hkv / p->heads * int64_t(p->row_tiles);
      const int64_t ranges = std::min((int64_t(cus) + units - 1) / units, (most + p->turns - 1) / p->turns);
      p->ranges = uint32_t(ranges > 1 ? ranges : 1);
      if (p->heads == 1 || ranges <= kMostRanges * batch) break;
      for (--p->heads; hkv % p->heads != 0;) --p->heads;
    }
  }
  const size_t all_rows = size_t(rows) * size_t(hq);
  const bool logits = sets > 0 && (dtype == CBK_DTYPE_F32 || n < kWindowRows || rows * hq / sets < kWindowSetRows ||
                                   batch * sets * (max_len / kWindowKeys) < cus - cus / 4);
  CBK_REQUIRE(!logits || size_t(most) * size_t(keys) <= (size_t(1) << 44) / all_rows, "logits of %zu rows and %lld tiles are too many",
              all_rows, (long long)most);
  const size_t parts = p->whole ? 0 : size_t(2) * p->ranges * all_rows;
  p->ml = padded(parts * sizeof(float2));
  p->o = padded(parts * size_t(d) * sizeof(float));
  p->stats = sets > 0 ? padded(size_t(batch) * all_rows * sizeof(float2)) : 0;
  p->logits = logits ? padded(size_t(most) * size_t(keys) * all_rows * sizeof(float)) : 0;
  return CBK_OK;
}

}  // namespace
}  // namespace cbk

extern "C" {

size_t cbk_paged_attention_workspace_bytes(int64_t batch, int64_t rows, int64_t hq, int64_t hkv, int64_t head_dim,
                                           int64_t max_len, int32_t dtype, int64_t weight_sets) {
  using namespace cbk;
  Plan p;
  if (batch <= 0 || head_dim <= 0 || plan_of(batch, rows, hq, hkv, head_dim, max_len, dtype, weight_sets, &p)) return 0;
  return p.bytes();
}

int cbk_paged_attention(const void* q_dev, int64_t q_batch_stride, int64_t q_row_stride, int64_t q_head_stride,
                        int64_t batch, int64_t rows, int64_t hq, const cbk_kv_desc* kv, int64_t hkv, int64_t head_dim,
                        const int32_t* tables_dev, int64_t table_stride, int64_t table_width, const int32_t* lens_dev,
                        float scale, int32_t dtype, void* out_dev, int64_t out_batch_stride, int64_t out_row_stride,
                        int64_t out_head_stride, float* key_weights_dev, int64_t weights_batch_stride,
                        int64_t weights_set_stride, int64_t weight_sets, void* workspace_dev, size_t workspace_bytes,
                        cbk_stream_t stream) {
  using namespace cbk;
  clear_error();
  if (int rc = validate_desc(kv)) return rc;
  CBK_REQUIRE(dtype == CBK_DTYPE_F32 || dtype == CBK_DTYPE_BF16 || dtype == CBK_DTYPE_F16, "dtype %d", int(dtype));
  CBK_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim %lld: 64 or 128 supported", (long long)head_dim);
  const int64_t es = dtype == CBK_DTYPE_F32 ? 4 : 2;
  CBK_REQUIRE(hkv > 0 && kv->row_bytes == hkv * head_dim * es, "a row of %lld x %lld is not %lld bytes", (long long)hkv,
              (long long)head_dim, (long long)kv->row_bytes);
  CBK_REQUIRE(std::isfinite(scale), "scale must be finite");
  CBK_REQUIRE(table_width >= 0 && table_width < (int64_t(1) << 31) && table_stride >= 0,
              "block table width out of range");
  CBK_REQUIRE(kv->num_blocks < (int64_t(1) << 31), "num_blocks out of range");
  CBK_REQUIRE(key_weights_dev == nullptr || weight_sets == 1 || weight_sets == hkv, "%lld sets of weights for %lld KV heads",
              (long long)weight_sets, (long long)hkv);
  CBK_REQUIRE(batch == 0 || q_dev != out_dev ||
                  ((batch == 1 || q_batch_stride == out_batch_stride) && (rows == 1 || q_row_stride == out_row_stride) &&
                   (hq == 1 || q_head_stride == out_head_stride)),
              "outputs in the queries' place need their strides");
  const int64_t max_len = table_width * kv->block_size;
  Plan p;
  if (int rc = plan_of(batch, rows, hq, hkv, head_dim, max_len, dtype, key_weights_dev ? weight_sets : 0, &p)) return rc;
  if (batch == 0) return CBK_OK;
  CBK_REQUIRE(q_dev && out_dev && lens_dev && (tables_dev || table_width == 0), "NULL pointer");
  const int64_t words[6] = {int64_t(reinterpret_cast<uintptr_t>(kv->k_base)),
                            int64_t(reinterpret_cast<uintptr_t>(kv->v_base)), kv->block_stride, kv->token_stride,
                            int64_t(reinterpret_cast<uintptr_t>(q_dev)), int64_t(reinterpret_cast<uintptr_t>(out_dev))};
  CBK_REQUIRE(common_vec_bytes(words, 6) >= es, "tensors must be aligned to their elements");
  if (p.bytes() > 0 && (workspace_dev == nullptr || workspace_bytes < p.bytes()))
    return set_error(CBK_ERR_WORKSPACE, "paged attention workspace %zu < %zu bytes", workspace_bytes, p.bytes());
  CBK_REQUIRE((reinterpret_cast<uintptr_t>(workspace_dev) & 255) == 0, "workspace must be 256-byte aligned");
  // (a second product reads the queries after the outputs are written)
  CBK_REQUIRE(!key_weights_dev || p.logits > 0 || max_len == 0 || q_dev != out_dev,
              "key weights of these sizes take the queries again: outputs cannot be in their place");
  PagedAttnArgs a;
  a.q = static_cast<const char*>(q_dev);
  a.out = static_cast<char*>(out_dev);
  a.q_batch = q_batch_stride * es;
  a.q_row = q_row_stride * es;
  a.q_head = q_head_stride * es;
  a.out_batch = out_batch_stride * es;
  a.out_row = out_row_stride * es;
  a.out_head = out_head_stride * es;
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
  a.max_tiles = p.max_tiles;
  a.row_tiles = p.row_tiles;
  a.ranges = p.ranges;
  a.rt = p.rt;
  a.stream = p.row_tiles == 1 && batch * max_len * 2 * kv->row_bytes > kStreamBytes;
  a.weights = key_weights_dev;
  a.w_batch = weights_batch_stride;
  a.w_set = weights_set_stride;
  a.w_sets = uint32_t(weight_sets);
  a.whole = p.whole;
  a.fast = kv->block_size % 16 == 0 && common_vec_bytes(words, 4) == 16 && kv->token_stride < (int64_t(1) << 26);
  a.heads = p.heads;
  a.turns = p.turns;
  a.c = scale * (kLog2e / kUnit);
  a.block_div = FastDiv::make(uint32_t(kv->block_size));
  char* at = static_cast<char*>(workspace_dev);
  a.ml = reinterpret_cast<float2*>(at);
  a.o = reinterpret_cast<float*>(at += p.ml);
  a.stats = p.stats ? reinterpret_cast<float2*>(at + p.o) : nullptr;
  a.logits = p.logits ? reinterpret_cast<float*>(at + p.o + p.stats) : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case CBK_DTYPE_F32: return launch_paged_attention_f32(a, head_dim, s);
    case CBK_DTYPE_BF16: return launch_paged_attention_bf16(a, head_dim, s);
    default: return launch_paged_attention_f16(a, head_dim, s);
  }
}

}  // extern "C"
