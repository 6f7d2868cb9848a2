// C ABI of the key/value cache in 4 bits: argument checks, work split, launches. Nothing here
// allocates, frees or synchronises.
#include <algorithm>
#include <cmath>

#include "gfa.h"
#include "gfa_kv4.h"
#include "gfa_launch.h"

namespace gfa {
int api_fail(int code, const char* fmt, ...);  // gfa_api.hip
int api_ok();
}  // namespace gfa

namespace {

using gfa::api_fail;

constexpr int64_t kMostWorkgroups = (1 << 24) - 1;  // of 256 threads: a launch holds fewer than 2^32

bool aligned(const void* p, unsigned n) { return p != nullptr && reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_cache(const gfa_kv4_cache& c) {
  if (!aligned(c.codes, 16) || !aligned(c.scales, 16))
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "codes and scales must be 16-byte aligned pointers");
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256 && c.head_dim != 512)
    return api_fail(GFA_ERR_UNSUPPORTED, "head_dim=%d not built (64, 128, 256, 512)", c.head_dim);
  if (c.block_size < 32 || c.block_size > 1024 || (c.block_size & (c.block_size - 1)) != 0)
    return api_fail(GFA_ERR_UNSUPPORTED, "block_size=%d must be a power of two, 32 to 1024", c.block_size);
  if (c.num_blocks < 1 || c.heads_kv < 1 || c.heads_kv > 65535)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "num_blocks=%d and heads_kv=%d must be positive", c.num_blocks, c.heads_kv);
  if (c.dtype != GFA_DTYPE_FP16 && c.dtype != GFA_DTYPE_BF16)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "dtype=%d is not a gfa_dtype", c.dtype);
  return GFA_OK;
}

gfa::Kv4Cache cache_of(const gfa_kv4_cache& c) {
  int log2 = 5;
  while ((1 << log2) < c.block_size) ++log2;
  return gfa::Kv4Cache{static_cast<uint8_t*>(c.codes), static_cast<uint8_t*>(c.scales), c.num_blocks, c.heads_kv, log2};
}

int check_rows(const char* name, const void* p, const gfa_strides& s) {
  if (!aligned(p, 16)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "%s must be a 16-byte aligned pointer", name);
  if (s.batch % 8 != 0 || s.head % 8 != 0 || s.row % 8 != 0 || s.batch < 0 || s.head < 0 || s.row < 0)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "%s strides must be non-negative multiples of 8 elements", name);
  return GFA_OK;
}

int launched(hipError_t err, const char* what) {
  if (err != hipSuccess) return api_fail(GFA_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(err));
  return gfa::api_ok();
}

int rows_call(const gfa_kv4_rows_args* a, bool write) {
  if (a == nullptr) return api_fail(GFA_ERR_INVALID_ARGUMENT, "args is NULL");
  if (int rc = check_cache(a->cache)) return rc;
  if (a->batch < 1 || a->seq_len < 1) return api_fail(GFA_ERR_INVALID_ARGUMENT, "batch=%d and seq_len=%d must be positive", a->batch, a->seq_len);
  if (int rc = check_rows("k", a->k, a->k_strides)) return rc;
  if (int rc = check_rows("v", a->v, a->v_strides)) return rc;
  if (!aligned(a->slots, 8)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "slots must be an 8-byte aligned pointer");
  const int64_t tokens = (int64_t)a->batch * a->seq_len;
  // a wave per 2048 / head_dim tokens and head, four waves a workgroup
  const int64_t per_wave = 2048 / a->cache.head_dim, waves = (tokens + per_wave - 1) / per_wave * a->cache.heads_kv;
  if (tokens > 0x7fffffff || (waves + 3) / 4 > kMostWorkgroups)
    return api_fail(GFA_ERR_UNSUPPORTED, "%lld tokens of %d heads exceed one launch", (long long)tokens, a->cache.heads_kv);
  gfa::Kv4RowsParams p{};
  p.cache = cache_of(a->cache);
  p.k = p.ko = static_cast<uint16_t*>(a->k);
  p.v = p.vo = static_cast<uint16_t*>(a->v);
  p.ksb = a->k_strides.batch;
  p.ksh = a->k_strides.head;
  p.ksn = a->k_strides.row;
  p.vsb = a->v_strides.batch;
  p.vsh = a->v_strides.head;
  p.vsn = a->v_strides.row;
  p.slots = a->slots;
  p.n.set(a->seq_len);
  p.hkv.set(a->cache.heads_kv);
  p.T = (int)tokens;
  const auto stream = static_cast<hipStream_t>(a->stream);
  const bool bf16 = a->cache.dtype == GFA_DTYPE_BF16;
  return launched(write ? gfa::launch_kv4_write(p, a->cache.head_dim, bf16, stream)
                        : gfa::launch_kv4_read(p, a->cache.head_dim, bf16, stream),
                  write ? "cache write" : "cache read");
}

// One kernel's part of an attention call. The lengths live on the device, so the host sizes the grid for any
// lengths the block tables can hold and the kernels divide what there is (gfa_kv4_sched.h).
struct Part {
  bool runs;
  int min_tiles;
  float share;
  int64_t nblocks, row_blocks, slots;
  int join_rows, join_slice, join_parts, window_tiles;
  bool join;  // some row block may take more than one chunk
  size_t part_bytes, ml_bytes;
  size_t bytes() const { return part_bytes + ml_bytes; }
};
struct Split {
  int row_limit;  // requests of more query rows (new tokens times heads of a KV head) take the chunk kernel
  bool one_block;  // as far as max_new says, no request has more than one row block
  Part few, many;
};

constexpr int kRows = gfa::kSplitRows;
// A request's rows from which the chunk kernel is faster: 16 requests at 8k, D = 512, 32 rows 101 us (chunk kernel 172),
// 64 rows 159 (176), 128 rows 261 (190); D = 128, 64 rows 97 (122), 128 rows 161 (127). Up to four requests and KV heads
// leave the GPU to the split kernel's smaller workgroups longer, 128 rows at every head dim from 1k to 16k: one request at
// 8k, D = 512, 25 us (45), D = 64 12 (29); the nearest, four requests at 8k and 16k, D = 512, 47 (52) and 60 (66).
int row_limit(const gfa_kv4_attn_args* a) { return (int64_t)a->requests * a->cache.heads_kv <= 4 ? 128 : 64; }

void size_part(Part& s, const gfa_kv4_attn_args* a, int64_t row_blocks, int rows, int64_t most_rows, int min_tiles, int target, int spare) {
  int64_t tiles = (int64_t)a->table_width * a->cache.block_size / 32;  // most tiles of a row block
  if (a->causal && a->window > 0) {
    const int64_t g = a->heads_q / a->cache.heads_kv, tokens = (rows + g - 2) / g + 1;  // a row block's, at most
    s.window_tiles = (int)std::min<int64_t>((a->window + tokens + 29) / 32 + 1, 0x40000000);
    tiles = std::min<int64_t>(tiles, s.window_tiles);
  }
  // One chunk and no join where no row block can see more than 16 tiles: tables of up to 512 tokens, windows of up to 466 (few
  // rows, one query head per KV head) to 480 (many heads). Lengths are not the host's to see, so a short request in a wide table is split and
  // joined like any other, and so is a window of 512, which can touch 18 tiles. One token of a request, one chunk against split
  // and join, us (16:16 D = 64, 32:8 D = 128, 8:1 D = 256, 8:1 D = 512; the same from 512-token and 16k-token tables):
  //   512 tokens  5.7 7.7, 7.0 8.8, 9.5 10.6, 14.9 15.6    768  6.9 8.1, 8.5 8.9, 11.6 10.9, 18.4 15.2
  //   1024        8.0 8.2, 9.9 9.0, 13.8 10.9, 21.9 15.2   window 512 of 16k  5.7 7.8, 7.0 8.8, 9.4 10.7, 15.0 15.2
  const int64_t chunks = tiles <= 16 ? 1 : (tiles + min_tiles - 1) / min_tiles;
  s.runs = row_blocks > 0;
  s.join = chunks > 1;
  s.min_tiles = s.join ? min_tiles : 0x3fffffff;
  s.row_blocks = row_blocks;
  // The join. Of the chunk kernel: its runs of 1 KB, four waves a workgroup. Of the split kernel: where rows are few, a
  // workgroup takes one row of 128 channels and its lanes share the chunks; else whole rows, where they are many
  // one per group of lanes.
  const int64_t hkv = a->cache.heads_kv, row_bound = std::min<int64_t>(rows, most_rows), n = row_blocks * hkv * row_bound;
  const int D = a->cache.head_dim;
  s.join_slice = rows == kRows && D > 128 && n * (D / 128) <= 1024 ? 128 : D;
  const int groups = 1024 / s.join_slice;
  s.join_parts = n <= 2048 ? groups : 1;
  const int64_t wgs = rows == kRows ? (row_bound * s.join_parts + groups - 1) / groups : rows / 32 * (D <= 128 ? 16 : D / 8) / 4;
  const int64_t most_wgs = 4096 / std::max<int64_t>(1, row_blocks * hkv);
  s.join_rows = (int)std::max<int64_t>(1, std::min(wgs, most_wgs));
  s.share = (float)((double)hkv / target * (1.0 + 1.0 / 4096));  // see chunk_tiles
  const int64_t items = std::min(row_blocks * chunks, row_blocks + (target + hkv - 1) / hkv);
  s.nblocks = items * hkv + spare;
  if (s.join) {
    s.slots = std::min(row_blocks * chunks, 2 * target / hkv + 1);
    s.part_bytes = (size_t)(s.slots * hkv) * rows * a->cache.head_dim * sizeof(float);
    s.ml_bytes = (size_t)(s.slots * hkv) * rows * 2 * sizeof(float);
  }
}

Split split_of(const gfa_kv4_attn_args* a) {
  Split s{};
  const int64_t G = a->heads_q / a->cache.heads_kv, R = a->requests;
  const int64_t T = (int64_t)a->batch * a->seq_len;
  const int64_t most = a->cu == nullptr ? T / R : a->max_new > 0 ? std::min<int64_t>(a->max_new, T) : T;
  // No request can have more rows than the limit: then all are the split kernel's, whatever max_new promised.
  s.one_block = most * G <= kRows;
  const int limit = row_limit(a);
  s.row_limit = most * G <= limit ? 0x7fffffff : limit;
  const int D = a->cache.head_dim, big = gfa::kv4_chunk_rows(D);
  int64_t few, many = 0;
  if (a->cu == nullptr) {
    const bool large = most * G > s.row_limit;
    few = large ? 0 : R * ((most * G + kRows - 1) / kRows);
    many = large ? R * ((most * G + big - 1) / big) : 0;
  } else {
    few = (T * G + (kRows - 1) * R) / kRows;
    if (s.row_limit == limit) {
      few = std::min<int64_t>(few, R * ((limit + kRows - 1) / kRows));
      many = T * G / big + std::min<int64_t>(R, T * G / (limit + 1));
    }
  }
  // with cu, workgroups to spare: rows behind the last request's
  // Chunks of at least 8 tiles, two a wave (16k keys, D = 512: 19.7 us; of 4: 21.0, of 2: 26.2). Twice the CUs' number
  // of workgroups where there is work for them (32 ragged requests: 512 96 us, 1024 107 us, 2048 129 us; 64 full
  // ones 152-154 us with each).
  size_part(s.few, a, few, kRows, most * G, 8, 512, a->cu ? 64 : 0);
  // Of the chunk kernel as many workgroups as the CUs hold at once (256 tokens at 16k, D = 512: 290 us, twice as many 314;
  // 1024 tokens, D = 128: 256 482 us, 512 375, 768 354, 1024 360). Its chunks cost as much again as some tiles, so the
  // more of the GPU the row blocks take by themselves the longer a chunk has to be: 256 tokens of one request, window
  // 1024, 33 us with chunks of 8 tiles, 57 unsplit; 1000 tokens beside seven requests 66 us with 18 tiles, 74 unsplit;
  // 512 tokens of four requests 76-84 us split, 71 unsplit.
  const int64_t alone = many * a->cache.heads_kv;
  size_part(s.many, a, many, big, most * G, alone >= 256 ? 64 : alone >= 128 ? 32 : 8, 256 * gfa::kv4_chunk_wgs(D), 0);
  return s;
}

int check_attn(const gfa_kv4_attn_args* a) {
  if (a == nullptr) return api_fail(GFA_ERR_INVALID_ARGUMENT, "args is NULL");
  if (int rc = check_cache(a->cache)) return rc;
  if (a->batch < 1 || a->seq_len < 1 || a->requests < 1 || a->table_width < 1)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "batch=%d, seq_len=%d, requests=%d and table_width=%d must be positive", a->batch,
                    a->seq_len, a->requests, a->table_width);
  if (a->requests > 65536) return api_fail(GFA_ERR_UNSUPPORTED, "%d requests (most 65536)", a->requests);
  if (a->heads_q < 1 || a->heads_q % a->cache.heads_kv != 0)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "heads_q=%d must be a multiple of heads_kv=%d", a->heads_q, a->cache.heads_kv);
  const int64_t T = (int64_t)a->batch * a->seq_len;
  if (T * a->heads_q > 0x7fffffff) return api_fail(GFA_ERR_UNSUPPORTED, "%lld query rows exceed one launch", (long long)(T * a->heads_q));
  if ((int64_t)a->table_width * a->cache.block_size > 0x40000000)
    return api_fail(GFA_ERR_UNSUPPORTED, "block tables of %lld tokens (most 2^30)", (long long)a->table_width * a->cache.block_size);
  if (a->cu == nullptr && T % a->requests != 0)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "%lld tokens do not divide among %d requests (pass cu)", (long long)T, a->requests);
  if (!std::isfinite(a->scale) || a->scale <= 0.f) return api_fail(GFA_ERR_INVALID_ARGUMENT, "scale=%g must be finite and > 0", (double)a->scale);
  if (!std::isfinite(a->softcap) || a->softcap < 0.f)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "softcap=%g must be finite and >= 0 (0 = off)", (double)a->softcap);
  if (a->window < 0 || a->max_new < 0) return api_fail(GFA_ERR_INVALID_ARGUMENT, "window=%d and max_new=%d must be >= 0", a->window, a->max_new);
  if (a->table_stride < a->table_width && a->requests > 1)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "table_stride=%lld below table_width=%d", (long long)a->table_stride, a->table_width);
  return GFA_OK;
}

}  // namespace

extern "C" {

int gfa_kv4_write(const gfa_kv4_rows_args* args) { return rows_call(args, true); }
int gfa_kv4_read(const gfa_kv4_rows_args* args) { return rows_call(args, false); }

int gfa_kv4_plan(const gfa_kv4_plan_args* a) {
  if (a == nullptr) return api_fail(GFA_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->block_size < 32 || a->block_size > 1024 || (a->block_size & (a->block_size - 1)) != 0)
    return api_fail(GFA_ERR_UNSUPPORTED, "block_size=%d must be a power of two, 32 to 1024", a->block_size);
  if (a->requests < 1 || a->table_width < 1 || a->free_count < 0 || a->tokens < 0)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "requests=%d and table_width=%d must be positive, free_count=%d and tokens=%d not negative",
                    a->requests, a->table_width, a->free_count, a->tokens);
  if (a->table_stride < a->table_width && a->requests > 1)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "table_stride=%lld below table_width=%d", (long long)a->table_stride, a->table_width);
  const void* ptrs[] = {a->lens, a->fresh, a->table, a->used, a->cu, a->lens_out, a->used_out};
  for (const void* p : ptrs)
    if (!aligned(p, 4)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "plan arrays must be 4-byte aligned pointers");
  if ((a->free_count > 0 && !aligned(a->free_ids, 4)) ||
      (a->tokens > 0 && (!aligned(a->slots, 8) || !aligned(a->positions, 4))))
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "plan arrays must be aligned pointers");
  gfa::Kv4PlanParams p{};
  p.lens = a->lens;
  p.fresh = a->fresh;
  p.free_ids = a->free_ids;
  p.used = a->used;
  p.table = a->table;
  p.table_stride = a->table_stride;
  p.B = a->requests;
  p.M = a->table_width;
  p.F = a->free_count;
  p.T = a->tokens;
  p.bs_log2 = 5;
  while ((1 << p.bs_log2) < a->block_size) ++p.bs_log2;
  p.slots = a->slots;
  p.positions = a->positions;
  p.cu = a->cu;
  p.lens_out = a->lens_out;
  p.used_out = a->used_out;
  return launched(gfa::launch_kv4_plan(p, static_cast<hipStream_t>(a->stream)), "plan");
}

size_t gfa_kv4_attn_workspace_bytes(const gfa_kv4_attn_args* a) {
  if (check_attn(a) != GFA_OK) return 0;
  const Split s = split_of(a);
  return s.few.bytes() + s.many.bytes();
}

int gfa_kv4_attn(const gfa_kv4_attn_args* a) {
  if (int rc = check_attn(a)) return rc;
  if (int rc = check_rows("q", a->q, a->q_strides)) return rc;
  if (int rc = check_rows("o", a->o, a->o_strides)) return rc;
  if (!aligned(a->table, 4) || !aligned(a->lens, 4) || (a->cu != nullptr && !aligned(a->cu, 4)))
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "table, lens and cu must be 4-byte aligned pointers");
  const Split s = split_of(a);
  for (const Part* part : {&s.few, &s.many}) {
    const int64_t join = part->join ? part->row_blocks * part->join_rows * (a->cache.head_dim / part->join_slice) * a->cache.heads_kv : 0;
    if (std::max(part->nblocks, join) > kMostWorkgroups)
      return api_fail(GFA_ERR_UNSUPPORTED, "%lld workgroups exceed one launch", (long long)std::max(part->nblocks, join));
  }
  const size_t need = s.few.bytes() + s.many.bytes();
  if (need > 0 && (!aligned(a->workspace, 16) || a->workspace_bytes < need))
    return api_fail(GFA_ERR_WORKSPACE, "workspace of %zu bytes (16-byte aligned) needed, got %zu", need, a->workspace_bytes);
  gfa::Kv4AttnParams p{};
  p.cache = cache_of(a->cache);
  p.q = static_cast<const uint16_t*>(a->q);
  p.o = static_cast<uint16_t*>(a->o);
  p.qsb = a->q_strides.batch;
  p.qsh = a->q_strides.head;
  p.qsn = a->q_strides.row;
  p.osb = a->o_strides.batch;
  p.osh = a->o_strides.head;
  p.osn = a->o_strides.row;
  p.T = a->batch * a->seq_len;
  p.n.set(a->seq_len);
  p.hkv.set(a->cache.heads_kv);
  p.g.set(a->heads_q / a->cache.heads_kv);
  p.each = p.T / a->requests;
  p.table = a->table;
  p.lens = a->lens;
  p.cu = a->cu;
  p.table_stride = a->table_stride;
  p.B = a->requests;
  p.M = a->table_width;
  p.Hq = a->heads_q;
  p.G = a->heads_q / a->cache.heads_kv;
  p.causal = a->causal != 0;
  p.window = a->causal && a->window <= 0x40000000 ? a->window : 0;  // no table holds 2^30 tokens
  const bool cap = a->softcap > 0.f;
  p.xs = (cap ? a->softcap : a->scale) * 1.4426950408889634f;
  p.cap_a = cap ? a->scale / a->softcap : 0.f;
  p.row_limit = s.row_limit;
  const auto stream = static_cast<hipStream_t>(a->stream);
  const int D = a->cache.head_dim;
  const bool bf16 = a->cache.dtype == GFA_DTYPE_BF16;
  char* ws = static_cast<char*>(a->workspace);
  for (const bool large : {true, false}) {
    const Part& part = large ? s.many : s.few;
    if (!part.runs) continue;
    p.min_tiles = part.min_tiles;
    p.share = part.share;
    p.window_tiles = part.window_tiles;
    p.row_blocks = (int)part.row_blocks;
    p.join_rows = part.join_rows;
    p.join_slice = part.join_slice;
    p.join_parts = part.join_parts;
    p.nblocks = (int)part.nblocks;
    p.slots = (int)part.slots;
    p.part = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + part.part_bytes);
    ws += part.bytes();
    hipError_t err = large ? gfa::launch_kv4_chunk(p, D, bf16, cap, stream) : gfa::launch_kv4_split(p, D, bf16, cap, s.one_block, stream);
    if (err == hipSuccess && part.join) err = gfa::launch_kv4_join(p, D, bf16, large, stream);
    if (err != hipSuccess) return launched(err, "cache attention");
  }
  return gfa::api_ok();
}

}  // extern "C"
