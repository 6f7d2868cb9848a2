// C ABI of the key/value cache in 4 bits: argument checks, work split, launches. Nothing here
// allocates, frees or synchronises.
#include <algorithm>
#include <cmath>

#include "gfa.h"
#include "gfa_kv4.h"
#include "gfa_launch.h"
#include "gfa_verify.h"

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
int row_limit(const gfa_kv4_attn_args* a, int64_t requests) { return requests * a->cache.heads_kv <= 4 ? 128 : 64; }

enum Kind { kWhole, kPrefix, kRest };  // a whole call, the groups' prefixes, the requests behind them

float share_of(int64_t hkv, int target) { return (float)((double)hkv / target * (1.0 + 1.0 / 4096)); }  // see chunk_tiles

void size_part(Part& s, const gfa_kv4_attn_args* a, Kind kind, int64_t row_blocks, int rows, int64_t most_rows, int min_tiles, int target, int spare) {
  int64_t tiles = (int64_t)a->table_width * a->cache.block_size / 32;  // most tiles of a row block
  if (kind == kWhole && a->causal && a->window > 0) {
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
  s.join = chunks > 1 || kind != kWhole;
  s.min_tiles = chunks > 1 ? min_tiles : 0x3fffffff;
  s.row_blocks = row_blocks;
  // The join. Of the chunk kernel: its runs of 1 KB, four waves a workgroup. Of the split kernel: where rows are few, a
  // workgroup takes one row of 128 channels and its lanes share the chunks; else whole rows, where they are many
  // one per group of lanes.
  const int64_t hkv = a->cache.heads_kv, row_bound = std::min<int64_t>(rows, most_rows), n = row_blocks * hkv * row_bound;
  const int D = a->cache.head_dim;
  s.join_slice = rows == kRows && D > 128 && n * (D / 128) <= 1024 ? 128 : D;
  const int groups = 1024 / s.join_slice;
  // (Over prefixes a row has many chunks: 64 answers to a 16k prompt, 32:8 D = 128, two groups of lanes a row 46.2 us, one 50.3;
  // 160 drawn calls: one within 1% of two, four 1 to 4% longer.)
  s.join_parts = n <= 2048 ? groups : kind == kRest ? 2 : 1;
  const int64_t wgs = rows == kRows ? (row_bound * s.join_parts + groups - 1) / groups : rows / 32 * (D <= 128 ? 16 : D / 8) / 4;
  const int64_t most_wgs = 4096 / std::max<int64_t>(1, row_blocks * hkv);
  s.join_rows = (int)std::max<int64_t>(1, std::min(wgs, most_wgs));
  s.share = share_of(hkv, target);
  const int64_t items = std::min(row_blocks * chunks, row_blocks + (target + hkv - 1) / hkv);
  s.nblocks = items * hkv + spare;
  if (s.join) {
    s.slots = kind != kWhole ? items : std::min(row_blocks * chunks, 2 * target / hkv + 1);
    s.part_bytes = (size_t)(s.slots * hkv) * rows * a->cache.head_dim * sizeof(float);
    s.ml_bytes = (size_t)(s.slots * hkv) * rows * 2 * sizeof(float);
  }
}

// The same of a group's rows. Below a workgroup's 128 the chunk kernel's waves share the keys (gfa_kv4_chunk.inc), so the line is lower
// where there are KV heads to fill the GPU with: four prompts of 8k with 12 answers each, 32:8 D = 128, 48 rows 37 us (split kernel 41),
// 16:8 D = 256 60 (69), 32:4 D = 512 60 (66); one KV head at D = 256 24.5 (23.4), 32:8 at D = 64 32.9 (30.3), 10 answers to four of 4k, 16:4
// D = 64, 22.2 (19.0).
int group_limit(const gfa_kv4_attn_args* a) { return a->cache.heads_kv >= 4 && a->cache.head_dim >= 128 ? 32 : 64; }

// Most new tokens of a request, as far as the host knows.
int64_t most_new(const gfa_kv4_attn_args* a) {
  const int64_t T = (int64_t)a->batch * a->seq_len;
  return a->cu == nullptr ? T / a->requests : a->max_new > 0 ? std::min<int64_t>(a->max_new, T) : T;
}

Split split_of(const gfa_kv4_attn_args* a, Kind kind) {
  Split s{};
  const int64_t G = a->heads_q / a->cache.heads_kv, T = (int64_t)a->batch * a->seq_len;
  // a prefix is that of two requests at least, and of any number of them
  const int64_t R = kind == kPrefix ? std::max<int64_t>(1, a->requests / 2) : a->requests;
  const int64_t most = kind == kPrefix ? T : most_new(a);
  // No request can have more rows than the limit: then all are the split kernel's, whatever max_new promised.
  s.one_block = most * G <= kRows;
  const int limit = kind == kPrefix ? group_limit(a) : row_limit(a, R);
  s.row_limit = kind == kRest || most * G <= limit ? 0x7fffffff : limit;
  const int D = a->cache.head_dim, big = kind == kPrefix ? gfa::kSharedRows : gfa::kv4_chunk_rows(D);
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
  const int spare = a->cu && kind != kPrefix ? 64 : 0;
  if (kind == kWhole) {
    // Chunks of at least 8 tiles, two a wave (16k keys, D = 512: 19.7 us; of 4: 21.0, of 2: 26.2). Twice the CUs' number
    // of workgroups where there is work for them (32 ragged requests: 512 96 us, 1024 107 us, 2048 129 us; 64 full
    // ones 152-154 us with each).
    size_part(s.few, a, kind, few, kRows, most * G, 8, 512, spare);
  } else {
    // At D = 512 a CU holds one workgroup, and the prefixes' and the requests' share the GPU (eight answers to each of four prompts,
    // 32:4: 160 of the chunk kernel and 128 52.8 us, 160 and 256 57-61, 256 and 256 63-71; 39 drawn calls: 64 or 256
    // of the requests within 0.5%, 128 of the prefixes' split kernel 3% shorter, 512 1% longer). A few answers leave it to
    // chunks of one tile a wave (four answers to 700 tokens, 8:1 D = 512, taken apart: 15.8 us, of two 17.5).
    const int min_tiles = (int64_t)a->requests * a->cache.heads_kv <= 16 ? 4 : 8;
    size_part(s.few, a, kind, few, kRows, most * G, min_tiles, D < 512 ? 512 : kind == kPrefix ? 256 : 128, spare);
  }
  // Of the chunk kernel as many workgroups as the CUs hold at once (256 tokens at 16k, D = 512: 290 us, twice as many 314;
  // 1024 tokens, D = 128: 256 482 us, 512 375, 768 354, 1024 360). Its chunks cost as much again as some tiles, so the
  // more of the GPU the row blocks take by themselves the longer a chunk has to be: 256 tokens of one request, window
  // 1024, 33 us with chunks of 8 tiles, 57 unsplit; 1000 tokens beside seven requests 66 us with 18 tiles, 74 unsplit;
  // 512 tokens of four requests 76-84 us split, 71 unsplit.
  // Of prefixes one workgroup a CU: their sums are as much again as what they read (64 answers to a 16k prompt, D = 128: 46.2 us, two
  // 57; 121 drawn calls: one and a half 2 to 4% shorter at D = 64 and 128, the same at 256, two 3% longer there; 39 at D = 512: 128 workgroups 5% and 256
  // 6% longer than 160), chunks of 8 tiles however many the row blocks could be (31 answers to each of three prompts of 500, 32:8 D = 128: 30 us, of 32
  // 36), of 4 where they are few (16 answers of 4 drafted tokens, 3k, 8:4 D = 256: 24.3 us, of 8 27.8).
  const int64_t alone = many * a->cache.heads_kv;
  const int target = kind != kPrefix ? 256 * gfa::kv4_chunk_wgs(D) : D < 512 ? 256 : 160;
  const int min_tiles = kind == kPrefix ? (alone <= 16 ? 4 : 8) : alone >= 256 ? 64 : alone >= 128 ? 32 : 8;
  size_part(s.many, a, kind, many, big, most * G, min_tiles, target, 0);
  return s;
}

// What taking prefixes apart saves is counted in passes of the split kernel over a tile (one row block, one KV head): `tiles` of them take
// a us of the whole GPU (by head dim, 151k passes 72 us and 60k 52 us, 24k 43 us, 43k 133 us), one of the chunk kernel takes as long as many_cost
// of them. many_cost, and what the choice has to promise, are the ones with which 1270 drawn calls, in tight tables and in wide ones, took the least time;
// soft-capping costs the chunk kernel most at D = 64, where scores are the larger part of its work.
struct Rate {
  float tiles, many_cost;
};
Rate rate_of(int D, bool cap) {
  return D == 64 ? Rate{2100.f, cap ? 7.f : 3.5f} : D == 128 ? Rate{1200.f, 6.f} : D == 256 ? Rate{570.f, cap ? 5.f : 4.f} : Rate{320.f, 5.2f};
}
// A row block whose request is taken apart leaves sums in two parts and is joined, about as much again as 10 tiles of it; and a call has
// the other kernel's start and the joins' latency more, which D = 512's one workgroup a CU makes longest. Apart against whole in the same launch, us: two
// answers of 5 tokens to a 2k prompt, 32:4 D = 512, 35.7 24.0; 16 answers of 8 to each of eight prompts of 740 tokens, 8:4 D = 256, 66 51;
// 44 to each of four of 1352, 32:8 D = 128, 41 52; 64 to one of 16k, 47 215.
constexpr float kApartCost = 10.f;
float worth_of(const gfa_kv4_attn_args* a) {
  const int D = a->cache.head_dim;
  return (D == 512 ? 10.f : 4.f) * rate_of(D, a->softcap > 0.f).tiles / (float)a->cache.heads_kv;
}
// The call without prefixes is a launch shorter, and its kernel keeps more workgroups on a CU: whole requests in the shared launch take 3 to 5 us
// longer, at D = 512 sometimes less (26 requests of 8 tokens over 1.5k, 8:1, 29.6 against 35.2). So it is left to calls whose tables
// can hold far more than the choice has to promise. Of the 1270 calls 138 take over a tenth longer than without prefixes then, most of
// them short requests in wide tables (lengths are not the host's to see); from the choice's own line on, 4 us, it was 344. (300 others, geometric
// mean: 25.7 us without prefixes, 24.3 so.)
float least_of(const gfa_kv4_attn_args* a) {
  const int D = a->cache.head_dim;
  return (D == 512 ? 8.f : 20.f) * rate_of(D, a->softcap > 0.f).tiles / (float)a->cache.heads_kv;
}

// Whether prefixes may be taken apart: without a window, which bounds what a request reads, and for requests of few rows; where
// max_new is not known, of few rows on average (those of many are the chunk kernel's then, see steps_of). Not where the tables are too narrow for it to pay.
bool takes_prefixes(const gfa_kv4_attn_args* a) {
  if (a->shared_skip == nullptr || (a->causal && a->window > 0) || a->requests < 2) return false;
  const int64_t T = (int64_t)a->batch * a->seq_len, G = a->heads_q / a->cache.heads_kv;
  const int64_t rows = a->max_new > 0 ? a->max_new : (T + a->requests - 1) / a->requests;
  if (rows * G > row_limit(a, a->requests)) return false;
  const double tiles = (double)a->table_width * a->cache.block_size / 32, row_blocks = (double)(T * G + (kRows - 1) * (int64_t)a->requests) / kRows;
  return a->shared_apart != 0 || (tiles - kApartCost) * row_blocks > least_of(a);
}

// The parts of a call.
struct Steps {
  Split whole, prefix, rest;  // whole; or the two others, and of whole the chunk kernel's part
  bool shared;
  size_t bytes() const {
    if (!shared) return whole.few.bytes() + whole.many.bytes();
    return prefix.few.bytes() + prefix.many.bytes() + rest.few.bytes() + 64 + (size_t)rest.few.row_blocks * sizeof(gfa::Kv4Join) + whole.many.bytes();
  }
};
Steps steps_of(const gfa_kv4_attn_args* a) {
  Steps s{};
  s.shared = takes_prefixes(a);
  s.whole = split_of(a, kWhole);
  if (!s.shared) return s;
  // Where max_new is not known a prompt's chunk may stand among requests of few rows, and belongs to the chunk kernel all the same: 8000
  // tokens over 8000 beside 200 of one token, 16:16 D = 64, 769 us (by 16 rows at a time 1191), 1000 over 8000, 32:4 D = 512, 771 (1168).
  s.whole.few = Part{};
  s.prefix = split_of(a, kPrefix);
  s.rest = split_of(a, kRest);
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

int log2_of(int block_size) {
  int log2 = 5;
  while ((1 << log2) < block_size) ++log2;
  return log2;
}

// ---- pages ----

int check_layers(const gfa_kv4_cache* caches, int layers) {
  if (caches == nullptr || layers < 1) return api_fail(GFA_ERR_INVALID_ARGUMENT, "at least one cache is needed");
  for (int i = 0; i < layers; ++i) {
    if (int rc = check_cache(caches[i])) return rc;
    if (caches[i].num_blocks != caches[0].num_blocks || caches[i].block_size != caches[0].block_size)
      return api_fail(GFA_ERR_INVALID_ARGUMENT, "caches of %d blocks of %d and %d blocks of %d tokens do not belong to one table",
                      caches[0].num_blocks, caches[0].block_size, caches[i].num_blocks, caches[i].block_size);
  }
  return GFA_OK;
}

constexpr int kLayersAtOnce = gfa::kKv4CopyArrays / 2;

int64_t block_bytes(const gfa_kv4_cache& c, bool scales) {
  return (int64_t)c.heads_kv * 2 * c.block_size * (scales ? c.head_dim / 32 : c.head_dim / 2);
}
int64_t pieces_of(int64_t bytes) { return (bytes + gfa::kKv4CopyPiece - 1) / gfa::kKv4CopyPiece; }

int check_copy(const gfa_kv4_cache* caches, int layers, int64_t pairs) {
  for (int l0 = 0; l0 < layers; l0 += kLayersAtOnce) {
    int64_t pieces = 0;
    for (int i = l0; i < std::min(layers, l0 + kLayersAtOnce); ++i) pieces += pieces_of(block_bytes(caches[i], false)) + pieces_of(block_bytes(caches[i], true));
    if (pieces * pairs > 0x7fffffff)
      return api_fail(GFA_ERR_UNSUPPORTED, "%lld pieces of %lld blocks exceed one launch", (long long)pieces, (long long)pairs);
  }
  return GFA_OK;
}

// (Of a call that check_copy has passed.)
int copy_blocks(const gfa_kv4_cache* caches, int layers, const int32_t* src, const int32_t* dst, const int32_t* count, int pairs, hipStream_t stream) {
  for (int l0 = 0; l0 < layers; l0 += kLayersAtOnce) {
    gfa::Kv4CopyParams p{};
    int pieces = 0;
    for (int i = l0; i < std::min(layers, l0 + kLayersAtOnce); ++i) {
      for (const bool scales : {false, true}) {
        p.base[p.arrays] = static_cast<uint8_t*>(scales ? caches[i].scales : caches[i].codes);
        p.bytes[p.arrays] = block_bytes(caches[i], scales);
        p.first[p.arrays] = pieces;
        pieces += (int)pieces_of(p.bytes[p.arrays]);
        ++p.arrays;
      }
    }
    p.num_blocks = caches[0].num_blocks;
    p.pairs = pairs;
    p.pieces.set(pieces);
    p.src = src;
    p.dst = dst;
    p.count = count;
    if (const hipError_t err = gfa::launch_kv4_copy(p, stream); err != hipSuccess) return launched(err, "block copy");
  }
  return gfa::api_ok();
}

int pages_call(const gfa_kv4_pages_args* a, bool fork) {
  if (a == nullptr) return api_fail(GFA_ERR_INVALID_ARGUMENT, "args is NULL");
  if (int rc = check_layers(a->caches, a->layers)) return rc;
  const int blocks = a->caches[0].num_blocks, bs = a->caches[0].block_size, rows = fork ? a->rows : a->requests;
  if (blocks > gfa::kKv4PagesBlocks) return api_fail(GFA_ERR_UNSUPPORTED, "a pool of %d blocks (most %d)", blocks, gfa::kKv4PagesBlocks);
  if (a->requests < 1 || a->table_width < 1 || rows < 1 || a->free_count < 0)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "requests=%d, table_width=%d and rows=%d must be positive, free_count=%d not negative",
                    a->requests, a->table_width, rows, a->free_count);
  if (a->requests > gfa::kKv4PagesRows || rows > gfa::kKv4PagesRows)
    return api_fail(GFA_ERR_UNSUPPORTED, "%d requests and %d rows (most %d)", a->requests, rows, gfa::kKv4PagesRows);
  if ((int64_t)a->table_width * bs > 0x40000000)
    return api_fail(GFA_ERR_UNSUPPORTED, "block tables of %lld tokens (most 2^30)", (long long)a->table_width * bs);
  if ((int64_t)std::max(a->requests, rows) * a->table_width > 0x40000000)
    return api_fail(GFA_ERR_UNSUPPORTED, "block tables of %d x %d entries (most 2^30)", std::max(a->requests, rows), a->table_width);
  if (a->table_stride < a->table_width && a->requests > 1)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "table_stride=%lld below table_width=%d", (long long)a->table_stride, a->table_width);
  if (!fork && a->free_count != blocks)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "free_count=%d: a compacted pool's free list holds all of its %d blocks", a->free_count, blocks);
  for (const void* p : {(const void*)a->table, (const void*)a->lens, (const void*)a->table_out, (const void*)a->used_out})
    if (!aligned(p, 4)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "page arrays must be 4-byte aligned pointers");
  if ((a->free_count > 0 && !aligned(a->free_ids, 4)) || (fork && (!aligned(a->used, 4) || !aligned(a->lens_out, 4))) ||
      (fork && a->parents != nullptr && !aligned(a->parents, 4)) || (fork && a->keep != nullptr && !aligned(a->keep, 4)))
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "page arrays must be 4-byte aligned pointers");
  const int most = fork ? rows : blocks / 2;  // pairs
  if (int rc = check_copy(a->caches, a->layers, most)) return rc;
  const size_t need = gfa_kv4_pages_workspace_bytes(fork ? rows : blocks);
  if (!aligned(a->workspace, 4) || a->workspace_bytes < need)
    return api_fail(GFA_ERR_WORKSPACE, "workspace of %zu bytes (4-byte aligned) needed, got %zu", need, a->workspace_bytes);
  gfa::Kv4PagesParams p{};
  p.table = a->table;
  p.lens = a->lens;
  p.parents = fork ? a->parents : nullptr;
  p.keep = fork ? a->keep : nullptr;
  p.used = a->used;
  p.table_stride = a->table_stride;
  p.B = a->requests;
  p.M = a->table_width;
  p.rows = rows;
  p.F = a->free_count;
  p.num_blocks = blocks;
  p.words = gfa::kv4_pages_words(blocks);
  p.bs_log2 = log2_of(bs);
  p.m.set(a->table_width);
  p.free_ids = a->free_ids;
  p.table_out = a->table_out;
  p.lens_out = a->lens_out;
  p.used_out = a->used_out;
  p.count = static_cast<int*>(a->workspace);
  p.src = p.count + 1;
  p.dst = p.src + most;
  const auto stream = static_cast<hipStream_t>(a->stream);
  const hipError_t err = fork ? gfa::launch_kv4_fork(p, stream) : gfa::launch_kv4_compact(p, stream);
  if (err != hipSuccess) return launched(err, fork ? "fork" : "compaction");
  return copy_blocks(a->caches, a->layers, p.src, p.dst, p.count, most, stream);
}

// ---- verification ----

// A wave's entries: about 4096 waves a call, one to four steps each (the entry drawn is then found in one pass of a workgroup).
struct Segments {
  int length;
  int64_t count;
};
Segments verify_segments(int64_t requests, int64_t vocab) {
  const int64_t step = gfa::kVerifyStep, length = std::max<int64_t>(1, std::min<int64_t>(4, (vocab * requests + 4096 * step - 1) / (4096 * step))) * step;
  return Segments{(int)std::min<int64_t>(length, (vocab + step - 1) / step * step), (vocab + length - 1) / length};
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

size_t gfa_kv4_pages_workspace_bytes(int32_t n) { return n < 0 ? 0 : (2 * (size_t)n + 1) * sizeof(int32_t); }

int gfa_kv4_copy(const gfa_kv4_cache* caches, int32_t layers, const int32_t* src, const int32_t* dst, int32_t pairs, void* stream) {
  if (int rc = check_layers(caches, layers)) return rc;
  if (pairs < 0) return api_fail(GFA_ERR_INVALID_ARGUMENT, "pairs=%d must not be negative", pairs);
  if (pairs == 0) return gfa::api_ok();
  if (!aligned(src, 4) || !aligned(dst, 4)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "src and dst must be 4-byte aligned pointers");
  if (int rc = check_copy(caches, layers, pairs)) return rc;
  return copy_blocks(caches, layers, src, dst, nullptr, pairs, static_cast<hipStream_t>(stream));
}

int gfa_kv4_fork(const gfa_kv4_pages_args* a) { return pages_call(a, true); }
int gfa_kv4_compact(const gfa_kv4_pages_args* a) { return pages_call(a, false); }

int gfa_kv4_share(const gfa_kv4_share_args* a) {
  if (a == nullptr) return api_fail(GFA_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->block_size < 32 || a->block_size > 1024 || (a->block_size & (a->block_size - 1)) != 0)
    return api_fail(GFA_ERR_UNSUPPORTED, "block_size=%d must be a power of two, 32 to 1024", a->block_size);
  if (a->requests < 1 || a->table_width < 1 || a->least < 1)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "requests=%d, table_width=%d and least=%d must be positive", a->requests, a->table_width, a->least);
  if (a->requests > gfa::kKv4ShareMost) return api_fail(GFA_ERR_UNSUPPORTED, "%d requests (most %d)", a->requests, gfa::kKv4ShareMost);
  if ((int64_t)a->table_width * a->block_size > 0x40000000)
    return api_fail(GFA_ERR_UNSUPPORTED, "block tables of %lld tokens (most 2^30)", (long long)a->table_width * a->block_size);
  if (a->table_stride < a->table_width && a->requests > 1)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "table_stride=%lld below table_width=%d", (long long)a->table_stride, a->table_width);
  for (const void* p : {(const void*)a->table, (const void*)a->lens, (const void*)a->cu, (const void*)a->skip, (const void*)a->cu_out,
                        (const void*)a->lens_out})
    if (!aligned(p, 4)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "share arrays must be 4-byte aligned pointers");
  gfa::Kv4ShareParams p{};
  p.table = a->table;
  p.lens = a->lens;
  p.cu = a->cu;
  p.table_stride = a->table_stride;
  p.R = a->requests;
  p.M = a->table_width;
  p.bs_log2 = log2_of(a->block_size);
  p.least = a->least;
  p.skip = a->skip;
  p.cu_out = a->cu_out;
  p.lens_out = a->lens_out;
  return launched(gfa::launch_kv4_share(p, static_cast<hipStream_t>(a->stream)), "share");
}

size_t gfa_kv4_verify_workspace_bytes(int32_t requests, int32_t vocab) {
  if (requests < 1 || vocab < 1) return 0;
  return (size_t)requests * (verify_segments(requests, vocab).count * 2 * sizeof(double) + sizeof(double));
}

int gfa_kv4_verify(const gfa_kv4_verify_args* a) {
  if (a == nullptr) return api_fail(GFA_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->token_count < 1 || a->vocab < 1 || a->requests < 1)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "token_count=%d, vocab=%d and requests=%d must be positive", a->token_count, a->vocab, a->requests);
  if (a->requests > 65535) return api_fail(GFA_ERR_UNSUPPORTED, "%d requests (most 65535)", a->requests);
  if (a->vocab > 1 << 30) return api_fail(GFA_ERR_UNSUPPORTED, "a vocabulary of %d (most 2^30)", a->vocab);
  if (a->type < 0 || a->type > 2) return api_fail(GFA_ERR_INVALID_ARGUMENT, "type=%d is none of 0, 1, 2", a->type);
  if (a->cu == nullptr && a->token_count % a->requests != 0)
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "%d tokens do not divide among %d requests (pass cu)", a->token_count, a->requests);
  const Segments s = verify_segments(a->requests, a->vocab);
  if ((s.count + 3) / 4 * a->requests > kMostWorkgroups)
    return api_fail(GFA_ERR_UNSUPPORTED, "%d requests over a vocabulary of %d exceed one launch", a->requests, a->vocab);
  if (a->target_stride < 0 || a->draft_stride < 0) return api_fail(GFA_ERR_INVALID_ARGUMENT, "row strides must not be negative");
  const unsigned size = a->type == 2 ? 4 : 2;
  if (!aligned(a->target, size) || (a->draft != nullptr && !aligned(a->draft, size)))
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "target and draft must be aligned to their type");
  if (!aligned(a->tokens, 8) || !aligned(a->follows, 8)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "tokens and follows must be 8-byte aligned pointers");
  for (const void* p : {(const void*)a->accept, (const void*)a->sample, (const void*)a->lens, (const void*)a->accepted, (const void*)a->lens_out})
    if (!aligned(p, 4)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "verify arrays must be 4-byte aligned pointers");
  if (a->cu != nullptr && !aligned(a->cu, 4)) return api_fail(GFA_ERR_INVALID_ARGUMENT, "cu must be a 4-byte aligned pointer");
  const size_t need = gfa_kv4_verify_workspace_bytes(a->requests, a->vocab);
  if (!aligned(a->workspace, 8) || a->workspace_bytes < need)
    return api_fail(GFA_ERR_WORKSPACE, "workspace of %zu bytes (8-byte aligned) needed, got %zu", need, a->workspace_bytes);
  gfa::VerifyParams p{};
  p.target = a->target;
  p.draft = a->draft;
  p.ts = a->target_stride;
  p.ds = a->draft_stride;
  p.tokens = a->tokens;
  p.accept = a->accept;
  p.sample = a->sample;
  p.lens = a->lens;
  p.cu = a->cu;
  p.T = a->token_count;
  p.V = a->vocab;
  p.R = a->requests;
  p.each = a->token_count / a->requests;
  p.segment = s.length;
  p.segments = s.count;
  p.sums = static_cast<double*>(a->workspace);
  p.taken = reinterpret_cast<int*>(p.sums + (size_t)a->requests * s.count * 2);
  p.follows = a->follows;
  p.accepted = a->accepted;
  p.lens_out = a->lens_out;
  return launched(gfa::launch_verify(p, a->type, static_cast<hipStream_t>(a->stream)), "verification");
}

size_t gfa_kv4_attn_workspace_bytes(const gfa_kv4_attn_args* a) {
  if (check_attn(a) != GFA_OK) return 0;
  return steps_of(a).bytes();
}

int gfa_kv4_attn(const gfa_kv4_attn_args* a) {
  if (int rc = check_attn(a)) return rc;
  if (int rc = check_rows("q", a->q, a->q_strides)) return rc;
  if (int rc = check_rows("o", a->o, a->o_strides)) return rc;
  if (!aligned(a->table, 4) || !aligned(a->lens, 4) || (a->cu != nullptr && !aligned(a->cu, 4)))
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "table, lens and cu must be 4-byte aligned pointers");
  if (a->shared_skip != nullptr &&
      (a->cu == nullptr || !aligned(a->shared_skip, 4) || !aligned(a->shared_cu, 4) || !aligned(a->shared_lens, 4)))
    return api_fail(GFA_ERR_INVALID_ARGUMENT, "shared prefixes need cu, and 4-byte aligned pointers");
  const Steps s = steps_of(a);
  int64_t most = s.prefix.many.nblocks + s.prefix.few.nblocks + s.rest.few.nblocks;
  for (const Part* part : {&s.whole.few, &s.whole.many, &s.rest.few}) {
    const int64_t join = part->join ? part->row_blocks * part->join_rows * (a->cache.head_dim / part->join_slice) * a->cache.heads_kv : 0;
    most = std::max({most, part->nblocks, join});
  }
  if (most > kMostWorkgroups) return api_fail(GFA_ERR_UNSUPPORTED, "%lld workgroups exceed one launch", (long long)most);
  const size_t need = s.bytes();
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
  const auto stream = static_cast<hipStream_t>(a->stream);
  const int D = a->cache.head_dim;
  const bool bf16 = a->cache.dtype == GFA_DTYPE_BF16;
  char* ws = static_cast<char*>(a->workspace);
  hipError_t err = hipSuccess;
  auto sums_of = [&](const Part& part) {
    gfa::Kv4Sums sums{part.min_tiles, part.share, (int)part.nblocks, (int)part.slots, reinterpret_cast<float*>(ws),
                      reinterpret_cast<float*>(ws + part.part_bytes)};
    ws += part.bytes();
    return sums;
  };
  if (s.shared) {
    gfa::Kv4SharedParams sp{};
    p.row_limit = s.whole.row_limit;
    p.row_blocks = (int)s.rest.few.row_blocks;
    p.join_rows = s.rest.few.join_rows;
    p.join_slice = s.rest.few.join_slice;
    p.join_parts = s.rest.few.join_parts;
    p.skip = a->shared_skip;
    sp.p = p;
    sp.group_cu = a->shared_cu;
    sp.group_lens = a->shared_lens;
    sp.row_limit = s.prefix.row_limit;
    sp.many = sums_of(s.prefix.many);
    sp.few = sums_of(s.prefix.few);
    sp.rest = sums_of(s.rest.few);
    sp.joined = reinterpret_cast<int*>(ws);
    sp.joins = reinterpret_cast<gfa::Kv4Join*>(ws + 64);
    sp.many_cost = rate_of(D, cap).many_cost;
    sp.apart_cost = kApartCost;
    const int64_t bound = s.prefix.many.nblocks + s.prefix.few.nblocks + s.rest.few.nblocks;
    sp.grid = (int)std::min<int64_t>(bound, 256 * gfa::kv4_shared_wgs(D) * 3);
    sp.group_blocks = (float)(s.prefix.many.row_blocks + s.prefix.few.row_blocks);
    sp.worth = a->shared_apart != 0 ? -INFINITY : worth_of(a);
    if (err = gfa::launch_kv4_shared(sp, D, bf16, cap, stream); err != hipSuccess) return launched(err, "attention over shared prefixes");
    ws += 64 + s.rest.few.row_blocks * sizeof(gfa::Kv4Join);
  }
  for (const bool large : {true, false}) {
    const Part& part = large ? s.whole.many : s.whole.few;
    if (!part.runs) continue;
    p.row_limit = s.whole.row_limit;
    p.window_tiles = part.window_tiles;
    p.row_blocks = (int)part.row_blocks;
    p.join_rows = part.join_rows;
    p.join_slice = part.join_slice;
    p.join_parts = part.join_parts;
    const gfa::Kv4Sums sums = sums_of(part);
    p.min_tiles = sums.min_tiles;
    p.share = sums.share;
    p.nblocks = sums.nblocks;
    p.slots = sums.slots;
    p.part = sums.part;
    p.part_ml = sums.part_ml;
    err = large ? gfa::launch_kv4_chunk(p, D, bf16, cap, stream) : gfa::launch_kv4_split(p, D, bf16, cap, s.whole.one_block, stream);
    if (err == hipSuccess && part.join) err = gfa::launch_kv4_join(p, D, bf16, large, stream);
    if (err != hipSuccess) break;
  }
  return err != hipSuccess ? launched(err, "cache attention") : gfa::api_ok();
}

}  // extern "C"
