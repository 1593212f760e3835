// Dense causal latent attention of a chunk of new tokens over a paged cache,
// in the absorbed form, for gfx950.
//
// Request r has the query tokens cu[r] .. cu[r + 1) (n of them) and lens[r]
// cached positions, its own tokens the last n.  Token i sees the positions
// j <= lens[r] - n + i:
//   s_j = sm_scale * q . k_j        (base 2 in the kernel: times log2 e)
//   out = sum_j softmax(s)_j * v_j,   v_j = k_j[:512]
// with one key a position for all heads: bf16 rows of 512 latents and 64
// rotary values, or the 528-byte INT8 rows (512 codes and their scale).
//
// Work: the (token, head) rows of a request are flattened and cut into tiles
// of kTM rows (16, 32 or 64), which share every key they read; a tile walks
// its keys in blocks of 64.  Per block, of one workgroup:
//   * the block's rows come into LDS (bf16 rows by direct global -> LDS loads,
//     INT8 rows converted to bf16 once), two buffers, the next block's loads
//     on their way while this one is used;
//   * S^T = K Q^T, the queries held in registers for the whole tile;
//   * softmax against a reference maximum that moves only when some row's
//     maximum passes it by 2^8 (sums and output are scaled to it in fp32), so
//     that most blocks need no exchange of maxima between the two products;
//   * O^T += V^T P^T, each wave its slice of the 512 latents for all rows: P
//     goes through LDS as bf16, V is read from the same rows with transposing
//     reads.
// 64 rows are bound by the products.  Four waves, one per SIMD, so that a lane
// has 512 registers (queries 144, output 128); products of 32 x 32 x 16, which
// need half the instructions and operand reads of the small ones - a single
// wave issues about one instruction in 4 to 5 cycles, and that, not the matrix
// cores, was the limit with 16 x 16 x 32 (6600 cycles a block).  A wave takes
// 32 keys x 32 rows in QK and 128 latents x 64 rows in PV.
// 16 and 32 rows are bound by memory.  Eight waves and products of 16 x 16 x
// 32: a wave takes 16 keys x 16 rows in QK (of a 16-row tile four waves take
// none) and 64 latents in PV.
// Few tiles (decode): the blocks of all tiles are laid end to end and cut
// into equal runs, one per workgroup; a tile that several workgroups share
// leaves fp32 partials that the merge kernel joins.  Many tiles: one
// workgroup each, longest first.
#include <type_traits>

#include "glm53_common.h"

namespace glm53 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kKeys = 64;           // keys per block
constexpr int kMaxSplitTiles = 512; // most tiles whose blocks are cut into equal runs
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;       // how far (log2) a row's maximum may pass the reference

struct ChunkArgs {
  const uint16_t* q;
  int64_t sq_t, sq_h;
  const uint8_t* kv;
  int64_t page_bytes, row_bytes;
  int num_blocks;
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* bt;
  int64_t bt_stride;
  int max_blocks;
  int block_size;
  int num_reqs;
  int first_step;  // of a binary search over the requests: the largest power of two below num_reqs, or 0
  int total_q;
  int heads;
  int num_tiles;   // bound: tile indexes are below it
  float scale_log2;
  uint16_t* out;
  int64_t so_t, so_h;
  int out_align16; // out rows 16-byte aligned (else 8)
  float* lse;      // [total_q][heads], or null
  float* part;     // [2 * workgroups] slots of kTM x 512, accumulator order
  float2* ml;      // [2 * workgroups][kTM]: reference maximum (log2) and sum
  int2* shares;    // [num_tiles]: first and last workgroup of a shared tile, or -1
};

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

template <int kTM>
struct ChunkShape {
  static constexpr bool kBig = kTM == 64;           // products of 32 x 32 x 16
  static constexpr int kWaves = kBig ? 4 : 8;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kOwn = kKeys / kWaves;       // rows of a block that a wave brings in
};

template <int kTM>
struct __attribute__((aligned(16))) ChunkShared {
  struct __attribute__((aligned(16))) Block {
    uint8_t lat[kKeys][2 * kLatent];   // chunk c of 16 bytes of row k at chunk c ^ swizzle(k)
    uint8_t rope[kKeys][2 * kRope];
  } kv[2];
  uint8_t p[kTM][2 * kKeys];           // P, chunk c of row r at c ^ (r % 8), keys in the order of the V operand
  float red[4][kTM];                   // per key group: maxima; at the end the sums
  float ref[kTM];                      // alpha when the reference moves, at the end the reference
  float scl[2][kKeys];                 // INT8 rows' scales
  uint64_t have[2];                    // bit k: key k of the block has a row
  int ends[kMaxSplitTiles];            // blocks up to and with each tile
  int reqs[kMaxSplitTiles];
  int sums[8];
  int flag[2];                         // some row's maximum passed its reference
  int first;
};

__device__ __forceinline__ void wg_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)(p)));
}

// 16 bytes per lane from base + off to LDS at dst + 16 * lane.  Written in asm
// so that the compiler does not wait for it before other LDS reads;
// loads_done() and a barrier come before the first read of what it brings.
// (m0 needs a wait state before its use, an SGPR from v_readlane five.  The
// compiler keeps m0 out of clobber lists and sets it before each use of its
// own; nothing else here uses it.)
__device__ __forceinline__ void load_lds16(uint32_t dst, const uint8_t* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base)
               : "memory");
}
__device__ __forceinline__ void load_lds16_at(uint32_t dst, const uint8_t* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(p) : "memory");
}

// Swizzle of a row's 16-byte chunks (on the low three bits of the chunk's
// index).  Eight lanes that read one chunk of rows 0..7 (the K operand, a
// 128-byte pass) meet eight different chunk columns; four rows 4g .. 4g + 3
// of a transposing read (two neighbouring chunks each) four different pairs.
__device__ __forceinline__ int swizzle(int key) { return ((key & 3) << 1) | ((key >> 2) & 1); }

// Maximum and sum over a row's lanes: four of 16 apart (quad), two of 32 (half).
__device__ __forceinline__ float quad_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_max(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float quad_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Eight INT8 codes as eight bf16 (exact): code + 128 by the byte conversions,
// which run at the full rate (the signed conversion does at a quarter of it).
__device__ __forceinline__ uint4 codes_to_bf16(uint2 v) {
  uint32_t o[4];
  const uint32_t w[2] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u};
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const float f0 = static_cast<float>(w[k] & 0xffu) - 128.f, f1 = static_cast<float>(w[k] >> 8 & 0xffu) - 128.f;
    const float f2 = static_cast<float>(w[k] >> 16 & 0xffu) - 128.f, f3 = static_cast<float>(w[k] >> 24) - 128.f;
    o[2 * k] = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
    o[2 * k + 1] = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A pair of bf16 with the infinities and NaNs replaced by zero.
__device__ __forceinline__ uint32_t finite_bf16x2(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  return w;
}

// One K-step's product of 32 keys and 32 rows, the queries in accumulation
// registers; with kFirst the sum starts at 0.  In asm because the compiler,
// with most of a lane's 512 registers in use, otherwise copies the queries to
// vector registers before the products.  The two wait states before the
// product are what a vector instruction that wrote one of its operands needs;
// nothing but these products writes s, and product_done() comes before its
// first other use.
template <bool kFirst>
__device__ __forceinline__ void product(f32x16& s, bf16x8 k, bf16x8 q) {
  if constexpr (kFirst)
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "a"(q));
  else
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "a"(q));
}
// Wait states between a product and a vector instruction that reads it (19
// for the longest products; 24 here).
__device__ __forceinline__ void product_done(f32x16& s) { asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s)); }

// What a request's tokens and keys are, from values that may be anything:
// token ranges are clipped to the queries there are, lengths to the table.
struct Request {
  int t0, n, len;
};
__device__ __forceinline__ Request request_of(int c0, int c1, int len, int total_q) {
  Request r;
  r.t0 = min(max(c0, 0), total_q);
  r.n = min(max(c1, r.t0), total_q) - r.t0;
  r.len = len;
  return r;
}

// Tile indexes: request r's tiles start at cu[r] * heads / kTM + r, which
// leaves room for a partial tile per request without a prefix sum over the
// requests (the indexes between are empty).
template <int kTM>
__device__ __forceinline__ int first_tile(int t0, int heads, int r) {
  return static_cast<int>(static_cast<int64_t>(t0) * heads / kTM) + r;
}

// The last position that the tile's last row sees (-1: none), within the table.
template <int kTM>
__device__ __forceinline__ int last_key(const Request& r, int row0, int heads, int max_pos) {
  const int rows = r.n * heads;
  const int last_row = min(row0 + kTM, rows) - 1;
  const int64_t k = static_cast<int64_t>(r.len) - r.n + last_row / heads;
  return k < 0 ? -1 : static_cast<int>(k < max_pos ? k : max_pos - 1);
}

// The kernel's arguments read where they are used, instead of being kept in
// scalar registers from the start.
typedef const __attribute__((address_space(4))) ChunkArgs LateArgs;
__device__ __forceinline__ LateArgs* late_args() {
  uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return (LateArgs*)p;
}

template <int kTM, bool kInt8, bool kSplit>
__global__ __launch_bounds__(ChunkShape<kTM>::kThreads, 1) void chunk_mla_kernel(const ChunkArgs a) {
  using Shape = ChunkShape<kTM>;
  constexpr bool kBig = Shape::kBig;
  constexpr int kWaves = Shape::kWaves, kThreads = Shape::kThreads, kOwn = Shape::kOwn;
  constexpr int kRowSize = kBig ? 32 : 16;         // rows and latents of a product
  constexpr int kRT = kTM / kRowSize;              // row tiles
  constexpr int kLT = kLatent / kRowSize / kWaves; // PV: latent tiles of a wave
  constexpr int kDepth = kBig ? 16 : 32;           // K-step of a product
  constexpr int kSteps = (kInt8 ? kLatent : kLatent + kRope) / kDepth;
  constexpr int kPvSteps = kLT * kKeys / kDepth;
  constexpr int kLoads = kOwn + (kInt8 ? 0 : kOwn / 8);   // loads a wave sends per block
  using Acc = std::conditional_t<kBig, f32x16, f32x4>;
  constexpr int kAcc = kBig ? 16 : 4;
  __shared__ ChunkShared<kTM> sh;

  const int w = uniform(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  // What depends on the lane alone would be kept in registers across the
  // block loop; forget() makes the compiler derive it anew from the lane.
  auto forget = [&]() { asm volatile("" : "+v"(lane)); };
  // QK: the wave's key group (32 or 16 keys) and row tile
  const int kg = kBig ? w & 1 : w & 3, rh = kBig ? w >> 1 : w >> 2;
  const bool takes_rows = rh < kRT;
  const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.block_size;
  const int max_pos = static_cast<int>(cap < 0x7fffff00 ? cap : 0x7fffff00);   // a block's positions stay ints

  // ---- which blocks of which tiles are this workgroup's
  int tile, lo = 0, hi = 0, total = 0;
  if (kSplit) {
    constexpr int kTiles = kMaxSplitTiles / kThreads;   // tiles of a thread
    int units[kTiles], req[kTiles], sum = 0;
    int* cu_s = reinterpret_cast<int*>(&sh.kv[0]);      // cu, then lens
    for (int r = threadIdx.x; r <= a.num_reqs; r += kThreads) cu_s[r] = min(max(a.cu[r], 0), a.total_q);
    int* len_s = cu_s + kMaxSplitTiles + 16;
    for (int r = threadIdx.x; r < a.num_reqs; r += kThreads) len_s[r] = a.lens[r];
    wg_barrier();
#pragma unroll
    for (int k = 0; k < kTiles; k++) {
      const int t = static_cast<int>(threadIdx.x) * kTiles + k;
      int at = 0;                                       // the last request that starts at or before tile t
      for (int step = a.first_step; step; step >>= 1) {
        const int r = at + step;
        if (r < a.num_reqs && first_tile<kTM>(cu_s[r], a.heads, r) <= t) at = r;
      }
      const Request rq = request_of(cu_s[at], cu_s[at + 1], len_s[at], a.total_q);
      const int row0 = (t - first_tile<kTM>(rq.t0, a.heads, at)) * kTM;
      req[k] = at;
      units[k] = 0;
      if (t < a.num_tiles && row0 >= 0 && row0 < rq.n * a.heads)
        units[k] = max(1, last_key<kTM>(rq, row0, a.heads, max_pos) / kKeys + 1);
      sum += units[k];
    }
    int upto = sum;                                     // inclusive scan over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 63) sh.sums[w] = upto;
    if (threadIdx.x == 0) sh.first = 0;
    wg_barrier();
    int before = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      const int s = sh.sums[i];
      if (i < w) before += s;
      total += s;
    }
    total = uniform(total);
    if (total == 0) {
      if (blockIdx.x == 0)
        for (int t = threadIdx.x; t < a.num_tiles; t += kThreads) a.shares[t] = make_int2(-1, -1);
      return;   // uniform over the workgroup
    }
    const int64_t groups = min(static_cast<int>(gridDim.x), total);
    if (static_cast<int>(blockIdx.x) >= groups) return;
    lo = static_cast<int>(blockIdx.x * static_cast<int64_t>(total) / groups);
    hi = static_cast<int>((blockIdx.x + 1) * static_cast<int64_t>(total) / groups);
    int end = before + upto - sum;
#pragma unroll
    for (int k = 0; k < kTiles; k++) {
      const int t = static_cast<int>(threadIdx.x) * kTiles + k;
      if (end <= lo && lo < end + units[k]) sh.first = t;
      end += units[k];
      sh.ends[t] = end;
      sh.reqs[t] = req[k];
      if (blockIdx.x == 0 && t < a.num_tiles && units[k] == 0) a.shares[t] = make_int2(-1, -1);
    }
    wg_barrier();
    tile = uniform(sh.first);
  } else {
    tile = a.num_tiles - 1 - static_cast<int>(blockIdx.x);
  }

  for (;; tile++) {
    // ---- the tile: its request, its rows, its blocks [b0, b1)
    int r, b0 = 0, b1 = 0, start = 0, units = 0;
    if (kSplit) {
      if (tile >= kMaxSplitTiles) return;
      start = tile ? uniform(sh.ends[tile - 1]) : 0;
      const int end = uniform(sh.ends[tile]);
      if (start >= hi) return;
      units = end - start;
      if (units == 0) continue;
      r = uniform(sh.reqs[tile]);
      b0 = max(lo - start, 0);
      b1 = min(hi - start, units);
    } else {
      // the last request that starts at or before this tile: its starts are in ascending order
      int begun = 0;
      for (int i = threadIdx.x; i < a.num_reqs; i += kThreads)
        begun += first_tile<kTM>(min(max(a.cu[i], 0), a.total_q), a.heads, i) <= tile;
#pragma unroll
      for (int d = 32; d; d >>= 1) begun += __shfl_xor(begun, d);
      if (lane == 0) sh.sums[w] = begun;
      wg_barrier();
      r = -1;
#pragma unroll
      for (int i = 0; i < kWaves; i++) r += sh.sums[i];
      r = uniform(max(r, 0));
    }
    const Request rq = request_of(uniform(a.cu[r]), uniform(a.cu[r + 1]), uniform(a.lens[r]), a.total_q);
    const int rows = rq.n * a.heads;
    const int row0 = (tile - first_tile<kTM>(rq.t0, a.heads, r)) * kTM;
    if (!kSplit && (row0 < 0 || row0 >= rows)) return;   // an index between two requests
    const int last = last_key<kTM>(rq, row0, a.heads, max_pos);
    if (!kSplit)
      b1 = last >= 0 ? last / kKeys + 1 : 0;
    else if (last < 0)
      b1 = b0;   // nothing to see: its one unit writes the zeros
    // the least of the rows' last positions: keys past it are masked for some row
    const int64_t least64 = static_cast<int64_t>(rq.len) - rq.n + row0 / a.heads;
    const int least = static_cast<int>(least64 < -1 ? -1 : least64 < last ? least64 : last);

    if (kSplit) wg_barrier();   // LDS is free (the tile before, the scan)

    // ---- bringing blocks in.  Wave w brings in the rows of keys kOwn w ... .
    // Lane c (of each kOwn) looks up key kOwn w + c: its page in the table, one
    // block ahead of its use, then its row's address.  A key past the last one
    // seen, or whose page is not in the table or the cache, has no row: the
    // cache's first is read in its place and zeroed.  After the last block
    // there are no rows, and the loads bring nothing that is used.
    uint2 codes[kInt8 ? kOwn : 1];
    float scale = 0.f;
    int pos = b0 * kKeys + kOwn * w + (lane & (kOwn - 1));   // of the block that `page` is for
    int pg = pos / a.block_size, in_page = pos - pg * a.block_size, page = -1;
    const int step_pg = kKeys / a.block_size, step_in = kKeys - step_pg * a.block_size;
    const int32_t* bt = a.bt + static_cast<int64_t>(r) * a.bt_stride;
    auto look_up = [&](int b) { page = b < b1 && pos <= last && pg < a.max_blocks ? bt[pg] : -1; };
    auto advance = [&]() {
      pos += kKeys;
      pg += step_pg;
      in_page += step_in;
      if (in_page >= a.block_size) in_page -= a.block_size, pg++;
    };
    uint32_t row_lo = 0, row_hi = 0, mine = 0;   // addresses; bit j: this wave's row j is there
    constexpr uint32_t kAll = (1u << kOwn) - 1;
    auto address = [&](int b) {
      const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_blocks);
      mine = static_cast<uint32_t>(__ballot(ok)) & kAll;
      const uint64_t at = reinterpret_cast<uint64_t>(a.kv) +
                          (ok ? page * static_cast<uint64_t>(a.page_bytes) + in_page * static_cast<uint64_t>(a.row_bytes) : 0);
      row_lo = static_cast<uint32_t>(at), row_hi = static_cast<uint32_t>(at >> 32);
      if (lane == 0) {
        if constexpr (kBig)
          reinterpret_cast<uint16_t*>(&sh.have[b & 1])[w] = static_cast<uint16_t>(mine);
        else
          reinterpret_cast<uint8_t*>(&sh.have[b & 1])[w] = static_cast<uint8_t>(mine);
      }
    };
    // load j of kLoads of block b
    auto bring = [&](int b, int j) {
      auto& blk = sh.kv[b & 1];
      if (j < kOwn) {
        const uint64_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(row_lo, j)) |
                            static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(row_hi, j))) << 32;
        const uint8_t* row = reinterpret_cast<const uint8_t*>(at);
        if constexpr (kInt8)
          codes[j] = *reinterpret_cast<const uint2*>(row + 8 * lane);
        else
          load_lds16(lds_offset(blk.lat[kOwn * w + j]), row, (16 * lane) ^ (16 * swizzle(j)));
      } else if constexpr (!kInt8) {
        const int key = 8 * (j - kOwn) + (lane >> 3);
        const uint64_t at = static_cast<uint32_t>(__shfl(static_cast<int>(row_lo), key)) |
                            static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(row_hi), key))) << 32;
        load_lds16_at(lds_offset(blk.rope[kOwn * w + 8 * (j - kOwn)]),
                      reinterpret_cast<const uint8_t*>(at) + 2 * kLatent + 16 * ((lane & 7) ^ swizzle(key)));
      }
      if (kInt8 && j == kOwn - 1)
        scale = *reinterpret_cast<const float*>((row_lo | static_cast<uint64_t>(row_hi) << 32) + kLatent);
    };
    // INT8: row j of the wave's rows of block b as bf16 into LDS (0 without a row)
    auto put_row = [&](int b, int j) {
      if constexpr (kInt8) {
        const uint32_t keep = 0u - (mine >> j & 1);
        *reinterpret_cast<uint4*>(&sh.kv[b & 1].lat[kOwn * w + j][(16 * lane) ^ (16 * swizzle(j))]) =
            codes_to_bf16(make_uint2(codes[j].x & keep, codes[j].y & keep));
        if (j == kOwn - 1 && lane < kOwn) sh.scl[b & 1][kOwn * w + lane] = mine >> lane & 1 ? scale : 0.f;
      }
    };

    if (b0 < b1) {
      look_up(b0);
      address(b0);
      advance();
#pragma unroll
      for (int j = 0; j < kLoads; j++) bring(b0, j);
      look_up(b0 + 1);
    }

    // ---- the queries (rows past the last: the last, not stored).  Several
    // waves need each, so they come through LDS once, in the buffer that the
    // second block will take, laid out like keys: wave w brings in every
    // kWaves-th row.
    bf16x8 qf[kSteps];
    {
      auto& qs = sh.kv[(b0 + 1) & 1];
      constexpr int kMine = kTM / kWaves;
      const int row = min(row0 + kWaves * min(lane & 15, kMine - 1) + w, rows - 1);
      const int tok = row / a.heads, head = row - tok * a.heads;
      const uint64_t at = reinterpret_cast<uint64_t>(a.q + static_cast<int64_t>(rq.t0 + tok) * a.sq_t +
                                                     static_cast<int64_t>(head) * a.sq_h);
      const int at_lo = static_cast<int>(at), at_hi = static_cast<int>(at >> 32);
#pragma unroll
      for (int j = 0; j < kMine; j++) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(
            static_cast<uint32_t>(__builtin_amdgcn_readlane(at_lo, j)) |
            static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(at_hi, j))) << 32);
        const int key = kWaves * j + w;
        load_lds16(lds_offset(qs.lat[key]), from, 16 * (lane ^ swizzle(key)));
        if constexpr (!kInt8) {
          if (lane < 8) load_lds16(lds_offset(qs.rope[key]), from, 2 * kLatent + 16 * (lane ^ swizzle(key)));
        }
      }
      loads_done();   // the queries, and the first block's rows
      wg_barrier();
      const int key = kRowSize * (takes_rows ? rh : 0) + (lane & (kRowSize - 1)), sw = swizzle(lane), part = lane / kRowSize;
      constexpr int kChunks = kDepth / 8;   // 16-byte chunks of a K-step
#pragma unroll
      for (int st = 0; st < kSteps; st++) {
        const int chunk = kChunks * st;     // + part
        const uint8_t* from = chunk < 64 ? qs.lat[key] + 16 * (((chunk & 7) + part) ^ sw) + 128 * (chunk >> 3)
                                         : qs.rope[key] + 16 * ((chunk - 64 + part) ^ sw);
        qf[st] = *reinterpret_cast<const bf16x8*>(from);
      }
    }
    Acc acc[kLT][kRT];
#pragma unroll
    for (int i = 0; i < kLT; i++)
#pragma unroll
      for (int j = 0; j < kRT; j++)
#pragma unroll
        for (int e = 0; e < kAcc; e++) acc[i][j][e] = 0.f;
    // the reference maximum (log2) of this lane's row, from the least number on: every other logit passes it
    float ref = -3.4028234663852886e38f, sum = 0.f;
    if (b0 < b1) {
#pragma unroll
      for (int j = 0; j < kOwn; j++) put_row(b0, j);
    }
    if (threadIdx.x == 0) sh.flag[0] = sh.flag[1] = 0;

    for (int b = b0; b < b1; b++) {
      loads_done();   // this wave's rows of block b
      auto& blk = sh.kv[b & 1];
      if (!kInt8 && mine != kAll) {
        for (int j = 0; j < kOwn; j++)
          if (!(mine >> j & 1)) {
            *reinterpret_cast<uint4*>(&blk.lat[kOwn * w + j][16 * lane]) = make_uint4(0, 0, 0, 0);
            if (lane < 8) *reinterpret_cast<uint4*>(&blk.rope[kOwn * w + j][16 * lane]) = make_uint4(0, 0, 0, 0);
          }
      }
      wg_barrier();   // every wave's rows are there; nobody reads the other buffer, P or the maxima any more
      forget();
      if (w == 0 && lane == 0) sh.flag[(b + 1) & 1] = 0;
      const uint64_t have_v = sh.have[b & 1];
      address(b + 1);

      // ---- S^T = K Q^T: the wave's keys, one row a lane.  Each K-step's
      // operand is read some steps before its product; between the steps the
      // next block's rows are asked for - all of them here where memory bounds
      // the loop, and spread over the block where the products do: sent at
      // once they fill the CU's miss queue and hold up the products behind.
      constexpr int kInQk = kBig && !kInt8 ? 12 : kLoads, kInSm = kBig && !kInt8 ? 3 : 0;
      Acc s;
      if (takes_rows) {
        constexpr int kRead = kBig ? 6 : 5, kChunks = kDepth / 8;
        const int key = kRowSize * kg + (lane & (kRowSize - 1)), sw = swizzle(lane), part = lane / kRowSize;
        const uint8_t* base[8 / kChunks];
#pragma unroll
        for (int i = 0; i < 8 / kChunks; i++) base[i] = blk.lat[key] + 16 * ((kChunks * i + part) ^ sw);
        const uint8_t* rope = blk.rope[key];
        auto operand = [&](int st) {
          const int chunk = kChunks * st;
          return *reinterpret_cast<const bf16x8*>(chunk < 64 ? base[st % (8 / kChunks)] + 128 * (chunk >> 3)
                                                             : rope + 16 * ((chunk - 64 + part) ^ sw));
        };
        bf16x8 k[kSteps];
        Acc odd;
#pragma unroll
        for (int e = 0; e < kAcc; e++) odd[e] = 0.f;
#pragma unroll
        for (int st = 0; st < kRead; st++) k[st] = operand(st);
#pragma unroll
        for (int st = 0; st < kSteps; st++) {
          if (st + kRead < kSteps) k[st + kRead] = operand(st + kRead);
          if constexpr (kBig) {
            if (st == 0)
              product<true>(s, k[st], qf[st]);
            else
              product<false>(s, k[st], qf[st]);
            if (kInt8 ? st % 2 == 0 : st % 3 == 0) bring(b + 1, kInt8 ? st / 2 : st / 3);
          } else {   // two sums, so that a product does not wait for the one before it
            if (st == 0)
#pragma unroll
              for (int e = 0; e < kAcc; e++) s[e] = 0.f;
            if (st & 1)
              odd = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[st], qf[st], odd, 0, 0, 0);
            else
              s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[st], qf[st], s, 0, 0, 0);
            if (st < kLoads) bring(b + 1, st);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (kBig) {
          product_done(s);
        } else {
#pragma unroll
          for (int e = 0; e < kAcc; e++) s[e] += odd[e];
        }
      } else {
#pragma unroll
        for (int j = 0; j < kLoads; j++) bring(b + 1, j);
      }
      forget();

      // ---- softmax.  Element e of a lane is key key_of(e) of the block, its
      // row c of row tile rh.
      const int part = lane / kRowSize, c = lane & (kRowSize - 1);
      auto key_of = [&](int e) { return kRowSize * kg + (kBig ? 8 * (e >> 2) + 4 * part + (e & 3) : 4 * part + e); };
      float weights = 0.f;
      float ksv[kInt8 ? kAcc : 1];
      auto put_p = [&]() {
        float p[kAcc];
#pragma unroll
        for (int e = 0; e < kAcc; e++) p[e] = __builtin_amdgcn_exp2f(s[e] - ref);
        float t[kAcc / 4];
#pragma unroll
        for (int e = 0; e < kAcc; e += 4) t[e / 4] = (p[e] + p[e + 1]) + (p[e + 2] + p[e + 3]);
        weights = kBig ? (t[0] + t[1 % (kAcc / 4)]) + (t[2 % (kAcc / 4)] + t[3 % (kAcc / 4)]) : t[0];
        if constexpr (kInt8) {   // V = codes * scale: the scale goes to P
#pragma unroll
          for (int e = 0; e < kAcc; e++) p[e] *= ksv[e];
        }
        // P is rounded to bf16 (like the output, 2^-9 of each weight on the
        // average); the sum keeps the unrounded weights.  Chunk of 8 keys and
        // half: with the small products the operand's keys of each 32 are
        // 4 g + i and 16 + 4 g + i.
        uint8_t* row = sh.p[kRowSize * rh + c];
#pragma unroll
        for (int e = 0; e < kAcc; e += 4) {
          const int chunk = kBig ? 4 * kg + e / 4 : 4 * (kg >> 1) + part, half = kBig ? part : kg & 1;
          *reinterpret_cast<uint2*>(row + 16 * (chunk ^ (c & 7)) + 8 * half) =
              make_uint2(pack_bf16x2(p[e], p[e + 1]), pack_bf16x2(p[e + 2], p[e + 3]));
        }
      };
      if (takes_rows) {
        const uint64_t have = static_cast<uint32_t>(uniform(static_cast<int>(have_v))) |
                              static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(have_v >> 32)))) << 32;
        if constexpr (kInt8) {
#pragma unroll
          for (int e = 0; e < kAcc; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(&sh.scl[b & 1][key_of(e)]);
            ksv[e] = v.x, ksv[e + 1] = v.y, ksv[e + 2] = v.z, ksv[e + 3] = v.w;
          }
        }
#pragma unroll
        for (int e = 0; e < kAcc; e++) s[e] *= kInt8 ? a.scale_log2 * ksv[kInt8 ? e : 0] : a.scale_log2;
        if (have != ~0ull || (b + 1) * kKeys - 1 > least) {
          const int row = min(row0 + kRowSize * rh + c, rows - 1);
          const int64_t see = static_cast<int64_t>(rq.len) - rq.n + row / a.heads;
          const int limit = static_cast<int>(see < last ? see < -1 ? -1 : see : last) - b * kKeys;
#pragma unroll
          for (int e = 0; e < kAcc; e++) {
            const int k = key_of(e);
            if (k > limit || !(have >> k & 1)) s[e] = -INFINITY;
          }
        }
        if constexpr (kInt8) {
          // a scale that is not a number has made its logits so; where it is
          // masked, the weight 0 has to stay 0
#pragma unroll
          for (int e = 0; e < kAcc; e++) ksv[e] = fabsf(ksv[e]) < INFINITY ? ksv[e] : 0.f;
        }
        if (kInSm > 0) bring(b + 1, kInQk);
        float top = s[0];
#pragma unroll
        for (int e = 1; e < kAcc; e++) top = fmaxf(top, s[e]);
        top = kBig ? half_max(top) : quad_max(top);
        if (lane < kRowSize) sh.red[kg][kRowSize * rh + c] = top;
        if (__ballot(top > ref + kSlack) && lane == 0) sh.flag[b & 1] = 1;
        if (kInSm > 1) bring(b + 1, kInQk + 1);
        put_p();
        if (kInSm > 2) bring(b + 1, kInQk + 2);
      }
      advance();
      look_up(b + 2);
      wg_barrier();   // P is whole

      if (uniform(sh.flag[b & 1])) {   // some row's maximum passed its reference: all rows take theirs
        if (takes_rows) {
          const int row = kRowSize * rh + c;
          float m = ref;
#pragma unroll
          for (int i = 0; i < kKeys / kRowSize; i++) m = fmaxf(m, sh.red[i][row]);
          const float alpha = __builtin_amdgcn_exp2f(ref - m);
          ref = m;
          sum *= alpha;
          if (kg == 0 && lane < kRowSize) sh.ref[row] = alpha;
          put_p();
        }
        wg_barrier();
#pragma unroll
        for (int j = 0; j < kRT; j++) {
          const float alpha = sh.ref[kRowSize * j + c];
#pragma unroll
          for (int i = 0; i < kLT; i++)
#pragma unroll
            for (int e = 0; e < kAcc; e++) acc[i][j][e] *= alpha;
        }
      }
      sum += weights;

      if constexpr (!kInt8) {
        // Keys that some row of the tile may not see: 0 * inf would put NaN
        // into that row.  A row that sees such a key has NaN from its logit.
        if ((b + 1) * kKeys - 1 > least && least < last) {
          for (int j = 0; j < kOwn; j++) {
            uint4* at = reinterpret_cast<uint4*>(&blk.lat[kOwn * w + j][16 * lane]);
            const uint4 v = *at;
            *at = make_uint4(finite_bf16x2(v.x), finite_bf16x2(v.y), finite_bf16x2(v.z), finite_bf16x2(v.w));
          }
          wg_barrier();
        }
      }
      forget();

      // ---- O^T += V^T P^T: the wave's latent tiles, all rows; V's operands are
      // read some steps ahead.  INT8: a row of the next block is converted
      // between the steps.
      {
        constexpr int kRead = kBig ? 4 : 3, kGroups = kKeys / kDepth;
        const int g = lane >> 4, c16 = lane & 15;
        // a transposing read gives a lane its column (latent) of four rows (keys)
        const int tr_row = kBig ? 8 * (lane >> 5) + (c16 >> 2) : 4 * g + (c16 >> 2);
        const int tr_col = (kBig ? 2 * (g & 1) : 0) + ((c16 & 3) >> 1);      // 16-byte chunk, + those of the tile
        constexpr int kTileChunks = kRowSize / 8, kBases = 8 / kTileChunks;  // the swizzle is on 8 chunks
        constexpr int kSecond = (kBig ? 4 : 16) * 2 * kLatent;               // rows of the operand's other half
        const uint8_t* base[kBases][kBig ? 2 : 1];
#pragma unroll
        for (int i = 0; i < kBases; i++)
#pragma unroll
          for (int h = 0; h < (kBig ? 2 : 1); h++)
            base[i][h] = &blk.lat[tr_row + 4 * h][128 * (kLT * kTileChunks * w / 8) +
                                                  16 * ((kTileChunks * i + tr_col) ^ swizzle(tr_row + 4 * h)) + 8 * (c16 & 1)];
        auto operand = [&](int u) {
          const int i = u % kLT, t = u / kLT;   // latent tile, keys
          const int off = 128 * (i / kBases) + kDepth * t * 2 * kLatent;
          const uint8_t* p0 = base[i % kBases][0] + off;
          const uint8_t* p1 = kBig ? base[i % kBases][kBig ? 1 : 0] + off : p0 + kSecond;
          const i32x2 v0 = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(GLM53_LDS(i16x4, p0)));
          const i32x2 v1 = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(GLM53_LDS(i16x4, p1)));
          return __builtin_bit_cast(bf16x8, make_uint4(v0[0], v0[1], v1[0], v1[1]));
        };
        auto weights_of = [&](int t, int j) {
          const int chunk = kDepth / 8 * t + part;
          return *reinterpret_cast<const bf16x8*>(sh.p[kRowSize * j + c] + 16 * (chunk ^ (c & 7)));
        };
        bf16x8 pb[kGroups][kRT], v[kPvSteps];
#pragma unroll
        for (int j = 0; j < kRT; j++) pb[0][j] = weights_of(0, j);
#pragma unroll
        for (int u = 0; u < kRead; u++) v[u] = operand(u);
#pragma unroll
        for (int u = 0; u < kPvSteps; u++) {
          const int i = u % kLT, t = u / kLT;
          if (u + kRead < kPvSteps) v[u + kRead] = operand(u + kRead);
          if (i < kRT && t + 1 < kGroups) pb[t + 1][i] = weights_of(t + 1, i);
#pragma unroll
          for (int j = 0; j < kRT; j++) {
            if constexpr (kBig)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[u], pb[t][j], acc[i][j], 0, 0, 0);
            else
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], pb[t][j], acc[i][j], 0, 0, 0);
          }
          if (u < kLoads - kInQk - kInSm) bring(b + 1, kInQk + kInSm + u);
          if (kInt8 && u < kOwn) put_row(b + 1, u);
          __builtin_amdgcn_sched_barrier(0);
        }
        static_assert(kOwn <= kPvSteps && kLoads - kInQk - kInSm <= kPvSteps, "every row has its step");
      }
    }
    loads_done();   // what was asked for past the last block

    // ---- the rows' sums and references, then the output or the partial
    wg_barrier();
    const int part = lane / kRowSize, c = lane & (kRowSize - 1);
    if (takes_rows) {
      const float l = kBig ? half_sum(sum) : quad_sum(sum);
      const int row = kRowSize * rh + c;
      if (lane < kRowSize) sh.red[kg][row] = l;
      if (kg == 0 && lane < kRowSize) sh.ref[row] = ref;
    }
    wg_barrier();
    auto sum_of = [&](int row) {
      float l = sh.red[0][row] + sh.red[1][row];
      if (!kBig) l += sh.red[2][row] + sh.red[3][row];
      return l;
    };
    LateArgs* e = late_args();
    if (!kSplit || (lo <= start && start + units <= hi)) {
      // whole rows go out: as bf16 through LDS (chunk c of row r at c ^ (r %
      // 8), so that rows fall on different banks), then each wave stores every
      // kWaves-th row
      uint8_t* os = sh.kv[0].lat[0];
#pragma unroll
      for (int j = 0; j < kRT; j++) {
        const float l = sum_of(kRowSize * j + c);
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < kLT; i++)
#pragma unroll
          for (int q = 0; q < kAcc; q += 4) {
            const Acc v = acc[i][j];
            const int lat = kRowSize * (kLT * w + i) + (kBig ? 8 * (q / 4) : 0) + 4 * part;   // of v[q]
            *reinterpret_cast<uint2*>(os + (kRowSize * j + c) * 2 * kLatent + ((2 * lat & ~15) ^ (16 * (c & 7))) + (2 * lat & 15)) =
                make_uint2(pack_bf16x2(v[q] * inv, v[q + 1] * inv), pack_bf16x2(v[q + 2] * inv, v[q + 3] * inv));
          }
      }
      wg_barrier();
      const int heads = e->heads, aligned = e->out_align16;
      const int64_t so_t = e->so_t, so_h = e->so_h;
      uint16_t* out = e->out;
      float* lse = e->lse;
      for (int j = w; j < kTM && row0 + j < rows; j += kWaves) {
        const int row = row0 + j, tok = row / heads, head = row - tok * heads;
        uint16_t* o = out + static_cast<int64_t>(rq.t0 + tok) * so_t + static_cast<int64_t>(head) * so_h;
        const uint4 v = *reinterpret_cast<const uint4*>(os + j * 2 * kLatent + ((16 * lane) ^ (16 * (j & 7))));
        if (aligned) {
          reinterpret_cast<uint4*>(o)[lane] = v;
        } else {
          reinterpret_cast<uint2*>(o)[2 * lane] = make_uint2(v.x, v.y);
          reinterpret_cast<uint2*>(o)[2 * lane + 1] = make_uint2(v.z, v.w);
        }
        if (lse && lane == 0) {
          const float l = sum_of(j);
          lse[static_cast<int64_t>(rq.t0 + tok) * heads + head] =
              l == 0.f ? -INFINITY : (sh.ref[j] + __builtin_amdgcn_logf(l)) * kLn2;
        }
      }
      if (kSplit && threadIdx.x == 0) e->shares[tile] = make_int2(-1, -1);
    } else {
      // slot 2 g: the tile began in an earlier workgroup; 2 g + 1: it begins
      // here.  In the accumulators' order: 16 bytes of each lane at a time.
      const int slot = 2 * static_cast<int>(blockIdx.x) + (lo <= start);
      float* out = e->part + static_cast<int64_t>(slot) * (kTM * kLatent);
#pragma unroll
      for (int i = 0; i < kLT; i++)
#pragma unroll
        for (int j = 0; j < kRT; j++)
#pragma unroll
          for (int q = 0; q < kAcc; q += 4) {
            const Acc v = acc[i][j];
            *reinterpret_cast<f32x4*>(out + (((kLT * w + i) * kRT + j) * (kAcc / 4) + q / 4) * 256 + 4 * lane) =
                f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]};
          }
      if (threadIdx.x < kTM) {
        const int row = threadIdx.x;
        e->ml[static_cast<int64_t>(slot) * kTM + row] = make_float2(sh.ref[row], sum_of(row));
      }
      if (lo <= start && threadIdx.x == 0) {
        const int64_t groups = min(static_cast<int>(gridDim.x), total);
        // the workgroup of the tile's last unit u: the largest g with g * total / groups <= u
        const int64_t last_unit = start + units;
        e->shares[tile] = make_int2(blockIdx.x, static_cast<int>((last_unit * groups - 1) / total));
      }
    }
    if (!kSplit) return;
  }
}

// Joins a shared tile's partials, 1 KB a job: 32 rows x 8 latents of a 64-row
// tile, 16 x 16 of the others.  kTogether
// waves take every kTogether-th partial each and join theirs through LDS (few
// tiles, whose partials are many), or each of a workgroup's four waves takes a
// job of its own.  kDeep partials are asked for at once.
template <int kTM, int kTogether>
__global__ __launch_bounds__(kTogether > 1 ? 64 * kTogether : 256) void chunk_mla_merge_kernel(const ChunkArgs a) {
  constexpr int kRowSize = ChunkShape<kTM>::kBig ? 32 : 16, kRT = kTM / kRowSize, kQuads = kRowSize == 32 ? 4 : 1;
  constexpr int kDeep = 8;
  __shared__ float acc_s[kTogether][64][4];
  __shared__ float2 ml_s[kTogether][kRowSize];
  const int tile = blockIdx.y;
  const int2 share = a.shares[tile];
  if (share.x < 0) return;
  const int w = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, part = lane / kRowSize, c = lane & (kRowSize - 1);
  const int job = kTogether > 1 ? blockIdx.x : 4 * blockIdx.x + w;
  const int j = job / kQuads % kRT;   // row tile
  const int lat = kRowSize * (job / (kQuads * kRT)) + 8 * (job % kQuads) + 4 * part;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int k0 = share.x + (kTogether > 1 ? w : 0); k0 <= share.y; k0 += kTogether * kDeep) {
    float2 ml[kDeep];
    f32x4 v[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; d++) {
      const int k = min(k0 + kTogether * d, share.y);
      const int64_t slot = 2 * static_cast<int64_t>(k) + (k == share.x);
      ml[d] = a.ml[slot * kTM + kRowSize * j + c];
      v[d] = *reinterpret_cast<const f32x4*>(a.part + slot * (kTM * kLatent) + job * 256 + 4 * lane);
    }
    float top = m;
#pragma unroll
    for (int d = 0; d < kDeep; d++) {
      if (k0 + kTogether * d > share.y) ml[d] = make_float2(-INFINITY, 0.f), v[d] = f32x4{0.f, 0.f, 0.f, 0.f};
      top = fmaxf(top, ml[d].x);
    }
    const float base = top == -INFINITY ? 0.f : top;
    const float old = __builtin_amdgcn_exp2f(m - base);
    m = top;
    l *= old;
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] *= old;
#pragma unroll
    for (int d = 0; d < kDeep; d++) {
      const float f = __builtin_amdgcn_exp2f(ml[d].x - base);
      l += f * ml[d].y;
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] += f * v[d][e];
    }
  }
  if constexpr (kTogether > 1) {
    *reinterpret_cast<f32x4*>(acc_s[w][lane]) = acc;
    if (lane < kRowSize) ml_s[w][c] = make_float2(m, l);
    __syncthreads();
    if (w) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kTogether; i++) top = fmaxf(top, ml_s[i][c].x);
    const float base = top == -INFINITY ? 0.f : top;
    m = top;
    l = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kTogether; i++) {
      const float2 ml = ml_s[i][c];
      const float f = __builtin_amdgcn_exp2f(ml.x - base);
      l += f * ml.y;
      const f32x4 v = *reinterpret_cast<const f32x4*>(acc_s[i][lane]);
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] += f * v[e];
    }
  }
  // the request of the tile
  int at = 0;
  for (int step = a.first_step; step; step >>= 1) {
    const int r = at + step;
    if (r < a.num_reqs && first_tile<kTM>(min(max(a.cu[r], 0), a.total_q), a.heads, r) <= tile) at = r;
  }
  const Request rq = request_of(a.cu[at], a.cu[at + 1], 0, a.total_q);
  const int row = (tile - first_tile<kTM>(rq.t0, a.heads, at)) * kTM + kRowSize * j + c;
  if (row >= rq.n * a.heads) return;
  const int tok = row / a.heads, head = row - tok * a.heads;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* o = a.out + static_cast<int64_t>(rq.t0 + tok) * a.so_t + static_cast<int64_t>(head) * a.so_h;
  *reinterpret_cast<uint2*>(o + lat) =
      make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  if (a.lse && lat == 0)
    a.lse[static_cast<int64_t>(rq.t0 + tok) * a.heads + head] =
        l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// Rows per tile: as many as a request's rows fill, 16, 32 or 64.
int tile_rows(int64_t total_q, int64_t num_reqs, int64_t heads) {
  const int64_t rows = num_reqs > 0 ? (total_q * heads + num_reqs - 1) / num_reqs : 0;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

int64_t tile_bound(int64_t total_q, int64_t num_reqs, int64_t heads, int tm) {
  return total_q * heads / tm + num_reqs;
}

// The split form's workspace: partials, (m, l), shares.
struct Workspace {
  int64_t part, ml, bytes;
};
Workspace workspace_of(int tm, int64_t tiles) {
  const int64_t slots = 2 * static_cast<int64_t>(num_cus());
  Workspace w;
  w.part = 0;
  w.ml = slots * tm * kLatent * 4;
  const int64_t shares = w.ml + slots * tm * 8;
  w.bytes = shares + tiles * 8;
  return w;
}

template <int kTM, bool kInt8>
int launch(ChunkArgs& a, void* workspace, hipStream_t st) {
  if (a.num_tiles > kMaxSplitTiles) {
    hipLaunchKernelGGL((chunk_mla_kernel<kTM, kInt8, false>), dim3(a.num_tiles), dim3(ChunkShape<kTM>::kThreads), 0, st, a);
  } else {
    const Workspace ws = workspace_of(kTM, a.num_tiles);
    uint8_t* p = static_cast<uint8_t*>(workspace);
    a.part = reinterpret_cast<float*>(p);
    a.ml = reinterpret_cast<float2*>(p + ws.ml);
    a.shares = reinterpret_cast<int2*>(p + ws.bytes - 8 * static_cast<int64_t>(a.num_tiles));
    hipLaunchKernelGGL((chunk_mla_kernel<kTM, kInt8, true>), dim3(num_cus()), dim3(ChunkShape<kTM>::kThreads), 0, st, a);
    // a shared tile has about CUs / tiles partials: 16 waves on a job where
    // that is many, one where it is few
    if (a.num_tiles <= 16)
      hipLaunchKernelGGL((chunk_mla_merge_kernel<kTM, 16>), dim3(2 * kTM, a.num_tiles), dim3(1024), 0, st, a);
    else
      hipLaunchKernelGGL((chunk_mla_merge_kernel<kTM, 1>), dim3(kTM / 2, a.num_tiles), dim3(256), 0, st, a);
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace
}  // namespace glm53

using namespace glm53;

extern "C" int64_t glm53_chunk_mla_workspace_bytes(int64_t total_q, int64_t num_reqs, int64_t num_heads) {
  if (total_q <= 0 || num_reqs <= 0 || num_heads <= 0) return 0;
  const int tm = tile_rows(total_q, num_reqs, num_heads);
  const int64_t tiles = tile_bound(total_q, num_reqs, num_heads, tm);
  return tiles > kMaxSplitTiles ? 0 : workspace_of(tm, tiles).bytes;
}

extern "C" int glm53_chunk_mla(const void* q, int64_t sq_t, int64_t sq_h, const void* kv_pages, int kv_is_int8,
                               int64_t page_bytes, int64_t row_bytes, int64_t num_blocks, int64_t block_size,
                               const int32_t* cu_seqlens_q, const int32_t* seq_lens, const int32_t* block_table,
                               int64_t num_reqs, int64_t bt_stride, int64_t max_blocks, int64_t total_q,
                               int64_t num_heads, double sm_scale, void* workspace, int64_t workspace_bytes,
                               void* out, int64_t so_t, int64_t so_h, float* lse, void* stream) {
  if (total_q < 0 || num_reqs < 0 || num_heads <= 0 || block_size <= 0 || max_blocks < 0 || num_blocks < 0)
    return GLM53_ERR_BAD_SHAPE;
  if (total_q == 0 || num_reqs == 0) return 0;
  const int64_t row = kv_is_int8 ? 528 : 2 * (kLatent + kRope);
  constexpr int64_t kInt = 0x7fffffff;
  if (total_q > kInt / num_heads || num_reqs >= kInt || block_size > kInt || max_blocks > kInt || num_blocks > kInt ||
      row_bytes < row || page_bytes < 0)
    return GLM53_ERR_BAD_SHAPE;
  if (!q || !out || !cu_seqlens_q || !seq_lens || (max_blocks > 0 && num_blocks > 0 && (!kv_pages || !block_table)))
    return GLM53_ERR_NULL_POINTER;
  const uintptr_t qa = reinterpret_cast<uintptr_t>(q), ka = reinterpret_cast<uintptr_t>(kv_pages),
                  oa = reinterpret_cast<uintptr_t>(out);
  if (qa % 16 || sq_t % 8 || sq_h % 8 || ka % 16 || page_bytes % 16 || row_bytes % 16 || oa % 8 || so_t % 4 || so_h % 4)
    return GLM53_ERR_MISALIGNED;
  const int tm = tile_rows(total_q, num_reqs, num_heads);
  const int64_t tiles = tile_bound(total_q, num_reqs, num_heads, tm);
  if (total_q * num_heads + num_reqs * tm > kInt) return GLM53_ERR_BAD_SHAPE;   // tile and row indexes are ints
  if (tiles <= kMaxSplitTiles) {
    if (!workspace || workspace_bytes < workspace_of(tm, tiles).bytes) return GLM53_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return GLM53_ERR_MISALIGNED;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  ChunkArgs a = {};
  a.q = static_cast<const uint16_t*>(q);
  a.sq_t = sq_t, a.sq_h = sq_h;
  a.kv = static_cast<const uint8_t*>(kv_pages);
  a.page_bytes = page_bytes, a.row_bytes = row_bytes;
  a.num_blocks = static_cast<int>(num_blocks);
  a.cu = cu_seqlens_q, a.lens = seq_lens, a.bt = block_table;
  a.bt_stride = bt_stride;
  a.max_blocks = num_blocks > 0 ? static_cast<int>(max_blocks) : 0;
  a.block_size = static_cast<int>(block_size);
  while (a.first_step < num_reqs && (a.first_step ? 2 * a.first_step : 1) < num_reqs)
    a.first_step = a.first_step ? 2 * a.first_step : 1;
  a.num_reqs = static_cast<int>(num_reqs), a.total_q = static_cast<int>(total_q), a.heads = static_cast<int>(num_heads);
  a.num_tiles = static_cast<int>(tiles);
  a.scale_log2 = static_cast<float>(sm_scale * 1.4426950408889634);
  a.out = static_cast<uint16_t*>(out);
  a.so_t = so_t, a.so_h = so_h;
  a.out_align16 = oa % 16 == 0 && so_t % 8 == 0 && so_h % 8 == 0;
  a.lse = lse;
  if (kv_is_int8) {
    if (tm == 16) return launch<16, true>(a, workspace, st);
    return tm == 32 ? launch<32, true>(a, workspace, st) : launch<64, true>(a, workspace, st);
  }
  if (tm == 16) return launch<16, false>(a, workspace, st);
  return tm == 32 ? launch<32, false>(a, workspace, st) : launch<64, false>(a, workspace, st);
}
