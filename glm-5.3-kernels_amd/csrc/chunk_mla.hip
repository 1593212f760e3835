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
// of kTM rows, which share every key they read; a tile walks its keys in
// blocks of 64.  One workgroup (4 waves for 16 or 32 rows, 8 for 64):
//   * a block's rows come into LDS (bf16 rows by direct global -> LDS loads,
//     INT8 rows through registers, converted once), two buffers, the next
//     block's loads in flight while this one is used;
//   * S^T = K Q^T: each wave takes 16 of the 64 keys (and half of the rows
//     where there are 64), its queries held in registers for the whole tile;
//   * softmax against a reference maximum that moves only when some row's
//     maximum passes it by 2^8 (the sums and products scale with it, in fp32),
//     so most blocks need one barrier between the two products;
//   * O^T += V^T P^T: each wave takes its slice of the 512 latents for all
//     rows; P goes through LDS as bf16, V is read from the same rows with
//     transposing reads.
// Few tiles (decode): the blocks of all tiles are laid end to end and cut
// into equal runs, one per workgroup; a tile that several workgroups share
// leaves fp32 partials that the merge kernel joins.  Many tiles: one
// workgroup each, longest first.
#include "glm53_common.h"

namespace glm53 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kKeys = 64;           // keys per block
constexpr int kMaxSplitTiles = 512; // most tiles whose blocks are cut into equal runs
constexpr int kPPitch = 2 * kKeys + 16;
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

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kOwn = kKeys / kWaves;      // keys of a block that a wave brings in, and takes in QK
constexpr int kLT = 32 / kWaves;          // PV: latent tiles of a wave

template <int kTM>
struct __attribute__((aligned(16))) ChunkShared {
  struct __attribute__((aligned(16))) Block {
    uint8_t lat[kKeys][2 * kLatent];   // chunk c of 16 bytes of row k at chunk c ^ swizzle(k)
    uint8_t rope[kKeys][2 * kRope];
  } kv[2];
  uint8_t p[kTM][kPPitch];             // P, keys of each 32 in the order of the V operand
  float red[kWaves][kTM];              // per wave: its keys' maximum, at the end their sum
  float ref[kTM];                      // alpha when the reference moves, at the end the reference
  float scl[2][kKeys];                 // INT8 rows' scales
  int ends[kMaxSplitTiles];            // blocks up to and with each tile
  int reqs[kMaxSplitTiles];
  int sums[kWaves];
  int flag[2];
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

__device__ __forceinline__ float quad_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Eight INT8 codes as eight bf16 (exact).
__device__ __forceinline__ uint4 codes_to_bf16(uint2 v) {
  uint32_t o[4];
  const uint32_t w[2] = {v.x, v.y};
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int32_t x = static_cast<int32_t>(w[k]);
    const float f0 = static_cast<float>((x << 24) >> 24), f1 = static_cast<float>((x << 16) >> 24);
    const float f2 = static_cast<float>((x << 8) >> 24), f3 = static_cast<float>(x >> 24);
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

// One K-step's products of four row tiles, the queries in accumulation
// registers (kAcc) or vector ones; with kFirst the sums start at 0.  In asm
// because the compiler, with nearly all 512 registers of a lane in use, copies
// the queries to vector registers before most products otherwise.  The two
// wait states before the products are what a vector instruction that wrote
// one of their operands needs; nothing but these products writes s, and
// products_done() comes before its first other use.
template <bool kFirst, bool kAcc>
__device__ __forceinline__ void four_products(f32x4 (&s)[4], bf16x8 k, bf16x8 q0, bf16x8 q1, bf16x8 q2, bf16x8 q3) {
  if constexpr (kFirst)
    asm("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %4, %5, 0\n\tv_mfma_f32_16x16x32_bf16 %1, %4, %6, 0\n\t"
        "v_mfma_f32_16x16x32_bf16 %2, %4, %7, 0\n\tv_mfma_f32_16x16x32_bf16 %3, %4, %8, 0"
        : "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
        : "v"(k), "a"(q0), "a"(q1), "a"(q2), "a"(q3));
  else if constexpr (kAcc)
    asm("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %4, %5, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %4, %6, %1\n\t"
        "v_mfma_f32_16x16x32_bf16 %2, %4, %7, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %4, %8, %3"
        : "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3])
        : "v"(k), "a"(q0), "a"(q1), "a"(q2), "a"(q3));
  else
    asm("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %4, %5, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %4, %6, %1\n\t"
        "v_mfma_f32_16x16x32_bf16 %2, %4, %7, %2\n\tv_mfma_f32_16x16x32_bf16 %3, %4, %8, %3"
        : "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3])
        : "v"(k), "v"(q0), "v"(q1), "v"(q2), "v"(q3));
}
// Wait states between a product and a vector instruction that reads it (11
// for products of this shape; 16 here).
__device__ __forceinline__ void products_done(f32x4 (&s)[4]) {
  asm volatile("s_nop 15" : "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3]));
}

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
__device__ __forceinline__ const ChunkArgs& late_args() {
  uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const ChunkArgs*)p;
}

template <int kTM, bool kInt8, bool kSplit>
__global__ __launch_bounds__(kThreads, 1) void chunk_mla_kernel(const ChunkArgs a) {
  constexpr int kRT = kTM / 16;              // row tiles
  constexpr int kSteps = kInt8 ? 16 : 18;    // K-steps of 32
  __shared__ ChunkShared<kTM> sh;

  const int w = uniform(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  // What depends on the lane alone would be kept in registers across the
  // block loop, which has none to spare: forget() makes the compiler derive it
  // anew from the lane.
  auto forget = [&]() { asm volatile("" : "+v"(lane)); };
  int g = lane >> 4, c = lane & 15;
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
      for (int step = kMaxSplitTiles / 2; step; step >>= 1) {
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
    int r, b0, b1, start = 0, units;
    Request rq;
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
      int count = 0;
      for (int i = threadIdx.x; i < a.num_reqs; i += kThreads)
        count += first_tile<kTM>(min(max(a.cu[i], 0), a.total_q), a.heads, i) <= tile;
#pragma unroll
      for (int d = 32; d; d >>= 1) count += __shfl_xor(count, d);
      if (lane == 0) sh.sums[w] = count;
      wg_barrier();
      r = -1;
#pragma unroll
      for (int i = 0; i < kWaves; i++) r += sh.sums[i];
      r = uniform(max(r, 0));
      b0 = b1 = units = 0;
    }
    rq = request_of(uniform(a.cu[r]), uniform(a.cu[r + 1]), uniform(a.lens[r]), a.total_q);
    const int rows = rq.n * a.heads;
    const int row0 = (tile - first_tile<kTM>(rq.t0, a.heads, r)) * kTM;
    if (!kSplit && (row0 < 0 || row0 >= rows)) return;   // an index between two requests
    const int last = last_key<kTM>(rq, row0, a.heads, max_pos);
    if (!kSplit) {
      units = b1 = last >= 0 ? last / kKeys + 1 : 0;
    } else if (last < 0) {
      b1 = b0;   // nothing to see: its one unit writes the zeros
    }
    // the least of the rows' last positions: keys past it are masked for some row
    const int64_t least64 = static_cast<int64_t>(rq.len) - rq.n + row0 / a.heads;
    const int least = static_cast<int>(least64 < -1 ? -1 : least64 < last ? least64 : last);

    if (kSplit) wg_barrier();   // the buffers are free (the tile before, the scan)

    // ---- bringing blocks in.  Wave w brings in the 16 keys that it takes in
    // QK.  Lane c (of each 16) looks up key 16 w + c: its page in the table,
    // one block ahead of its use, then its row's address.  A key past the
    // sequence, or whose page is not in the table or the cache, has none: the
    // cache's first row is read in its place and zeroed.
    uint2 codes[kInt8 ? kOwn : 1];
    float scale = 0.f;
    int pos = b0 * kKeys + kOwn * w + c;   // of the block that `page` is for
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
    uint32_t row_lo = 0, row_hi = 0, have = 0, have_next = 0;   // addresses; bit j: key 16 w + j has a row
    auto address = [&]() {
      const bool ok = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_blocks);
      have_next = static_cast<uint32_t>(__ballot(ok)) & 0xffff;
      const uint64_t at = reinterpret_cast<uint64_t>(a.kv) +
                          (ok ? page * static_cast<uint64_t>(a.page_bytes) + in_page * static_cast<uint64_t>(a.row_bytes) : 0);
      row_lo = static_cast<uint32_t>(at), row_hi = static_cast<uint32_t>(at >> 32);
    };
    // Step j of kSteps of bringing in block b.  With 64 rows the products
    // bound the loop, and the loads are spread over it: sent at once they
    // fill the CU's miss queue and hold up the products behind them.
    constexpr bool kSpread = kRT == 4 && !kInt8;
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
    // INT8: row j of the wave's keys of block b as bf16 into LDS (0 without a row)
    auto put_row = [&](int b, int j) {
      if constexpr (kInt8) {
        const uint2 v = have_next >> j & 1 ? codes[j] : make_uint2(0, 0);
        *reinterpret_cast<uint4*>(&sh.kv[b & 1].lat[kOwn * w + j][(16 * lane) ^ (16 * swizzle(j))]) = codes_to_bf16(v);
        if (j == kOwn - 1 && lane < kOwn) sh.scl[b & 1][kOwn * w + lane] = have_next >> lane & 1 ? scale : 0.f;
      }
    };

    if (b0 < b1) {
      look_up(b0);
      address();
      advance();
#pragma unroll
      for (int j = 0; j < kSteps; j++) bring(b0, j);
      look_up(b0 + 1);
    }

    // ---- the queries: row c of row tile rt (rows past the last: the last,
    // not stored).  Every wave needs all of them, so they come through LDS
    // once, in the buffer that the second block will take, laid out like keys:
    // wave w brings in every fourth row.
    bf16x8 qf[kRT][kSteps];
    {
      auto& qs = sh.kv[(b0 + 1) & 1];
      constexpr int kMine = kTM / kWaves;
      const int row = min(row0 + kWaves * min(c, kMine - 1) + w, rows - 1);
      const int tok = row / a.heads, head = row - tok * a.heads;
      const uint64_t at = reinterpret_cast<uint64_t>(a.q + static_cast<int64_t>(rq.t0 + tok) * a.sq_t +
                                                     static_cast<int64_t>(head) * a.sq_h);
      const int at_lo = static_cast<int>(at), at_hi = static_cast<int>(at >> 32);
#pragma unroll
      for (int j = 0; j < kMine; j++) {
        const uint64_t from = static_cast<uint32_t>(__builtin_amdgcn_readlane(at_lo, j)) |
                              static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(at_hi, j))) << 32;
        const int key = kWaves * j + w;
        load_lds16(lds_offset(qs.lat[key]), reinterpret_cast<const uint8_t*>(from), 16 * (lane ^ swizzle(key)));
        if constexpr (!kInt8) {
          if (lane < 8)
            load_lds16(lds_offset(qs.rope[key]), reinterpret_cast<const uint8_t*>(from),
                       2 * kLatent + 16 * (lane ^ swizzle(key)));
        }
      }
      loads_done();   // the queries, and the first block's rows
      wg_barrier();
#pragma unroll
      for (int rt = 0; rt < kRT; rt++) {
        const int key = 16 * rt + c, sw = swizzle(c);
#pragma unroll
        for (int st = 0; st < kSteps; st++) {
          const uint8_t* from = st < 16 ? qs.lat[key] + 16 * ((4 * (st & 1) + g) ^ sw) + 128 * (st >> 1)
                                        : qs.rope[key] + 16 * ((4 * (st - 16) + g) ^ sw);
          qf[rt][st] = *reinterpret_cast<const bf16x8*>(from);
        }
      }
    }
    f32x4 acc[kLT][kRT];
#pragma unroll
    for (int i = 0; i < kLT; i++)
#pragma unroll
      for (int j = 0; j < kRT; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref[kRT], sum[kRT];
#pragma unroll
    for (int rt = 0; rt < kRT; rt++) ref[rt] = -INFINITY, sum[rt] = 0.f;
    if (b0 < b1) {
#pragma unroll
      for (int j = 0; j < kOwn; j++) put_row(b0, j);
    }
    if (threadIdx.x == 0) sh.flag[0] = sh.flag[1] = 0;

    for (int b = b0; b < b1; b++) {
      loads_done();   // this wave's rows of block b
      wg_barrier();   // nobody reads the other buffer, P or the maxima any more
      have = have_next;
      auto& blk = sh.kv[b & 1];
      forget();
      g = lane >> 4, c = lane & 15;
      if (!kInt8 && have != 0xffff) {
        for (int j = 0; j < kOwn; j++)
          if (!(have >> j & 1)) {
            *reinterpret_cast<uint4*>(&blk.lat[kOwn * w + j][16 * lane]) = make_uint4(0, 0, 0, 0);
            if (lane < 8) *reinterpret_cast<uint4*>(&blk.rope[kOwn * w + j][16 * lane]) = make_uint4(0, 0, 0, 0);
          }
      }
      if (w == 0 && lane == 0) sh.flag[(b + 1) & 1] = 0;

      // ---- S^T = K Q^T: keys 16 w + 4 g + i of the block, rows c.  Each
      // K-step's operand is read kAhead steps before its products, and between
      // the steps a row of the next block is asked for.
      f32x4 s[kRT];
      if constexpr (kRT != 4) {
#pragma unroll
        for (int rt = 0; rt < kRT; rt++) s[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      address();   // after the last block: no rows, the cache's first in their place
      {
        constexpr int kAhead = 5;
        const int key = kOwn * w + c, sw = swizzle(c);
        const uint8_t* even = blk.lat[key] + 16 * (g ^ sw);
        const uint8_t* odd = blk.lat[key] + 16 * ((4 + g) ^ sw);
        const uint8_t* rope = blk.rope[key];
        auto operand = [&](int st) {
          return *reinterpret_cast<const bf16x8*>(st < 16 ? (st & 1 ? odd : even) + 128 * (st >> 1)
                                                          : rope + 16 * ((4 * (st - 16) + g) ^ sw));
        };
        bf16x8 k[kSteps];
#pragma unroll
        for (int st = 0; st < kAhead; st++) k[st] = operand(st);
#pragma unroll
        for (int st = 0; st < kSteps; st++) {
          if (st + kAhead < kSteps) k[st + kAhead] = operand(st + kAhead);
          if constexpr (kRT == 4) {
            if (st == 0)
              four_products<true, true>(s, k[st], qf[0][st], qf[1][st], qf[2][st], qf[3][st]);
            else if (st < 16)
              four_products<false, true>(s, k[st], qf[0][st], qf[1][st], qf[2][st], qf[3][st]);
            else
              four_products<false, false>(s, k[st], qf[0][st], qf[1][st], qf[2][st], qf[3][st]);
          } else {
#pragma unroll
            for (int rt = 0; rt < kRT; rt++)
              s[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[st], qf[rt][st], s[rt], 0, 0, 0);
          }
          if (!kSpread || st % 2 == 0) bring(b + 1, kSpread ? st / 2 : st);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (kRT == 4) products_done(s);
      }
      if (kSpread) bring(b + 1, 9), bring(b + 1, 10);

      forget();
      g = lane >> 4, c = lane & 15;
      const bool masked = (b + 1) * kKeys - 1 > least || have != 0xffff;   // uniform
      float ksv[4] = {1.f, 1.f, 1.f, 1.f};
      if constexpr (kInt8) {
        const float4 ks = *reinterpret_cast<const float4*>(&sh.scl[b & 1][kOwn * w + 4 * g]);
        ksv[0] = ks.x, ksv[1] = ks.y, ksv[2] = ks.z, ksv[3] = ks.w;
      }
#pragma unroll
      for (int rt = 0; rt < kRT; rt++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[rt][i] *= kInt8 ? a.scale_log2 * ksv[i] : a.scale_log2;
      if (masked) {
#pragma unroll
        for (int rt = 0; rt < kRT; rt++) {
          const int row = min(row0 + 16 * rt + c, rows - 1);
          const int64_t see = static_cast<int64_t>(rq.len) - rq.n + row / a.heads;
          const int limit = static_cast<int>(see < last ? see < -1 ? -1 : see : last) - b * kKeys;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int k = 4 * g + i;
            if (kOwn * w + k > limit || !(have >> k & 1)) s[rt][i] = -INFINITY;
          }
        }
      }
      float top[kRT], mine = 0.f;
      bool moved = false;
#pragma unroll
      for (int rt = 0; rt < kRT; rt++) {
        top[rt] = quad_max(fmaxf(fmaxf(s[rt][0], s[rt][1]), fmaxf(s[rt][2], s[rt][3])));
        moved |= top[rt] > ref[rt] + kSlack;
        if (g == rt) mine = top[rt];
      }
      if (lane < kTM) sh.red[w][lane] = mine;   // row 16 g + c
      if (__ballot(moved) && lane == 0) sh.flag[b & 1] = 1;

      // P of this wave's keys, against the reference (0 where a row has seen nothing)
      float part[kRT];
      auto put_p = [&]() {
#pragma unroll
        for (int rt = 0; rt < kRT; rt++) {
          const float m = ref[rt] == -INFINITY ? 0.f : ref[rt];
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; i++) p[i] = __builtin_amdgcn_exp2f(s[rt][i] - m);
          part[rt] = (p[0] + p[1]) + (p[2] + p[3]);
          if constexpr (kInt8) {
            // V = codes * scale: the scale goes to P, which a masked key has as 0 whatever its scale is
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = s[rt][i] == -INFINITY ? 0.f : p[i] * ksv[i];
          }
          // P is rounded to bf16 (2^-9 of each weight on the average, like the
          // output's own rounding); the sum keeps the unrounded weights
          *reinterpret_cast<uint2*>(&sh.p[16 * rt + c][64 * (w >> 1) + 16 * g + 8 * (w & 1)]) =
              make_uint2(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]));
        }
      };
      put_p();
      if (kSpread) bring(b + 1, 11), bring(b + 1, 12);
      advance();
      look_up(b + 2);
      wg_barrier();   // P is whole; every wave's rows are there

      if (uniform(sh.flag[b & 1])) {   // some row's maximum passed its reference: all rows take theirs
#pragma unroll
        for (int rt = 0; rt < kRT; rt++) {
          const int row = 16 * rt + c;
          float m = ref[rt];
#pragma unroll
          for (int i = 0; i < kWaves; i++) m = fmaxf(m, sh.red[i][row]);
          const float alpha = __builtin_amdgcn_exp2f(ref[rt] - (m == -INFINITY ? 0.f : m));
          ref[rt] = m;
          sum[rt] *= alpha;
#pragma unroll
          for (int i = 0; i < kLT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][rt][e] *= alpha;
        }
        put_p();
        wg_barrier();
      }
#pragma unroll
      for (int rt = 0; rt < kRT; rt++) sum[rt] += part[rt];

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
      g = lane >> 4, c = lane & 15;
      // ---- O^T += V^T P^T: latents 16 (kLT w + i) + 4 g + e, rows 16 j + c;
      // V's operands two steps ahead.  INT8: a row of the next block is
      // converted between the steps.
      {
        constexpr int kPv = 2 * kLT, kAhead = 3;
        const int tr_row = 4 * g + (c >> 2), tr_sw = swizzle(tr_row);
        const uint8_t* vr[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
          vr[i] = &blk.lat[tr_row][256 * w + 16 * ((2 * i + ((c & 3) >> 1)) ^ tr_sw) + 8 * (c & 1)];
        auto operand = [&](int u) {
          const uint8_t* p = vr[u & 3] + 128 * (u >> 2 & 1) + 32 * 2 * kLatent * (u >> 3);
          const i32x2 v0 = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(GLM53_LDS(i16x4, p)));
          const i32x2 v1 = __builtin_bit_cast(
              i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(GLM53_LDS(i16x4, p + 16 * 2 * kLatent)));
          return __builtin_bit_cast(bf16x8, make_uint4(v0[0], v0[1], v1[0], v1[1]));
        };
        bf16x8 pb[2][kRT], v[kPv];
#pragma unroll
        for (int j = 0; j < kRT; j++) pb[0][j] = *reinterpret_cast<const bf16x8*>(&sh.p[16 * j + c][16 * g]);
#pragma unroll
        for (int u = 0; u < kAhead; u++) v[u] = operand(u);
#pragma unroll
        for (int u = 0; u < kPv; u++) {
          if (u + kAhead < kPv) v[u + kAhead] = operand(u + kAhead);
          if (u >= kLT - kRT && u < kLT) {
            const int j = u - (kLT - kRT);
            pb[1][j] = *reinterpret_cast<const bf16x8*>(&sh.p[16 * j + c][64 + 16 * g]);
          }
#pragma unroll
          for (int j = 0; j < kRT; j++)
            acc[u % kLT][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], pb[u / kLT][j], acc[u % kLT][j], 0, 0, 0);
          if (kSpread && u < 5) bring(b + 1, 13 + u);
          put_row(b + 1, u);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    loads_done();   // what the last block asked for

    // ---- the rows' sums and references, then the output or the partial
    wg_barrier();
#pragma unroll
    for (int rt = 0; rt < kRT; rt++) {
      const float l = quad_sum(sum[rt]);
      if (g == 0) sh.red[w][16 * rt + c] = l;
      if (w == 0 && g == 0) sh.ref[16 * rt + c] = ref[rt];
    }
    wg_barrier();
    const ChunkArgs& e = late_args();
    if (!kSplit || (lo <= start && start + units <= hi)) {
      // whole rows go out: the row tiles as bf16 through LDS (8 bytes of row
      // c at 16-byte chunk ^ (c % 8), so that rows fall on different banks),
      // then each wave stores every fourth row
      uint8_t(*os)[2 * kLatent] = sh.kv[0].lat;
#pragma unroll
      for (int j = 0; j < kRT; j++) {
        const float l = (sh.red[0][16 * j + c] + sh.red[1][16 * j + c]) + (sh.red[2][16 * j + c] + sh.red[3][16 * j + c]);
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < kLT; i++) {
          const f32x4 v = acc[i][j];
          *reinterpret_cast<uint2*>(&os[16 * j + c][((32 * (kLT * w + i) + 16 * (g >> 1)) ^ (16 * (c & 7))) + 8 * (g & 1)]) =
              make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
        }
      }
      wg_barrier();
      for (int j = w; j < kTM && row0 + j < rows; j += kWaves) {
        const int row = row0 + j, tok = row / e.heads, head = row - tok * e.heads;
        uint16_t* o = e.out + static_cast<int64_t>(rq.t0 + tok) * e.so_t + static_cast<int64_t>(head) * e.so_h;
        const uint4 v = *reinterpret_cast<const uint4*>(&os[j][(16 * lane) ^ (16 * (j & 7))]);
        if (e.out_align16) {
          reinterpret_cast<uint4*>(o)[lane] = v;
        } else {
          reinterpret_cast<uint2*>(o)[2 * lane] = make_uint2(v.x, v.y);
          reinterpret_cast<uint2*>(o)[2 * lane + 1] = make_uint2(v.z, v.w);
        }
        if (e.lse && lane == 0) {
          const float l = (sh.red[0][j] + sh.red[1][j]) + (sh.red[2][j] + sh.red[3][j]);
          e.lse[static_cast<int64_t>(rq.t0 + tok) * e.heads + head] =
              l == 0.f ? -INFINITY : (sh.ref[j] + __builtin_amdgcn_logf(l)) * kLn2;
        }
      }
      if (kSplit && threadIdx.x == 0) e.shares[tile] = make_int2(-1, -1);
    } else {
      // slot 2 g: the tile began in an earlier workgroup; 2 g + 1: it begins here
      const int slot = 2 * static_cast<int>(blockIdx.x) + (lo <= start);
      float* part = e.part + static_cast<int64_t>(slot) * (kTM * kLatent);
#pragma unroll
      for (int i = 0; i < kLT; i++)
#pragma unroll
        for (int j = 0; j < kRT; j++)
          *reinterpret_cast<f32x4*>(part + ((kLT * w + i) * kRT + j) * 256 + 4 * lane) = acc[i][j];
      if (threadIdx.x < kTM) {
        const int row = threadIdx.x;
        e.ml[static_cast<int64_t>(slot) * kTM + row] =
            make_float2(sh.ref[row], (sh.red[0][row] + sh.red[1][row]) + (sh.red[2][row] + sh.red[3][row]));
      }
      if (lo <= start && threadIdx.x == 0) {
        const int64_t groups = min(static_cast<int>(gridDim.x), total);
        // the workgroup of the tile's last unit u: the largest g with g * total / groups <= u
        const int64_t last_unit = start + units;
        e.shares[tile] = make_int2(blockIdx.x, static_cast<int>((last_unit * groups - 1) / total));
      }
    }
    if (!kSplit) return;
  }
}

// Joins a shared tile's partials, 16 rows x 16 latents a job.  kTogether
// waves take every kTogether-th partial each and join theirs through LDS (few
// tiles, whose partials are many), or each of a workgroup's four waves takes a
// job of its own.  kDeep partials are asked for at once.
template <int kTM, int kTogether>
__global__ __launch_bounds__(kTogether > 1 ? 64 * kTogether : 256) void chunk_mla_merge_kernel(const ChunkArgs a) {
  constexpr int kRT = kTM / 16, kDeep = 8;
  __shared__ float acc_s[kTogether][64][4];
  __shared__ float2 ml_s[kTogether][16];
  const int tile = blockIdx.y;
  const int2 share = a.shares[tile];
  if (share.x < 0) return;
  const int w = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int job = kTogether > 1 ? blockIdx.x : 4 * blockIdx.x + w;
  const int j = job % kRT, lt = job / kRT;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int k0 = share.x + (kTogether > 1 ? w : 0); k0 <= share.y; k0 += kTogether * kDeep) {
    float2 ml[kDeep];
    f32x4 v[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; d++) {
      const int k = min(k0 + kTogether * d, share.y);
      const int64_t slot = 2 * static_cast<int64_t>(k) + (k == share.x);
      ml[d] = a.ml[slot * kTM + 16 * j + c];
      v[d] = *reinterpret_cast<const f32x4*>(a.part + slot * (kTM * kLatent) + (lt * kRT + j) * 256 + 4 * lane);
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
    if (g == 0) ml_s[w][c] = make_float2(m, l);
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
  for (int step = kMaxSplitTiles / 2; step; step >>= 1) {
    const int r = at + step;
    if (r < a.num_reqs && first_tile<kTM>(min(max(a.cu[r], 0), a.total_q), a.heads, r) <= tile) at = r;
  }
  const Request rq = request_of(a.cu[at], a.cu[at + 1], 0, a.total_q);
  const int row = (tile - first_tile<kTM>(rq.t0, a.heads, at)) * kTM + 16 * j + c;
  if (row >= rq.n * a.heads) return;
  const int tok = row / a.heads, head = row - tok * a.heads;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* o = a.out + static_cast<int64_t>(rq.t0 + tok) * a.so_t + static_cast<int64_t>(head) * a.so_h;
  *reinterpret_cast<uint2*>(o + 16 * lt + 4 * g) =
      make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  if (a.lse && lt == 0 && g == 0)
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
    hipLaunchKernelGGL((chunk_mla_kernel<kTM, kInt8, false>), dim3(a.num_tiles), dim3(kThreads), 0, st, a);
  } else {
    const Workspace ws = workspace_of(kTM, a.num_tiles);
    uint8_t* p = static_cast<uint8_t*>(workspace);
    a.part = reinterpret_cast<float*>(p);
    a.ml = reinterpret_cast<float2*>(p + ws.ml);
    a.shares = reinterpret_cast<int2*>(p + ws.bytes - 8 * static_cast<int64_t>(a.num_tiles));
    hipLaunchKernelGGL((chunk_mla_kernel<kTM, kInt8, true>), dim3(num_cus()), dim3(kThreads), 0, st, a);
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
