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
// its keys in blocks of 32.  A workgroup is eight waves, two per SIMD, of two
// kinds, so that each kind's big operand stays in its registers and one
// kind's products run beside the other's vector work:
//   * waves 0 .. 3, rows: S^T = K Q^T of block n + 1 with the queries in
//     registers (wave w: keys 16 (w & 1) .. + 16, row half w >> 1; of a 16-row
//     tile waves 0 and 1 alone), then its softmax;
//   * waves 4 .. 7, latents: O^T += V^T P^T of block n, 128 of the 512 latents
//     each with the output in registers, and the loads.  bf16 rows come into a
//     ring of four blocks in LDS by direct global -> LDS loads, three blocks
//     ahead; INT8 rows as they are, four ahead, converted to bf16 once, two
//     blocks before their use as V, by waves of both kinds.  Nothing waits for memory but the count of
//     outstanding loads, once a block: the block table's entries come ahead too.
// The softmax goes against a row's reference, which stays until a logit passes
// it by 2^16 (in the first block, and seldom after it): then the block is
// weighted again with the row's maximum for a reference, and the output is
// rescaled.  So a block costs one barrier, and the two waves that share a row
// exchange their maxima only then.  Sums, output and references are fp32.  P
// goes through LDS as bf16; V is read from the rows that served as K, with
// transposing reads.
// Few tiles (decode): the blocks of all tiles are laid end to end and cut
// into equal runs, one per workgroup; a tile that several workgroups share
// leaves fp32 partials that the merge kernel joins.  Many tiles: one
// workgroup each, longest first.
//
// Measured (inputs that no cache holds):
//   * long chunks are bound by the products and the clock that the card holds
//     beside them: 2048 tokens of 16 heads on 16k, 895 - 968 us, 1130 - 1220
//     TFLOP/s (a large library product of plain matrices: 1225 - 1344).  A
//     block of 32 keys and 64 rows takes 1900 cycles for 1088 of products a
//     SIMD and 590 of LDS;
//   * INT8 prompts also by the conversion, 12 instructions for 8 codes: 1234
//     tokens of 20 heads in five requests, 145 us, 620 TFLOP/s;
//   * bf16 decode by memory: one request on 128k 41 us, 33 of them this kernel
//     (4.6 TB/s with its start, 6.5 in its loop), 24 requests of up to four
//     tokens 46 us; INT8 decode by the conversion and LDS (3.9 TB/s, 64 ragged
//     requests 77 us);
//   * small calls by their start: about 8 us of dependent loads (lengths,
//     table, rows), scan and first block, then 4 for the merge's launch.
#include <math.h>

#include <type_traits>

#include "glm53_common.h"

namespace glm53 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kKeys = 32;           // keys per block
constexpr int kMaxSplitTiles = 512; // most tiles whose blocks are cut into equal runs
// Five INT8 prompts took 185 us with 2 here, 166 with 4, 154 with 7 and 10; 24
// requests of four tokens 50, 49, 46 and 45.
constexpr int kTileCost = 10;       // what starting and ending a tile costs, in blocks
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kSlack = 16.f;      // how far (log2) a logit may pass its row's reference

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
  Divider by_block, by_heads;
  int num_reqs;
  int first_step;  // of a binary search over the requests: the largest power of two below num_reqs, or 0
  int total_q;
  int heads;
  int num_tiles;   // bound: tile indexes are below it
  float scale_log2;
  uint32_t flip;   // a negative scale: the sign bits of two bf16, for the queries
  uint16_t* out;
  int64_t so_t, so_h;
  int out_align16; // out rows 16-byte aligned (else 8)
  float* lse;      // [total_q][heads], or null
  float* part;     // [2 * workgroups] slots of kTM x 512, accumulator order
  float2* ml;      // [2 * workgroups][kTM]: reference maximum (log2) and sum
  int4* shares;    // [num_tiles]: of a shared tile its first and last workgroup, its first row over all
                   // tokens and its rows, or -1
};

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kHalf = 4;                  // waves of a kind
constexpr int kOwn = kKeys / kHalf;       // rows of a block that a latent wave brings in

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

// Products of PV: 32 latents x 32 rows x 16 keys, or 16 x 16 x 32 of a 16-row tile.
template <int kTM>
struct ChunkShape {
  static constexpr bool kBig = kTM >= 32;
};

// Row m of wave y's latent tile i: tiles of 32 are two runs of 16, 64 apart.
__device__ __forceinline__ int latent_of(int y, int i, int m) { return 128 * y + 16 * i + (m & 15) + 64 * (m >> 4); }

template <int kTM, bool kInt8>
struct __attribute__((aligned(16))) ChunkShared {
  static constexpr int kBufs = kInt8 ? 3 : 4;
  struct __attribute__((aligned(16))) Bf16Block {
    uint8_t lat[kKeys][2 * kLatent];   // chunk c of 16 bytes of row k at chunk c ^ swizzle(k)
    uint8_t rope[kKeys][2 * kRope];    // chunk c of row k at chunk c ^ rope_swizzle(k)
  };
  struct __attribute__((aligned(16))) Int8Block {
    uint8_t lat[kKeys][2 * kLatent];
  };
  std::conditional_t<kInt8, Int8Block, Bf16Block> kv[kBufs];
  uint8_t raw[kInt8 ? 3 : 0][kKeys][kLatent];   // INT8 rows as they are in the cache
  float raw_scale[kInt8 ? 3 : 0][kKeys];
  float4 scl[kInt8 ? 3 : 0][kKeys];             // what a key's scale s = f d comes to: scale_log2 s, log2 d, 1 / d, f
  uint8_t p[2][kTM][2 * kKeys];        // P, chunk c of 16 bytes of row r at c ^ (r / 4 % 4)
  int32_t page[kHalf * 64];            // block table entries of the coming blocks
  float red[2][kTM];                   // per key half: maxima; at the end the sums
  float alpha[kTM];                    // what new references scale the output with; at the end the references
  int ends[kMaxSplitTiles];            // blocks up to and with each tile
  int reqs[kMaxSplitTiles];
  uint8_t have[8][kHalf];              // bit j of byte y: key 8 y + j of the block has a row
  int again[2];                        // the last (odd, even) block that is weighted again
  int sums[kWaves], tiles[kWaves];
  struct __attribute__((aligned(16))) {
    int tile, start, end, req, t0, n, len;
  } first;                             // the first tile, its units and its request
};

__device__ __forceinline__ void wg_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// At most n loads that this wave sent are still on their way.
template <int n>
__device__ __forceinline__ void loads_left() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)(p)));
}

// 16 bytes per lane from base + off to LDS at dst + 16 * lane, and the same
// for off2, ... at dst + 1024 + 16 * lane, ...  Written in asm so that the
// compiler does not wait for it before other LDS reads; loads_left() and a
// barrier come before the first read of what it brings.  (m0 needs a wait
// state before its use, an SGPR from v_readlane five.  The compiler keeps m0
// out of clobber lists and sets it before each use of its own; nothing else
// here uses it.)
__device__ __forceinline__ void load_lds16(uint32_t dst, const uint8_t* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base)
               : "memory");
}
__device__ __forceinline__ void load_lds16_2(uint32_t dst, const uint8_t* base, uint32_t off, uint32_t off2) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
      "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3" ::"s"(dst),
      "v"(off), "v"(off2), "s"(base)
      : "memory", "scc");
}
__device__ __forceinline__ void load_lds16_at(uint32_t dst, const uint8_t* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(p) : "memory");
}

// 4 bytes per lane to LDS at dst + 4 * lane
__device__ __forceinline__ void load_lds4(uint32_t dst, const void* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_lds4_at(uint32_t dst, const void* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(p) : "memory");
}

// Swizzles of a row's 16-byte chunks, on the low bits of the chunk's index, for
// LDS passes of 256 bytes.  The row's place among its four, i, goes to bits 1
// and 2, its four q to bits 3 and 0:
//   * a transposing read takes pairs of chunks of four rows, of 32 lanes either
//     both pairs (eight chunks apart) of one q or the same pair of two q's
//     (0 and 1, or 2 and 3): i, the pair's bit 3 and q's bit 3 tell them apart;
//   * the K operand's 16-byte reads take chunk 4 k + g of row 4 q + i in lane
//     16 g + 4 q + i, and a pass serves lanes of q = 0, 3 and, from the next g,
//     1, 2 (or the reverse): g differs in bit 0, where only 0 and 3, and only 1
//     and 2, differ.
__device__ __forceinline__ int swizzle(int key) {
  return ((key >> 2 ^ key >> 3) & 1) << 3 | (key & 3) << 1 | (key >> 3 & 1);
}
// Rotary parts are 128 bytes: two rows a pass's width.
__device__ __forceinline__ int rope_swizzle(int key) { return key >> 1 & 7; }

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

// Inclusive sum over the wave: within rows of 16 lanes by shifts, then the last
// lane of row 0 (2) into row 1 (3) and that of row 1 into rows 2 and 3.
template <int kCtrl, int kRows>
__device__ __forceinline__ int add_from(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, true);
}
__device__ __forceinline__ int wave_scan(int v) {
  v = add_from<0x111, 0xf>(v);
  v = add_from<0x112, 0xf>(v);
  v = add_from<0x114, 0xf>(v);
  v = add_from<0x118, 0xf>(v);
  v = add_from<0x142, 0xa>(v);
  return add_from<0x143, 0xc>(v);
}

// Eight INT8 codes as eight bf16 (exact): 12 instructions, all at the full rate.
__device__ __forceinline__ uint4 codes_to_bf16(uint2 v) {
  uint32_t o[4];
  const uint32_t w[2] = {v.x, v.y};
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int32_t x = static_cast<int32_t>(w[k]);
    const float f0 = static_cast<float>((x << 24) >> 24), f1 = static_cast<float>((x << 16) >> 24);
    const float f2 = static_cast<float>((x << 8) >> 24), f3 = static_cast<float>(x >> 24);
    // small whole numbers: the bf16 is the high half of the fp32
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
__device__ __forceinline__ int last_key(const Request& r, int row0, int heads, const Divider& by_heads, int max_pos) {
  const int rows = r.n * heads;
  const int last_row = min(row0 + kTM, rows) - 1;
  const int64_t k = static_cast<int64_t>(r.len) - r.n + divide(last_row, by_heads);
  return k < 0 ? -1 : static_cast<int>(k < max_pos ? k : max_pos - 1);
}

// The arguments of the kernel's first loads lead (they come preloaded in
// registers), the others follow in a struct this many bytes later.
constexpr int kLeading = 24;

// The kernel's arguments read where they are used, instead of being kept in
// scalar registers from the start.
typedef const __attribute__((address_space(4))) ChunkArgs LateArgs;
__device__ __forceinline__ LateArgs* late_args() {
  uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr() + kLeading;
  asm volatile("" : "+s"(p));
  return (LateArgs*)p;
}

// Brings the arguments into the scalar cache (a line of 64 bytes each), while
// something else is waited for.
__device__ __forceinline__ void touch_args() {
  static_assert(sizeof(ChunkArgs) + kLeading > 192 && sizeof(ChunkArgs) + kLeading <= 256, "four lines");
  uint32_t x, y, z;
  asm volatile(
      "s_load_dword %0, %3, 0x40\n\ts_load_dword %1, %3, 0x80\n\ts_load_dword %2, %3, 0xc0\n\ts_waitcnt lgkmcnt(0)"
      : "=&s"(x), "=&s"(y), "=&s"(z)
      : "s"(__builtin_amdgcn_kernarg_segment_ptr()));
}

// kRuns: pages of a multiple of eight rows, so that the eight rows of a block
// that a wave brings in lie behind one another in one page.
template <int kTM, bool kInt8, bool kSplit, bool kRuns>
__global__ __launch_bounds__(kThreads, 1) void chunk_mla_kernel(const int32_t* cu, const int32_t* lens, int num_reqs,
                                                                 int total_q, const ChunkArgs a) {
  using Shared = ChunkShared<kTM, kInt8>;
  constexpr bool kBig = ChunkShape<kTM>::kBig;
  constexpr int kRQ = kTM == 64 ? 2 : 1;           // QK: row tiles (of 16) of a wave
  constexpr int kSteps = kInt8 ? 16 : 18;          // QK: K-steps of 32
  constexpr int kSize = kBig ? 32 : 16;            // PV: rows and latents of a product
  constexpr int kRT = kTM / kSize, kLT = 128 / kSize;   // PV: row and latent tiles of a wave
  constexpr int kDepth = kBig ? 16 : 32;           // PV: keys of a product
  constexpr int kPvSteps = kLT * kKeys / kDepth;
  constexpr int kBufs = Shared::kBufs;
  constexpr int kAhead = kInt8 ? 4 : 3;            // blocks between a row's load and its use as V
  constexpr int kEarly = kAhead - 1;               // blocks that are asked for before the loop
  constexpr int kRowLoads = kInt8 ? 5 : 9;         // loads a latent wave sends per block for rows,
  constexpr int kLoads = kRowLoads + !kRuns;       // and with those for table entries
  using Acc = std::conditional_t<kBig, f32x16, f32x4>;
  constexpr int kAcc = kBig ? 16 : 4;
  __shared__ Shared sh;

  const int w = uniform(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.block_size;
  const int max_pos = static_cast<int>(cap < 0x7fffff00 ? cap : 0x7fffff00);   // a block's positions stay ints

  // ---- which blocks of which tiles are this workgroup's
  int r = 0, start = 0, end = 0;   // the tile's request and units
  Request rq = {};
  int tile, lo = 0, hi = 0, each = 0, more = 0;   // the first `more` of the runs are each + 1 units long
  if (kSplit) {
    constexpr int kTiles = kMaxSplitTiles / kThreads;   // tiles of a thread
    int units[kTiles], req[kTiles], sum = 0;
    Request of[kTiles];
    int* cu_s = reinterpret_cast<int*>(&sh.kv[0]);      // cu, then lens
    int* len_s = cu_s + kMaxSplitTiles + 16;
    // (both loads at once, and with them the arguments that come into use later)
    static_assert(kMaxSplitTiles <= kThreads, "a request a thread");
    const int rc = min(static_cast<int>(threadIdx.x), num_reqs), rl = min(static_cast<int>(threadIdx.x), num_reqs - 1);
    const int cu_r = cu[rc], len_r = lens[rl], cu_end = cu[num_reqs];
    touch_args();
    cu_s[rc] = min(max(cu_r, 0), total_q);
    len_s[rl] = len_r;
    if (threadIdx.x == 0) cu_s[num_reqs] = min(max(cu_end, 0), total_q);
    wg_barrier();
#pragma unroll
    for (int k = 0; k < kTiles; k++) {
      const int t = static_cast<int>(threadIdx.x) * kTiles + k;
      int at = 0;                                       // the last request that starts at or before tile t
      for (int step = a.first_step; step; step >>= 1) {
        const int r = at + step;
        if (r < num_reqs && first_tile<kTM>(cu_s[r], a.heads, r) <= t) at = r;
      }
      const Request rq = request_of(cu_s[at], cu_s[at + 1], len_s[at], total_q);
      const int row0 = (t - first_tile<kTM>(rq.t0, a.heads, at)) * kTM;
      req[k] = at;
      of[k] = rq;
      units[k] = 0;
      if (t < a.num_tiles && row0 >= 0 && row0 < rq.n * a.heads)
        units[k] = kTileCost + max(1, last_key<kTM>(rq, row0, a.heads, a.by_heads, max_pos) / kKeys + 1);
      sum += units[k];
    }
    int upto = wave_scan(sum);                          // inclusive
    int filled = 0;
#pragma unroll
    for (int k = 0; k < kTiles; k++) filled += __popcll(__ballot(units[k] > 0));
    if (lane == 63) sh.sums[w] = upto, sh.tiles[w] = filled;
    wg_barrier();
    int before = 0, tiles = 0, total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
      const int s = sh.sums[i];
      if (i < w) before += s;
      total += s;
      tiles += sh.tiles[i];
    }
    total = uniform(total), tiles = uniform(tiles);
    if (total == 0) {
      if (blockIdx.x == 0)
        for (int t = threadIdx.x; t < a.num_tiles; t += kThreads) a.shares[t].x = -1;
      return;   // uniform over the workgroup
    }
    // A run of u blocks takes u times a block's time, and its partial (written,
    // read, joined) kTM / 1024 of that: the sum of both is least with
    // sqrt(total * 1024 / kTM) runs (one INT8 request on 2k: 15.9, 15.5 and 14.9
    // us with 256, 512 and 1024 there; with 2048 one on 19k takes 25.8 instead
    // of 24.5).  No fewer than tiles: those come without partials.
    const int best = max(tiles, static_cast<int>(sqrtf(static_cast<float>(total) * (1024 / kTM))));
    const int groups = min(min(static_cast<int>(gridDim.x), total), best), g = blockIdx.x;
    if (g >= groups) return;
    each = static_cast<uint32_t>(total) / static_cast<uint32_t>(groups), more = total - each * groups;
    lo = g * each + min(g, more), hi = lo + each + (g < more);
    int upto_t = before + upto - sum;
#pragma unroll
    for (int k = 0; k < kTiles; k++) {
      const int t = static_cast<int>(threadIdx.x) * kTiles + k;
      if (upto_t <= lo && lo < upto_t + units[k])
        sh.first = {t, upto_t, upto_t + units[k], req[k], of[k].t0, of[k].n, of[k].len};
      upto_t += units[k];
      sh.ends[t] = upto_t;
      sh.reqs[t] = req[k];
      if (blockIdx.x == 0 && t < a.num_tiles && units[k] == 0) a.shares[t].x = -1;
    }
    wg_barrier();
    const auto first = sh.first;
    tile = uniform(first.tile), start = uniform(first.start), end = uniform(first.end), r = uniform(first.req);
    rq = {uniform(first.t0), uniform(first.n), uniform(first.len)};
  } else {
    tile = a.num_tiles - 1 - static_cast<int>(blockIdx.x);
  }

  for (bool known = kSplit;; tile++, known = false) {
    asm volatile("" : "+v"(lane));   // nothing that depends on the lane alone is kept from tile to tile
    // ---- the tile: its request, its rows, its blocks [b0, b0 + count)
    int b0 = 0, count = 0, last_unit = 0;
    bool whole = true;
    if (kSplit) {
      if (!known) {
        if (tile >= kMaxSplitTiles) return;
        start = end, end = uniform(sh.ends[tile]), r = uniform(sh.reqs[tile]);
      }
      if (start >= hi) return;
      if (start == end) continue;
      // (its blocks come after kTileCost units that stand for its start and end)
      const int first = start + kTileCost;
      b0 = max(lo - first, 0);
      count = min(hi, end) - first - b0;
      if (count <= 0) continue;
      last_unit = end - 1;
      whole = b0 == 0 && count == end - first;
    } else {
      // the last request that starts at or before this tile: its starts are in ascending order
      int begun = 0;
      for (int i = threadIdx.x; i < num_reqs; i += kThreads)
        begun += first_tile<kTM>(min(max(cu[i], 0), total_q), a.heads, i) <= tile;
#pragma unroll
      for (int d = 32; d; d >>= 1) begun += __shfl_xor(begun, d);
      if (lane == 0) sh.sums[w] = begun;
      wg_barrier();
      r = -1;
#pragma unroll
      for (int i = 0; i < kWaves; i++) r += sh.sums[i];
      r = uniform(max(r, 0));
    }
    if (!known) rq = request_of(uniform(cu[r]), uniform(cu[r + 1]), uniform(lens[r]), total_q);
    const int rows = rq.n * a.heads;
    const int row0 = (tile - first_tile<kTM>(rq.t0, a.heads, r)) * kTM;
    if (!kSplit && (row0 < 0 || row0 >= rows)) return;   // an index between two requests
    const int last = last_key<kTM>(rq, row0, a.heads, a.by_heads, max_pos);
    if (!kSplit)
      count = last >= 0 ? last / kKeys + 1 : 0;
    else if (last < 0)
      count = 0;   // nothing to see: its one unit writes the zeros
    // the least of the rows' last positions: keys past it are masked for some row
    const int64_t least64 = static_cast<int64_t>(rq.len) - rq.n + divide(row0, a.by_heads);
    const int least = static_cast<int>(least64 < -1 ? -1 : least64 < last ? least64 : last);

    if (kSplit) wg_barrier();   // LDS is free (the tile before, the scan)

    const int g = lane >> 4, c = lane & 15;
    LateArgs* e = late_args();

    // The queries come through LDS, laid out like keys, in the ring's buffers
    // that the first blocks leave: wave w brings in every eighth row.
    constexpr int kQBuf = kInt8 ? 1 : 2;
    constexpr int kQueries = kTM / kWaves, kQueryLoads = kInt8 ? kQueries : 2 * kQueries;
    auto bring_queries = [&]() {
      const int row = min(row0 + kWaves * min(c, kQueries - 1) + w, rows - 1);   // (rows past the last: the last, not stored)
      const int tok = divide(row, a.by_heads), head = row - tok * a.heads;
      const uint64_t at = reinterpret_cast<uint64_t>(a.q + static_cast<int64_t>(rq.t0 + tok) * a.sq_t +
                                                     static_cast<int64_t>(head) * a.sq_h);
      const int at_lo = static_cast<int>(at), at_hi = static_cast<int>(at >> 32);
#pragma unroll
      for (int j = 0; j < kQueries; j++) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(
            static_cast<uint32_t>(__builtin_amdgcn_readlane(at_lo, j)) |
            static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(at_hi, j))) << 32);
        const int key = kWaves * j + w;
        auto& qs = sh.kv[kQBuf + (key >> 5)];
        load_lds16(lds_offset(qs.lat[key & 31]), from, 16 * (lane ^ swizzle(key)));
        if constexpr (!kInt8) {
          if (lane < 8) load_lds16(lds_offset(qs.rope[key & 31]), from, 2 * kLatent + 16 * (lane ^ rope_swizzle(key)));
        }
      }
    };

    // INT8: a block's conversion: kMine of a latent wave's eight rows by itself,
    // kOthers by the rows' waves (five prompts 147 us with 4 and 4, 143 with 3
    // and 5; 16-row tiles 74.6 with 4 and 4 in the two waves without rows, 75.6
    // with 3 and 5)
    constexpr int kMine = kTM == 16 ? 4 : 3, kOthers = kOwn - kMine;
    // INT8: row 8 z + j of raw block `in`, and as bf16 into the block there
    // (without a row: any codes, with the scale 0)
    auto codes_of = [&](int in, int z, int j) {
      if constexpr (kInt8)
        return *reinterpret_cast<const uint2*>(&sh.raw[in][kOwn * z + j][8 * lane]);
      else
        return make_uint2(0, 0);
    };
    auto convert = [&](int in, int z, int j, uint2 v) {
      if constexpr (kInt8)
        *reinterpret_cast<uint4*>(&sh.kv[in].lat[kOwn * z + j][(16 * lane) ^ (16 * swizzle(kOwn * z + j))]) = codes_to_bf16(v);
    };

    if (w < kHalf) {
      // ================ rows: QK and softmax, a block ahead of PV
      const int kh = w & 1, rh = w >> 1;
      const bool takes_rows = rh * 16 * kRQ < kTM;
      bring_queries();
      loads_left<0>();
      wg_barrier();   // the queries, the first blocks' rows
      bf16x8 qf[kRQ][kSteps];
#pragma unroll
      for (int rt = 0; rt < kRQ; rt++) {
        const int key = 16 * (takes_rows ? rh * kRQ + rt : 0) + c, sw = swizzle(c);
        const auto& qs = sh.kv[kQBuf + (key >> 5)];
#pragma unroll
        for (int st = 0; st < kSteps; st++) {
          const uint8_t* from = qs.lat[key & 31] + 16 * ((4 * (st & 3) + g) ^ sw) + 256 * (st >> 2);
          if constexpr (!kInt8) {
            if (st >= 16) from = qs.rope[key & 31] + 16 * ((4 * (st - 16) + g) ^ rope_swizzle(c));
          }
          const uint4 v = *reinterpret_cast<const uint4*>(from);
          qf[rt][st] = __builtin_bit_cast(bf16x8, make_uint4(v.x ^ a.flip, v.y ^ a.flip, v.z ^ a.flip, v.w ^ a.flip));
        }
      }
      wg_barrier();   // the queries have been read
      // the references (log2) of this lane's rows, from the least number on: every logit passes it
      float ref[kRQ], sum[kRQ];
#pragma unroll
      for (int rt = 0; rt < kRQ; rt++) ref[rt] = -3.4028234663852886e38f, sum[rt] = 0.f;
      f32x4 s[kRQ] = {};            // the last block's logits (log2)
      float part_sum[kRQ] = {};     // its part of the sums
      float4 ks[4] = {};            // INT8: the keys' scales
      // The weights of block n, for PV.
      auto weigh = [&](int n) {
#pragma unroll
        for (int rt = 0; rt < kRQ; rt++) {
          float p[4];
#pragma unroll
          for (int i = 0; i < 4; i++) p[i] = __builtin_amdgcn_exp2f(s[rt][i] - ref[rt]);
          if constexpr (kInt8) {
            // V = codes * f d.  The logits have log2 d in them, so that P has d
            // (and the weight that counts most in a block is a power of two,
            // which bf16 holds); the sum has not.
            part_sum[rt] = (p[0] * ks[0].z + p[1] * ks[1].z) + (p[2] * ks[2].z + p[3] * ks[3].z);
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] *= ks[i].w;
          } else {
            part_sum[rt] = (p[0] + p[1]) + (p[2] + p[3]);
          }
          // P is rounded to bf16 (like the output, 2^-9 of each weight on
          // the average); the sum keeps the unrounded weights.  With the
          // small products of PV the operand's keys are 4 g + i, 16 + 4 g + i.
          const int chunk = kBig ? 2 * kh + (g >> 1) : g, half = kBig ? g & 1 : kh;
          *reinterpret_cast<uint2*>(sh.p[n & 1][16 * (rh * kRQ + rt) + c] + 16 * (chunk ^ (c >> 2 & 3)) + 8 * half) =
              make_uint2(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]));
        }
      };
      int buf = 0;
      for (int n = 0;; n++) {
        // ---- S^T = K Q^T: keys 16 kh + 4 g + i of block n, rows c.  Each
        // K-step's operand is read some steps before its products.
        constexpr int kRead = 6;
        const int key = 16 * kh + c, sw = swizzle(c);
        const auto& blk = sh.kv[buf];
        auto operand = [&](int st) {
          const uint8_t* from = blk.lat[key] + 16 * ((4 * (st & 3) + g) ^ sw) + 256 * (st >> 2);
          if constexpr (!kInt8) {
            if (st >= 16) from = blk.rope[key] + 16 * ((4 * (st - 16) + g) ^ rope_swizzle(c));
          }
          return *reinterpret_cast<const bf16x8*>(from);
        };
        bf16x8 k[kSteps];
        const int again = sh.again[(n & 1) ^ 1];
        const uint32_t have_v = static_cast<uint32_t>(*reinterpret_cast<const int*>(sh.have[n & 7]));
        if (takes_rows) {   // (after the last block: not used)
#pragma unroll
          for (int st = 0; st < kRead; st++) k[st] = operand(st);
        }
        if (n && uniform(again) == n - 1) {
          // ---- the block before again: both waves of a row find its reference
          float top[kRQ];
          if (takes_rows) {
#pragma unroll
            for (int rt = 0; rt < kRQ; rt++) {
              top[rt] = quad_max(fmaxf(fmaxf(s[rt][0], s[rt][1]), fmaxf(s[rt][2], s[rt][3])));
              if (lane < 16) sh.red[kh][16 * (rh * kRQ + rt) + c] = top[rt];
            }
          }
          wg_barrier();   // the maxima
          if (takes_rows) {
#pragma unroll
            for (int rt = 0; rt < kRQ; rt++) {
              const int row = 16 * (rh * kRQ + rt) + c;
              const float m = fmaxf(ref[rt], fmaxf(sh.red[0][row], sh.red[1][row]));
              const float alpha = __builtin_amdgcn_exp2f(ref[rt] - m);
              ref[rt] = m;
              sum[rt] *= alpha;
              if (kh == 0 && lane < 16) sh.alpha[row] = alpha;
            }
            weigh(n - 1);
          }
          wg_barrier();   // P
        }
#pragma unroll
        for (int rt = 0; rt < kRQ; rt++) sum[rt] += part_sum[rt];
        if (n == count) break;
        // INT8: a part of the next block's conversion, between the products
        const int next = buf + 1 < kBufs ? buf + 1 : 0;
        uint2 codes[kOthers];
        if (kTM > 16) {
#pragma unroll
          for (int j = 0; j < kOthers; j++) codes[j] = codes_of(next, w, kMine + j);
        }
        if (!takes_rows) {   // (of a 16-row tile: waves 2 and 3, each for two)
#pragma unroll
          for (int z = 0; z < 2; z++) {
#pragma unroll
            for (int j = 0; j < kOthers; j++) codes[j] = codes_of(next, 2 * kh + z, kMine + j);
#pragma unroll
            for (int j = 0; j < kOthers; j++) convert(next, 2 * kh + z, kMine + j, codes[j]);
          }
        } else {
          const uint32_t have = static_cast<uint32_t>(uniform(static_cast<int>(have_v)));
          if constexpr (kInt8) {
#pragma unroll
            for (int i = 0; i < 4; i++) ks[i] = sh.scl[buf][16 * kh + 4 * g + i];
          }
          static_assert(!kInt8 || (kSteps - 2) / 3 + 1 >= kOthers, "a step for each of the rows to convert");
          // two sums with one row tile, so that a product does not wait for the one before it
          constexpr int kSums = kRQ == 1 ? 2 : 1;
          f32x4 t[kRQ][kSums];
#pragma unroll
          for (int rt = 0; rt < kRQ; rt++)
#pragma unroll
            for (int u = 0; u < kSums; u++) t[rt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < kSteps; st++) {
            if (st + kRead < kSteps) k[st + kRead] = operand(st + kRead);
#pragma unroll
            for (int rt = 0; rt < kRQ; rt++)
              t[rt][st % kSums] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[st], qf[rt][st], t[rt][st % kSums], 0, 0, 0);
            if (kTM > 16 && st % 3 == 1 && st / 3 < kOthers) convert(next, w, kMine + st / 3, codes[st / 3]);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int rt = 0; rt < kRQ; rt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const float dot = kSums == 1 ? t[rt][0][i] : t[rt][0][i] + t[rt][kSums - 1][i];
              s[rt][i] = kInt8 ? __builtin_fmaf(dot, ks[i].x, ks[i].y) : dot * a.scale_log2;
            }
          if (have != ~0u || (b0 + n + 1) * kKeys - 1 > least) {
#pragma unroll
            for (int rt = 0; rt < kRQ; rt++) {
              const int row = min(row0 + 16 * (rh * kRQ + rt) + c, rows - 1);
              const int64_t see = static_cast<int64_t>(rq.len) - rq.n + divide(row, a.by_heads);
              const int limit = static_cast<int>(see < last ? see < -1 ? -1 : see : last) - (b0 + n) * kKeys;
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const int key = 16 * kh + 4 * g + i;
                if (key > limit || !(have >> key & 1)) s[rt][i] = -INFINITY;
              }
            }
          }
          bool far = false;
#pragma unroll
          for (int rt = 0; rt < kRQ; rt++)
            far |= fmaxf(fmaxf(s[rt][0], s[rt][1]), fmaxf(s[rt][2], s[rt][3])) > ref[rt] + kSlack;
          if (far) sh.again[n & 1] = n;
          weigh(n);
        }
        wg_barrier();   // P
        buf = next;
      }
      if (count) wg_barrier();   // PV has read P and the rescaling for the last time
      if (takes_rows) {
#pragma unroll
        for (int rt = 0; rt < kRQ; rt++) {
          const float l = quad_sum(sum[rt]);
          const int row = 16 * (rh * kRQ + rt) + c;
          if (lane < 16) sh.red[kh][row] = l;
          if (kh == 0 && lane < 16) sh.alpha[row] = ref[rt];
        }
      }
      wg_barrier();   // the sums
    } else {
      // ================ latents: loads, PV
      const int y = w - kHalf;
      // ---- bringing blocks in, counted from the first (block n has the
      // positions 32 (b0 + n) + [0, 32)).  Wave y brings in rows 8 y .. 8 y + 7.
      // A key past the last one seen, or whose page is not in the table or the
      // cache, has no row: the cache's first is read in its place (or, past the
      // last one, what the page has there), and zeroed if it is bf16, so that
      // every wave sends kLoads loads a block, also for blocks past the end.
      //
      // With kRuns the wave needs one table entry a block: lane l keeps that of
      // block l of 64, and the next 64 come while they are used.  Without, lane
      // l looks after row l / 8 (INT8: l % 8).
      const int32_t* bt = a.bt + static_cast<int64_t>(r) * a.bt_stride;
      auto look_up = [&](int n) {       // the table's entries for block n, kRuns: for blocks n .. n + 63
        const int64_t at = kRuns ? (b0 + n + lane) * static_cast<int64_t>(kKeys) + kOwn * y : (b0 + n) * kKeys + (lane & 31);
        const int pg = divide(static_cast<int>(at < last ? at : last), a.by_block);
        if constexpr (kRuns) {
          load_lds4_at(lds_offset(&sh.page[64 * y]), bt + pg);
        } else {
          if (lane < 32) load_lds4_at(lds_offset(&sh.page[32 * (n & 7)]), bt + pg);   // by every wave
        }
      };
      uint32_t masks = 0;               // a byte per block on its way, of this wave's rows
      int pages = 0;                    // kRuns
      uint64_t run = 0;                 // kRuns: the address of the eight rows
      uint32_t row_lo = 0, row_hi = 0;  // of the lane's row, without kRuns
      uint32_t row_off[kRuns ? kRowLoads : 1];
      if constexpr (kRuns) {
        const uint32_t rb = static_cast<uint32_t>(a.row_bytes);
#pragma unroll
        for (int j = 0; j < kRowLoads; j++) {
          if (kInt8)
            row_off[j] = j < 4 ? (2 * j + (lane >> 5)) * rb + 16 * (lane & 31) : (lane & 7) * rb + kLatent;
          else
            row_off[j] = j < kOwn ? j * rb + ((16 * lane) ^ (16 * swizzle(kOwn * y + j)))
                                  : (lane >> 3) * rb + 2 * kLatent + 16 * ((lane & 7) ^ rope_swizzle(kOwn * y + (lane >> 3)));
        }
      }
      const int of_lane = kInt8 ? lane & 7 : lane >> 3;
      // where block n's rows are; what of them there is, a bit each
      auto address = [&](int n) {
        uint32_t mask;
        if constexpr (kRuns) {
          if ((n & 63) == 0) pages = sh.page[64 * y + lane];
          const uint32_t page = static_cast<uint32_t>(__builtin_amdgcn_readlane(pages, n & 63));
          const int pos = (b0 + n) * kKeys + kOwn * y;
          const uint32_t in_page = static_cast<uint32_t>(pos - divide(pos, a.by_block) * a.block_size);
          const int left = n < count && page < static_cast<uint32_t>(a.num_blocks) ? last - pos + 1 : 0;
          mask = left >= kOwn ? 0xffu : left > 0 ? (1u << left) - 1 : 0u;
          run = reinterpret_cast<uint64_t>(a.kv) +
                (mask ? page * static_cast<uint64_t>(a.page_bytes) + in_page * static_cast<uint64_t>(a.row_bytes) : 0);
        } else {
          const int key = kOwn * y + of_lane, pos = (b0 + n) * kKeys + key;
          const int page = sh.page[32 * (n & 7) + key];
          const int in_page = pos - divide(pos, a.by_block) * a.block_size;
          const bool ok = n < count && pos <= last && static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_blocks);
          const uint64_t at = reinterpret_cast<uint64_t>(a.kv) +
                              (ok ? page * static_cast<uint64_t>(a.page_bytes) + in_page * static_cast<uint64_t>(a.row_bytes) : 0);
          row_lo = static_cast<uint32_t>(at), row_hi = static_cast<uint32_t>(at >> 32);
          const uint64_t all = __ballot(ok);
          // INT8: the low byte; bf16: bit 8 j to bit j
          mask = kInt8 ? static_cast<uint32_t>(all) & 0xff
                       : static_cast<uint32_t>(((all & 0x0101010101010101ull) * 0x0102040810204080ull) >> 56);
        }
        if (lane == 0) sh.have[n & 7][y] = static_cast<uint8_t>(mask);
        return mask;
      };
      auto row_of = [&](int j) {        // uniform: row j of the wave's
        const int from = kInt8 ? j : 8 * j;
        return static_cast<uint32_t>(__builtin_amdgcn_readlane(row_lo, from)) |
               static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(row_hi, from))) << 32;
      };
      // loads 2 j and 2 j + 1 (of kRowLoads) of the block whose addresses are there into buffer `to`
      constexpr int kPairs = (kRowLoads + 1) / 2;
      auto bring = [&](int to, int j) {
        const uint8_t* own = reinterpret_cast<const uint8_t*>(row_lo | static_cast<uint64_t>(row_hi) << 32);
        const uint8_t* base = reinterpret_cast<const uint8_t*>(run);
        if constexpr (kInt8) {
          const uint32_t dst = lds_offset(sh.raw[to][kOwn * y + 4 * j]);
          if (j == 2) {
            if (lane < kOwn) {
              if constexpr (kRuns)
                load_lds4(lds_offset(&sh.raw_scale[to][kOwn * y]), base, row_off[kRowLoads - 1]);
              else
                load_lds4_at(lds_offset(&sh.raw_scale[to][kOwn * y]), own + kLatent);
            }
          } else if constexpr (kRuns) {
            load_lds16_2(dst, base, row_off[2 * j], row_off[2 * j + 1]);
          } else {
            for (int i = 0; i < 2; i++) {
              const uint64_t row = lane < 32 ? row_of(4 * j + 2 * i) : row_of(4 * j + 2 * i + 1);
              load_lds16_at(dst + 1024 * i, reinterpret_cast<const uint8_t*>(row) + 16 * (lane & 31));
            }
          }
        } else {
          const uint32_t dst = lds_offset(sh.kv[to].lat[kOwn * y + 2 * j]);
          if (j == 4) {
            if constexpr (kRuns)
              load_lds16(lds_offset(sh.kv[to].rope[kOwn * y]), base, row_off[kRowLoads - 1]);
            else
              load_lds16_at(lds_offset(sh.kv[to].rope[kOwn * y]), own + 2 * kLatent + 16 * ((lane & 7) ^ rope_swizzle(kOwn * y + (lane >> 3))));
          } else if constexpr (kRuns) {
            load_lds16_2(dst, base, row_off[2 * j], row_off[2 * j + 1]);
          } else {
            for (int i = 0; i < 2; i++)
              load_lds16(dst + 1024 * i, reinterpret_cast<const uint8_t*>(row_of(2 * j + i)), (16 * lane) ^ (16 * swizzle(kOwn * y + 2 * j + i)));
          }
        }
      };
      auto zero_rows = [&](int in, uint32_t mask) {   // bf16: rows that are not there, after the loads in their place
        if constexpr (!kInt8) {
          for (int j = 0; j < kOwn; j++)
            if (!(mask >> j & 1)) {
              *reinterpret_cast<uint4*>(&sh.kv[in].lat[kOwn * y + j][16 * lane]) = make_uint4(0, 0, 0, 0);
              if (lane < 8) *reinterpret_cast<uint4*>(&sh.kv[in].rope[kOwn * y + j][16 * lane]) = make_uint4(0, 0, 0, 0);
            }
        }
      };
      // INT8: scales s = f d.  d is |s| and f its sign where |s| is in the middle
      // of fp32's range (2^-64 .. 2^64: then log2 d moves no weight out of it),
      // else 1 and s; without a row, or with no number for a scale, f is 0: a
      // masked weight 0 has to stay 0.
      auto scales = [&](int in, uint32_t mask) {
        if constexpr (kInt8) {
          if (lane < kOwn) {
            const float v = mask >> lane & 1 ? sh.raw_scale[in][kOwn * y + lane] : 0.f, size = fabsf(v);
            const bool middle = size >= 0x1p-64f && size <= 0x1p64f;
            const float d = middle ? size : 1.f;
            sh.scl[in][kOwn * y + lane] =
                make_float4(a.scale_log2 * v, __builtin_amdgcn_logf(d), __builtin_amdgcn_rcpf(d),
                            middle ? copysignf(1.f, v) : size < INFINITY ? v : 0.f);
          }
        }
      };

      if (count) {
        if constexpr (kRuns) {
          look_up(0);
        } else {
#pragma unroll
          for (int n = 0; n < kAhead + 2; n++) look_up(n);
        }
      }
      bring_queries();
      if (count) {
        loads_left<kQueryLoads>();
#pragma unroll
        for (int n = 0; n < kEarly; n++) {
          masks |= address(n) << (8 * n);
#pragma unroll
          for (int j = 0; j < kPairs; j++) bring(n, j);
        }
        masks |= address(kEarly) << (8 * kEarly);
        loads_left<kRowLoads>();   // the last of these blocks may be on its way
        if (kInt8) {
#pragma unroll
          for (int j = 0; j < kOwn; j++) convert(0, y, j, codes_of(0, y, j));
          scales(0, masks);
        } else {
          if ((masks & 0xff) != 0xff) zero_rows(0, masks);
        }
        masks >>= 8;   // of the blocks from 1
      } else {
        loads_left<0>();
      }
      if (w == kHalf && lane < 2) sh.again[lane] = -1;
      wg_barrier();   // the queries, the first block's rows
      Acc acc[kLT][kRT];
#pragma unroll
      for (int i = 0; i < kLT; i++)
#pragma unroll
        for (int j = 0; j < kRT; j++)
#pragma unroll
          for (int q = 0; q < kAcc; q++) acc[i][j][q] = 0.f;
      wg_barrier();   // the queries have been read

      // iteration n: PV of block n (the rows' waves are at block n + 1).  Of
      // 16-row tiles this side is the longer one, and goes first where both
      // could (64 ragged INT8 requests 85.4 -> 81.8 us; 64-row tiles lose 6 %).
      if (kTM == 16) __builtin_amdgcn_s_setprio(1);
      int buf = kBufs - 1;   // of block n
      for (int n = -1; n < count && count; n++) {
        const int next = buf + 1 < kBufs ? buf + 1 : 0, after = next + 1 < kBufs ? next + 1 : 0;
        // bf16: block n + 3 comes into the buffer of block n - 1; INT8: block n
        // + 4 into the raw one of block n + 1 (converted in the iteration
        // before), and block n + 2 is converted
        const int into = kInt8 ? next : buf > 0 ? buf - 1 : kBufs - 1;
        constexpr int kRead = 4, kGroups = kKeys / kDepth;
        const int part = lane / kSize, pr = lane & (kSize - 1), c16 = lane & 15;
        bf16x8 pb[kGroups][kRT], v[kPvSteps];
        const int again = sh.again[n & 1];
        auto weights = [&]() {
#pragma unroll
          for (int t = 0; t < kGroups; t++)
#pragma unroll
            for (int j = 0; j < kRT; j++) {
              const int chunk = kDepth / 8 * t + part;
              pb[t][j] = *reinterpret_cast<const bf16x8*>(sh.p[n & 1][kSize * j + pr] + 16 * (chunk ^ (pr >> 2 & 3)));
            }
        };
        weights();   // (before block 0: not used)
        if constexpr (!kInt8) {
          // Keys that some row of the tile may not see: 0 * inf would put NaN
          // into that row.  A row that sees such a key has NaN from its logit.
          // (This wave's latents of all rows.)
          if (n >= 0 && (b0 + n + 1) * kKeys - 1 > least && least < last) {
            for (int j = 0; j < kKeys; j += 4) {
              uint4* at = reinterpret_cast<uint4*>(&sh.kv[buf].lat[j + g][256 * y + 16 * c]);
              const uint4 v = *at;
              *at = make_uint4(finite_bf16x2(v.x), finite_bf16x2(v.y), finite_bf16x2(v.z), finite_bf16x2(v.w));
            }
          }
        }

        // ---- O^T += V^T P^T: V's operands are read some steps ahead; between
        // the steps come the loads of a later block and the conversion.  In
        // the iteration before block 0 the weights and the output are zero.
        // a transposing read gives a lane its column (latent) of four rows (keys)
        const int tr_row = kBig ? 8 * (lane >> 5) + (c16 >> 2) : 4 * g + (c16 >> 2);
        const int tr_col = (kBig ? 8 * (g & 1) : 0) + ((c16 & 3) >> 1);      // 16-byte chunk, + those of the tile
        const uint8_t* base[kLT][kBig ? 2 : 1];
#pragma unroll
        for (int i = 0; i < kLT; i++)
#pragma unroll
          for (int h = 0; h < (kBig ? 2 : 1); h++)
            base[i][h] = &sh.kv[buf].lat[tr_row + 4 * h][256 * y + 16 * ((2 * i + tr_col) ^ swizzle(tr_row + 4 * h)) +
                                                         8 * (c16 & 1)];
        auto operand = [&](int u) {
          const int i = u % kLT, t = u / kLT;   // latent tile, keys
          const uint8_t* p0 = base[i][0] + kDepth * t * 2 * kLatent;
          const uint8_t* p1 = kBig ? base[i][kBig ? 1 : 0] + kDepth * t * 2 * kLatent : p0 + 16 * 2 * kLatent;
          const i32x2 v0 = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(GLM53_LDS(i16x4, p0)));
          const i32x2 v1 = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(GLM53_LDS(i16x4, p1)));
          return __builtin_bit_cast(bf16x8, make_uint4(v0[0], v0[1], v1[0], v1[1]));
        };
        if (n >= 0) {
#pragma unroll
          for (int u = 0; u < kRead; u++) v[u] = operand(u);
        }
        uint2 codes[kMine];
#pragma unroll
        for (int j = 0; j < kMine; j++) codes[j] = codes_of(after, y, j);
        if (n >= 0 && uniform(again) == n) {
          wg_barrier();   // the maxima
          wg_barrier();   // P
          weights();
#pragma unroll
          for (int j = 0; j < kRT; j++) {
            const float alpha = sh.alpha[kSize * j + pr];
#pragma unroll
            for (int i = 0; i < kLT; i++)
#pragma unroll
              for (int q = 0; q < kAcc; q++) acc[i][j][q] *= alpha;
          }
        }
        const bool group = kRuns && ((n + kAhead + 1) & 63) == 32;
        if (group) look_up(n + kAhead + 1 + 32);
        auto between = [&](int u) {   // kPvSteps = 8
          if (u < kMine) convert(after, y, u, codes[u]);
          if (u == 7) scales(after, masks);
          if (u < kPairs) bring(into, u);
          if (u == 5 && !kRuns) look_up(n + kAhead + 3);
          if (u == 6) masks |= address(n + kAhead + 1) << (kInt8 ? 24 : 16);
        };
        static_assert(kPvSteps == 8 && kOwn == 8, "a row a step");
        if (n >= 0) {
#pragma unroll
          for (int u = 0; u < kPvSteps; u++) {
            const int i = u % kLT, t = u / kLT;
            if (u + kRead < kPvSteps) v[u + kRead] = operand(u + kRead);
#pragma unroll
            for (int j = 0; j < kRT; j++) {
              if constexpr (kBig)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[u], pb[t][j], acc[i][j], 0, 0, 0);
              else
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], pb[t][j], acc[i][j], 0, 0, 0);
            }
            between(u);
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
#pragma unroll
          for (int u = 0; u < kPvSteps; u++) between(u);
        }
        // all but this iteration's: block n + 2's rows (INT8: n + 3's) are there
        if (group)
          loads_left<kLoads + 1>();
        else
          loads_left<kLoads>();
        if (!kInt8 && (masks & 0xff) != 0xff) zero_rows(after, masks);
        masks >>= 8;   // from block n + 3 on
        wg_barrier();    // P
        buf = next;
      }
      if (kTM == 16) __builtin_amdgcn_s_setprio(0);
      loads_left<0>();   // what was asked for past the last block
      wg_barrier();      // the sums

      // ---- the output as bf16 into LDS, or the partial
      auto sum_of = [&](int row) { return sh.red[0][row] + sh.red[1][row]; };
      const int part = lane / kSize, pr = lane & (kSize - 1);
      if (whole) {
        // chunk c of 16 bytes of row r at c ^ (r % 16), so that rows fall on different banks
        uint8_t* os = sh.kv[0].lat[0];
#pragma unroll
        for (int j = 0; j < kRT; j++) {
          const float l = sum_of(kSize * j + pr);
          const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
          for (int i = 0; i < kLT; i++)
#pragma unroll
            for (int q = 0; q < kAcc; q += 4) {
              const Acc v = acc[i][j];
              const int lat = latent_of(y, i, 2 * q + 4 * part);   // of v[q]
              *reinterpret_cast<uint2*>(os + (kSize * j + pr) * 2 * kLatent + ((2 * lat & ~15) ^ (16 * (pr & 15))) + (2 * lat & 15)) =
                  make_uint2(pack_bf16x2(v[q] * inv, v[q + 1] * inv), pack_bf16x2(v[q + 2] * inv, v[q + 3] * inv));
            }
        }
      } else {
        // slot 2 g: the tile began in an earlier workgroup; 2 g + 1: it begins
        // here.  In the accumulators' order: 16 bytes of each lane at a time.
        const int slot = 2 * static_cast<int>(blockIdx.x) + (b0 == 0);
        float* out = e->part + static_cast<int64_t>(slot) * (kTM * kLatent);
#pragma unroll
        for (int i = 0; i < kLT; i++)
#pragma unroll
          for (int j = 0; j < kRT; j++)
#pragma unroll
            for (int q = 0; q < kAcc; q += 4) {
              const Acc v = acc[i][j];
              *reinterpret_cast<f32x4*>(out + (((kLT * y + i) * kRT + j) * (kAcc / 4) + q / 4) * 256 + 4 * lane) =
                  f32x4{v[q], v[q + 1], v[q + 2], v[q + 3]};
            }
        if (y == 0 && lane < kTM)
          e->ml[static_cast<int64_t>(slot) * kTM + lane] = make_float2(sh.alpha[lane], sum_of(lane));
        if (b0 == 0 && y == 0 && lane == 0) {
          const int longer = more * (each + 1);   // units of the longer runs
          e->shares[tile] = make_int4(blockIdx.x, last_unit < longer ? last_unit / (each + 1) : more + (last_unit - longer) / each,
                                       rq.t0 * a.heads + row0, min(rows - row0, kTM));
        }
      }
    }

    if (whole) {   // whole rows go out, every eighth of each wave's
      wg_barrier();
      const uint8_t* os = sh.kv[0].lat[0];
      const int heads = e->heads, aligned = e->out_align16;
      const Divider by_heads = {e->by_heads.mul, e->by_heads.sh1, e->by_heads.sh2};
      const int64_t so_t = e->so_t, so_h = e->so_h;
      uint16_t* out = e->out;
      float* lse = e->lse;
      for (int j = w; j < kTM && row0 + j < rows; j += kWaves) {
        const int row = row0 + j, tok = divide(row, by_heads), head = row - tok * heads;
        uint16_t* o = out + static_cast<int64_t>(rq.t0 + tok) * so_t + static_cast<int64_t>(head) * so_h;
        const uint4 v = *reinterpret_cast<const uint4*>(os + j * 2 * kLatent + ((16 * lane) ^ (16 * (j & 15))));
        if (aligned) {
          reinterpret_cast<uint4*>(o)[lane] = v;
        } else {
          reinterpret_cast<uint2*>(o)[2 * lane] = make_uint2(v.x, v.y);
          reinterpret_cast<uint2*>(o)[2 * lane + 1] = make_uint2(v.z, v.w);
        }
        if (lse && lane == 0) {
          const float l = sh.red[0][j] + sh.red[1][j];
          lse[static_cast<int64_t>(rq.t0 + tok) * heads + head] =
              l == 0.f ? -INFINITY : (sh.alpha[j] + __builtin_amdgcn_logf(l)) * kLn2;
        }
      }
      if (kSplit && threadIdx.x == 0) e->shares[tile].x = -1;
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
__global__ __launch_bounds__(kTogether > 1 ? 64 * kTogether : 256) void chunk_mla_merge_kernel(
    const int4* shares, const float2* part_ml, const float* partials, const ChunkArgs a) {
  constexpr int kRowSize = ChunkShape<kTM>::kBig ? 32 : 16, kRT = kTM / kRowSize, kQuads = kRowSize == 32 ? 4 : 1;
  constexpr int kDeep = kTogether == 4 ? 4 : 16;
  __shared__ float acc_s[kTogether][64][4];
  __shared__ float2 ml_s[kTogether][kRowSize];
  const int tile = blockIdx.y;
  const int4 share = shares[tile];
  if (share.x < 0) return;
  const int first = uniform(share.x), last = uniform(share.y);
  const int w = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, part = lane / kRowSize, c = lane & (kRowSize - 1);
  const int job = kTogether > 1 ? blockIdx.x : 4 * blockIdx.x + w;
  const int j = job / kQuads % kRT;   // row tile
  constexpr int kLT = 128 / kRowSize;
  const int tile_l = job / (kQuads * kRT), lat = latent_of(tile_l / kLT, tile_l % kLT, 8 * (job % kQuads) + 4 * part);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int k0 = first + (kTogether > 1 ? w : 0); k0 <= last; k0 += kTogether * kDeep) {
    float2 ml[kDeep];
    f32x4 v[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; d++) {
      const int k = k0 + kTogether * d;
      ml[d] = make_float2(-INFINITY, 0.f), v[d] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (k <= last) {   // uniform
        const int64_t slot = 2 * static_cast<int64_t>(k) + (k == first);
        ml[d] = part_ml[slot * kTM + kRowSize * j + c];
        v[d] = *reinterpret_cast<const f32x4*>(partials + slot * (kTM * kLatent) + job * 256 + 4 * lane);
      }
    }
    float top = m;
#pragma unroll
    for (int d = 0; d < kDeep; d++) top = fmaxf(top, ml[d].x);
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
  if (kRowSize * j + c >= share.w) return;
  const int row = share.z + kRowSize * j + c, tok = divide(row, a.by_heads), head = row - tok * a.heads;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* o = a.out + static_cast<int64_t>(tok) * a.so_t + static_cast<int64_t>(head) * a.so_h;
  *reinterpret_cast<uint2*>(o + lat) =
      make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  if (a.lse && lat == 0)
    a.lse[static_cast<int64_t>(tok) * a.heads + head] =
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
  w.bytes = shares + tiles * 16;
  return w;
}

template <int kTM, bool kInt8, bool kRuns>
int launch(ChunkArgs& a, void* workspace, hipStream_t st) {
  // (units of all tiles are counted in an int)
  const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.block_size;
  if (a.num_tiles > kMaxSplitTiles || (cap / kKeys + 1 + kTileCost) * a.num_tiles > 0x7fffffff) {
    hipLaunchKernelGGL((chunk_mla_kernel<kTM, kInt8, false, kRuns>), dim3(a.num_tiles), dim3(kThreads), 0, st,
                       a.cu, a.lens, a.num_reqs, a.total_q, a);
  } else {
    const Workspace ws = workspace_of(kTM, a.num_tiles);
    uint8_t* p = static_cast<uint8_t*>(workspace);
    a.part = reinterpret_cast<float*>(p);
    a.ml = reinterpret_cast<float2*>(p + ws.ml);
    a.shares = reinterpret_cast<int4*>(p + ws.bytes - 16 * static_cast<int64_t>(a.num_tiles));
    hipLaunchKernelGGL((chunk_mla_kernel<kTM, kInt8, true, kRuns>), dim3(num_cus()), dim3(kThreads), 0, st, a.cu,
                       a.lens, a.num_reqs, a.total_q, a);
    // a shared tile has at most about CUs / tiles partials: 16 waves on a job
    // where that is many, four or one where it is few (24 requests of 64 rows,
    // about ten each: 47.7 us with one, 45.4 with four; 23 of 32 rows 21.3, 22.0)
    const int partials = num_cus() / a.num_tiles;
    if (partials > 64)
      hipLaunchKernelGGL((chunk_mla_merge_kernel<kTM, 16>), dim3(2 * kTM, a.num_tiles), dim3(1024), 0, st,
                         a.shares, a.ml, a.part, a);
    else if (partials > (kTM == 64 ? 4 : 24))
      hipLaunchKernelGGL((chunk_mla_merge_kernel<kTM, 4>), dim3(2 * kTM, a.num_tiles), dim3(256), 0, st,
                         a.shares, a.ml, a.part, a);
    else
      hipLaunchKernelGGL((chunk_mla_merge_kernel<kTM, 1>), dim3(kTM / 2, a.num_tiles), dim3(256), 0, st,
                         a.shares, a.ml, a.part, a);
  }
  return static_cast<int>(hipGetLastError());
}

template <bool kInt8, bool kRuns>
int launch_of(int tm, ChunkArgs& a, void* workspace, hipStream_t st) {
  if (tm == 16) return launch<16, kInt8, kRuns>(a, workspace, st);
  return tm == 32 ? launch<32, kInt8, kRuns>(a, workspace, st) : launch<64, kInt8, kRuns>(a, workspace, st);
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
  a.by_block = divider(block_size), a.by_heads = divider(num_heads);
  a.num_reqs = static_cast<int>(num_reqs), a.total_q = static_cast<int>(total_q), a.heads = static_cast<int>(num_heads);
  a.num_tiles = static_cast<int>(tiles);
  const float scale_log2 = static_cast<float>(sm_scale * 1.4426950408889634);
  a.scale_log2 = fabsf(scale_log2);
  a.flip = scale_log2 < 0.f ? 0x80008000u : 0;
  a.out = static_cast<uint16_t*>(out);
  a.so_t = so_t, a.so_h = so_h;
  a.out_align16 = oa % 16 == 0 && so_t % 8 == 0 && so_h % 8 == 0;
  a.lse = lse;
  // (a row's offset from the first of eight is 32 bits)
  const bool runs = block_size % kOwn == 0 && row_bytes < (INT64_C(1) << 28);
  if (kv_is_int8) return runs ? launch_of<true, true>(tm, a, workspace, st) : launch_of<true, false>(tm, a, workspace, st);
  return runs ? launch_of<false, true>(tm, a, workspace, st) : launch_of<false, false>(tm, a, workspace, st);
}
