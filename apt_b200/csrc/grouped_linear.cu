// Products of rows in ragged groups with the weights of their group, on the tensor cores.
//
//   out[r, n] = sum_k x[r, k] w[g, n, k] + b[g, n]      rows r of group g
//   dx[r, k]  = sum_n dy[r, n] w[g, n, k]
//   dw[g, n, k] = sum_{r in g} dy[r, n] x[r, k],   db[g, n] = sum_{r in g} dy[r, n]
//
// One persistent kernel for all three (k_grouped), a block an SM: a thread has boxes of both operands copied to a ring of stages in
// shared memory, one issues the products of a stage into tensor memory, eight warps (fp32: four) bring finished tiles out, from one half of
// tensor memory while the products of the next go to the other. Where the groups end is on the device only, so every block makes the list of
// tiles from the ends and its warps walk it. In dw a run of stages, as long for every block, may begin and end within a sum: it leaves
// partial sums, which k_join_weights adds up.
//
// The tensor cores cut their sums off instead of rounding them: sums of one sign lose half a unit of the 24th bit with every 16 terms (8192 terms in one
// sum: 2.6e-5; 262144 rows in dw: 1.1e-3, twice the rounding of f16). So a sum is brought out in parts (GroupedTraits::kCut), which are added up in
// fp32, rounded to nearest: 3e-6 in fp32, 3e-5 in dw of 16 bits, where the rounding of f16 is 4.9e-4. A contraction of out or dx in 16 bits has 8192 terms at
// most and is not cut.
//
// Operands stay as they are in memory, row by row; whether rows run along the contraction or across it is a bit of the product. A box
// that reaches past a matrix is filled with zeros. Past the end of a group within a matrix it has the next group's rows: in out and dx those are
// rows of the tile that are not written, in dw they are part of the sum and are overwritten with zeros first, in both operands.
//
// fp32: x = h + m + l exactly, each bf16 (the upper 8, the next 8 and the last 8 bits: cut off, so nothing overflows). Of the nine
// products of two such sums the six of more than 2^-24 of the whole are made: h h in one sum, the five small ones in another, which loses
// nothing to the large one's roundings. Two teams of four warps take the stages apart in turn. Infinities are their own upper bits, and NaN below
// them: where the two sums make a NaN the large one, which has everything that is not finite in its upper bits, is the result.
#include <algorithm>

#include "dense.cuh"
#include "umma.cuh"
#include "widen.cuh"

namespace apt {

enum GroupedMode { kOut = 0, kGradX = 1, kGradW = 2 };

constexpr int kTileM = 128;                  // rows of a product
constexpr int kMostShared = 227 * 1024 - 640;      // shared memory of a block but for the barriers' and the scan's
constexpr int kAccColumns = 256;             // tensor memory of a tile: there is room for two
constexpr int kMaxStages = 12;
constexpr int kPlanWords = 5;                // of a run
constexpr int kJoinParts = 16;               // blocks for a sum of dw
constexpr int kKeepChange = 2;               // tiles that changing kept weights takes the time of (5 us to 2.4 a tile of bf16, 8 to 4 of fp32)

template <typename T, int MODE>
struct GroupedTraits {
  static constexpr bool kSplit = sizeof(T) == 4;
  static constexpr bool kMnA = MODE == kGradW, kMnB = MODE != kOut;
  static constexpr int kBlock = kSplit ? 32 : 64;              // of the contraction in a stage
  static constexpr int kBox = 128 / (int)sizeof(T);            // elements of a box's row
  static constexpr int kMostN = kSplit ? 128 : 256;            // columns of a tile
  // warps that bring tiles out: two for each quarter of tensor memory's lanes, or one beside the eight that take fp32 apart
  static constexpr int kOutWarps = kSplit ? 4 : 8;
  static constexpr int kThreads = kSplit ? 512 : 384;
  // a sum in tensor memory has so many stages at most: 1024 terms of fp32, 8192 rows of 16 bits (with 4096, 65536 x 1024 -> 1024 bf16, dw and db 182 -> 205 us:
  // the warps that bring parts out are those that add up db, for which the stages wait)
  static constexpr bool kCuts = kSplit || MODE == kGradW;
  static constexpr int kCut = kSplit ? 32 : 128;
  // bytes of a tile of n rows (or columns) in a stage as copied, and of one bf16 piece of it
  static __host__ __device__ constexpr int copied(int n, bool mn) { return mn ? (n + kBox - 1) / kBox * kBlock * 128 : n * 128; }
  static __host__ __device__ constexpr int piece(int n, bool mn) { return mn ? (n + 63) / 64 * kBlock * 128 : (n + 31) / 32 * 32 * kBlock * 2; }
};

struct GroupedCall {
  const int64_t* offsets;
  int64_t rows;
  int groups;
  int num_m, num_n, num_k;      // num_m: rows of dw, num_k: contraction of out and dx
  int tile_m, tile_n, tiles_m, tiles_n;
  int copied_stages, piece_stages;
  int keep;                     // out and dx: a group's weights stay in shared memory while a block has tiles of it
  int halves;                   // out and dx: tiles of 128 rows that share a stage's weights
  int deep;                     // out and dx: blocks of the contraction in a stage
  int polls;                    // of a wait
  int64_t ranges;               // dw: into how many runs of stages the work is cut at most, each a block's
  const void *a, *b;            // the operands, as the copies read them
  int64_t pitch_a, pitch_b;     // elements
  const void* bias;
  void *out, *grad_bias;
  float *partial, *partial_bias;
  float* carry;                 // a tile a block: the parts so far of a sum that is brought out in parts
  int64_t* plan;                // dw, for k_join_weights: units, runs, and of each run its first piece's tile and group and the sum's first unit, the run's
                                // beginning and that of the run before, the sum's last run
  int32_t* status;
};

// ---- the list of tiles ------------------------------------------------------------
struct GroupedItem {
  int g;
  int64_t row;                  // first row of x
  int rows;                     // of the group from there on, in out and dx at most halves tile_m
  int m0, n0, stages;
  int before = 0, after = 0;    // stages of the same sum (in dw, of the run's piece of it) in parts before this one, and behind it
  int64_t piece;                // dw: number of the partial sum, -1: all of the sum
  int64_t first, last;          // dw: units of all of the sum
};

// Runs of stages of dw: every run is as long as any other within one, whatever the groups are. A run has all stages of the tiles and
// groups in its middle; two at most, at its ends, it has parts of.
struct GroupedRuns {
  int64_t units, runs;
  __device__ __forceinline__ int64_t begin(int64_t v) const { return v * units / runs; }
  __device__ __forceinline__ int64_t of(int64_t u) const { return ((u + 1) * runs - 1) / units; }
};
constexpr int kLeastRun = 4;
__host__ __device__ __forceinline__ GroupedRuns grouped_runs(int64_t units, int64_t most) {
  const int64_t r = units / kLeastRun;
  return {units, r < 1 ? 1 : r < most ? r : most};
}

template <typename T, int MODE>
struct GroupedWalk {
  using Tr = GroupedTraits<T, MODE>;
  const GroupedCall& c;
  const int *prefix, *begin;    // of each group: tiles (stages in dw) of those before, first row
  int64_t next, end, step;
  int last_g = 0, last_n = 0, last_t = -2;      // of the tile before
  GroupedRuns runs;
  __device__ GroupedWalk(const GroupedCall& call, const int* p, const int* rows) : c(call), prefix(p), begin(rows) {
    if constexpr (MODE == kGradW) {
      runs = grouped_runs((int64_t)prefix[c.groups] * c.tiles_m * c.tiles_n, c.ranges);
      next = end = 0;
      if (runs.units && blockIdx.x < runs.runs) next = runs.begin(blockIdx.x), end = runs.begin(blockIdx.x + 1);
    } else {
      const int64_t all = (int64_t)prefix[c.groups + 1] * c.tiles_n;
      next = c.keep ? blockIdx.x * all / gridDim.x : blockIdx.x, step = c.keep ? 1 : gridDim.x, end = c.keep ? (blockIdx.x + 1) * all / gridDim.x : all;
    }
  }
  static __device__ __forceinline__ int64_t quotient(int64_t a, int b) { return a >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }
  __device__ __forceinline__ int group_of(int t, int n) const {
    int lo = 0, hi = n;         // the last group whose prefix is at most t
    while (hi - lo > 1) {
      const int m = (lo + hi) / 2;
      if (prefix[m] <= t) lo = m; else hi = m;
    }
    return lo;
  }
  // The first part of n stages.
  __device__ __forceinline__ void take_part(GroupedItem* item, int n) const {
    item->stages = Tr::kCuts ? min(n, Tr::kCut) : n;
    item->after = n - item->stages;
  }
  __device__ bool take(GroupedItem* item) {
    if (Tr::kCuts && item->after) {
      item->before += item->stages;
      if constexpr (MODE == kGradW) item->row += (int64_t)item->stages * Tr::kBlock;
      take_part(item, item->after);
      if constexpr (MODE == kGradW) item->rows = (int)min((int64_t)item->stages * Tr::kBlock, begin[item->g + 1] - item->row);
      return true;
    }
    item->before = 0;
    if constexpr (MODE == kGradW) {
      if (next >= end) return false;
      const int total = prefix[c.groups];
      const int tile = (int)quotient(next, total), t = (int)(next - (int64_t)tile * total);
      const int g = group_of(t, c.groups);
      const int64_t n = min(end - next, (int64_t)(prefix[g + 1] - t));
      item->g = g;
      item->row = begin[g] + (int64_t)(t - prefix[g]) * Tr::kBlock;
      take_part(item, (int)n);
      item->rows = (int)min((int64_t)item->stages * Tr::kBlock, begin[g + 1] - item->row);
      item->m0 = tile / c.tiles_n * kTileM;
      item->n0 = tile % c.tiles_n * c.tile_n;
      item->piece = n == prefix[g + 1] - prefix[g] ? -1 : 2 * (int64_t)blockIdx.x + (next != runs.begin(blockIdx.x));
      item->first = (int64_t)tile * total + prefix[g], item->last = (int64_t)tile * total + prefix[g + 1];
      next += n;
      return true;
    } else {
      if (next >= end) return false;
      int t, n, g;
      if (c.keep && last_t >= 0 && last_t + 1 < prefix[last_g + 1]) {      // the next rows of the same weights
        t = last_t + 1, n = last_n, g = last_g;
      } else {
        t = c.tiles_n == 1 ? (int)next : (int)quotient(next, c.tiles_n);
        g = t < prefix[last_g + 1] && !c.keep ? last_g : group_of(t, c.groups + 1);
        n = (int)(next - (int64_t)t * c.tiles_n);
        if (c.keep) {      // a group's tiles column by column, not row by row; the first of each column stand for the change of weights
          const int here = prefix[g + 1] - prefix[g];
          const int64_t at = next - (int64_t)prefix[g] * c.tiles_n;
          n = (int)quotient(at, here), t = (int)(at - (int64_t)n * here);
          if (t < kKeepChange) {
            next += kKeepChange - t, t = kKeepChange;
            if (next >= end) return false;
          }
          t += prefix[g];
        }
      }
      last_t = t, last_n = n, last_g = g;
      item->g = g;
      item->row = begin[g] + (int64_t)(t - prefix[g] - (c.keep ? kKeepChange : 0)) * (c.tile_m * c.halves);
      item->rows = (int)min((int64_t)(c.tile_m * c.halves), begin[g + 1] - item->row);
      item->m0 = 0;
      item->n0 = n * c.tile_n;
      take_part(item, g < c.groups ? (c.num_k + Tr::kBlock * c.deep - 1) / (Tr::kBlock * c.deep) : 0);      // rows of no group: zeros
      item->piece = -1, item->first = item->last = 0;
      next += step;
      return true;
    }
  }
};

// ---- taking fp32 apart --------------------------------------------------------------
struct Pieces {
  uint4 p[3];
};
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }
// The same, cut off by the conversion, which leaves a NaN one that has its bits in its lower half.
__device__ __forceinline__ uint32_t upper_numbers(float lo, float hi) {
  uint32_t r;
  asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float below(float v) { return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ Pieces take_apart(float4 a, float4 b) {
  Pieces r;
  r.p[0] = make_uint4(upper_numbers(a.x, a.y), upper_numbers(a.z, a.w), upper_numbers(b.x, b.y), upper_numbers(b.z, b.w));
#pragma unroll
  for (int k = 1; k < 3; ++k) {
    a = make_float4(below(a.x), below(a.y), below(a.z), below(a.w));
    b = make_float4(below(b.x), below(b.y), below(b.z), below(b.w));
    r.p[k] = make_uint4(upper_halves(a.x, a.y), upper_halves(a.z, a.w), upper_halves(b.x, b.y), upper_halves(b.z, b.w));
  }
  return r;
}
// One operand's stage by a team of 128 threads. Its rows (of 128 bytes as copied) run along the contraction, 8 elements of a row a thread, or
// across it in boxes of 32: 8 elements of one k a thread. Everything is a constant of the thread away from the stage's beginning, and
// nothing is compared: with few warps at work, a stage's time is the latency of its instructions. What lies beyond the operand's rows is taken
// apart with them (the pieces have room for whole rounds) and never used. `valid`: k's from there on are zero.
constexpr int kApartTeam = 128;
template <bool MN, int U, bool CUT>
__device__ __forceinline__ void take_rounds_apart(const char* from, char* to, int piece_bytes, bool zero) {
  float4 lo[U], hi[U];
  const int thread = threadIdx.x % kApartTeam, s = thread & 3, line = thread >> 2;      // a row, or a k
  const int at = line * 128, lo_at = at + (((2 * s) ^ (line & 7)) << 4), hi_at = at + (((2 * s + 1) ^ (line & 7)) << 4);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int box = MN ? (u ^ (line & 1)) * 4096 : u * 4096;
    lo[u] = *(const float4*)(from + lo_at + box), hi[u] = *(const float4*)(from + hi_at + box);
  }
  const int to_at = MN ? line * 128 + ((s ^ (line & 7)) << 4) : line * 64 + ((s ^ ((line >> 1) & 3)) << 4);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (CUT && zero) lo[u] = hi[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const Pieces v = take_apart(lo[u], hi[u]);
    // two rounds make a block of 64 across, of two boxes: of neighbouring k's one is at the first box and one at the second, so that eight lanes
    // read, and write, all banks of a row between them
    char* const p = to + (MN ? (to_at ^ ((u ^ line) & 1) << 6) + (u >> 1) * 4096 : to_at + u * 2048);
#pragma unroll
    for (int k = 0; k < 3; ++k) *(uint4*)(p + k * piece_bytes) = v.p[k];
  }
}
template <bool MN, bool CUT>
__device__ __forceinline__ void take_stage_apart(const char* copied, char* pieces, int n, int piece_bytes, int valid) {
  const bool zero = CUT && (int)(threadIdx.x % kApartTeam >> 2) >= valid;
  const int rounds = MN ? (n + 63) / 64 * 2 : (n + 31) / 32;
  if (rounds == 4) {
    take_rounds_apart<MN, 4, CUT>(copied, pieces, piece_bytes, zero);
  } else if (MN) {
    take_rounds_apart<MN, 2, CUT>(copied, pieces, piece_bytes, zero);
  } else {
    for (int u = 0; u < rounds; ++u) take_rounds_apart<MN, 1, CUT>(copied + u * 4096, pieces + u * 2048, piece_bytes, zero);
  }
}

// Sums over the rows of a stage of dy as copied: of a column (fp32, 128 threads), or over a quarter of the rows of a pair of columns.
template <typename T>
__device__ __forceinline__ void add_columns(const char* stage, int valid, int thread, float (&sum)[2]) {
  constexpr bool kWide = sizeof(T) == 4;
  const int word = kWide ? thread : thread & 63, k0 = kWide ? 0 : (thread >> 6) * 16;
  const char* const from = stage + (word >> 5) * ((kWide ? 32 : 64) * 128) + k0 * 128 + (word & 3) * 4;
  const int slice = (word & 31) >> 2, rows = min(valid - k0, kWide ? 32 : 16);
  const auto add = [](uint32_t v, float& a, float& b) {
    if constexpr (kWide) {
      a += __uint_as_float(v);
    } else if constexpr (Elem<T>::kIsBf16) {
      a += __uint_as_float(v << 16), b += __uint_as_float(v & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*(const __half2*)&v);
      a += f.x, b += f.y;
    }
  };
  if (rows == (kWide ? 32 : 16)) {
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f}, b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k0 = 0; k0 < (kWide ? 32 : 16); k0 += 16) {
      uint32_t v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = *(const uint32_t*)(from + (k0 + k) * 128 + ((slice ^ (k & 7)) << 4));
#pragma unroll
      for (int k = 0; k < 16; ++k) add(v[k], a[k % 4], b[k % 4]);
    }
    sum[0] += (a[0] + a[1]) + (a[2] + a[3]), sum[1] += (b[0] + b[1]) + (b[2] + b[3]);
  } else {
    for (int k = 0; k < rows; ++k) add(*(const uint32_t*)(from + k * 128 + ((slice ^ (k & 7)) << 4)), sum[0], sum[1]);
  }
}

// ---- bringing a tile out -------------------------------------------------------------
// 32 rows of 128 bytes from shared memory to `to`, `rows` of them and of each the first `columns` elements, where rows are no whole 16-byte
// slices: in words as wide as rows are aligned to. Eight words a lane are read before any is stored: the compiler does not know that the
// stores go elsewhere. Not inlined, nor unrolled further: it would take the registers of every tile.
template <typename O, typename W>
__device__ __noinline__ void put_narrow_rows(const char* staging, int lane, O* to, int64_t ld, int rows, int columns) {
  constexpr int kLanes = 128 / sizeof(W) < 32 ? 128 / (int)sizeof(W) : 32, kSide = 32 / kLanes;      // lanes of a row, rows at once
  const int r0 = lane / kLanes;
#pragma unroll 1
  for (int at = lane % kLanes * (int)sizeof(W); at < 128; at += kLanes * (int)sizeof(W)) {
    const int col = at / (int)sizeof(O);
    if (col >= columns) break;
    O* p = to + r0 * ld + col;
#pragma unroll 1
    for (int k0 = r0; k0 < rows; k0 += 8 * kSide) {
      W word[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = k0 + k * kSide;
        word[k] = *(const W*)(staging + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15));
      }
#pragma unroll
      for (int k = 0; k < 8; ++k, p += kSide * ld)
        if (k0 + k * kSide < rows) *(W*)p = word[k];
    }
  }
}
// A warp's 32 rows, 128 bytes of each at a time, through shared memory, so that the stores are whole rows of 128 bytes. Warps that share
// rows take turns. Parts of a sum `before` this one are in carry, where this one is added to them while more come `after`: 128 columns of 16 slices a lane,
// its own.
template <typename T, typename O, int MODE>
__device__ __forceinline__ void store_tile(uint32_t acc, bool empty, char* staging, int lane, int quarter, int turn, int turns, O* out, int64_t ld, int rows,
                                           int columns, const float* bias, uint32_t acc_free, float* carry, int before, int after) {
  using Tr = GroupedTraits<T, MODE>;
  constexpr int kWide = 128 / (int)sizeof(O), kPer = 16 / (int)sizeof(O);
  const int here = min(32, rows - quarter * 32);
  const bool whole = (ld * (int64_t)sizeof(O)) % 16 == 0;
  O* const first = out + (int64_t)quarter * 32 * ld;
  acc += (uint32_t)quarter << 21;
  for (int c0 = turn * kWide; c0 < columns; c0 += turns * kWide) {
    float v[kWide / 32][32];
    if (empty) {
#pragma unroll
      for (int h = 0; h < kWide / 32; ++h)
#pragma unroll
        for (int k = 0; k < 32; ++k) v[h][k] = 0.0f;
    } else {
#pragma unroll
      for (int h = 0; h < kWide / 32; ++h) tmem_load_32(acc + c0 + 32 * h, v[h]);
      if constexpr (Tr::kSplit) {
        float small[32];
        tmem_load_32(acc + Tr::kMostN + c0, small);
        tmem_wait_loads();
        settled(small);
        settled(v[0]);
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float sum = v[0][k] + small[k];
          v[0][k] = sum == sum ? sum : v[0][k];      // infinite, see above
        }
      } else {
        tmem_wait_loads();
#pragma unroll
        for (int h = 0; h < kWide / 32; ++h) settled(v[h]);
      }
      if (acc_free && c0 + turns * kWide >= columns) {      // the tile's sums are read
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) barrier_arrive(acc_free);
      }
      if constexpr (Tr::kCuts) {
        float* const at = carry + c0 * 32;
        if (before)
#pragma unroll
          for (int h = 0; h < kWide / 32; ++h)
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              const float4 p = *(const float4*)(at + (32 * h + k) * 32);
              v[h][k] += p.x, v[h][k + 1] += p.y, v[h][k + 2] += p.z, v[h][k + 3] += p.w;
            }
        if (after) {
#pragma unroll
          for (int h = 0; h < kWide / 32; ++h)
#pragma unroll
            for (int k = 0; k < 32; k += 4) *(float4*)(at + (32 * h + k) * 32) = make_float4(v[h][k], v[h][k + 1], v[h][k + 2], v[h][k + 3]);
          continue;
        }
      }
    }
    if (bias)
#pragma unroll
      for (int h = 0; h < kWide / 32; ++h)
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 b = *(const float4*)(bias + c0 + 32 * h + k);
          v[h][k] += b.x, v[h][k + 1] += b.y, v[h][k + 2] += b.z, v[h][k + 3] += b.w;
        }
#pragma unroll
    for (int s = 0; s < 8; ++s) *(uint4*)(staging + lane * 128 + ((s ^ (lane & 7)) << 4)) = rounded_slice<O>(&v[s * kPer / 32][s * kPer % 32]);
    __syncwarp();
    if (whole) {
      const int s = lane & 7, r1 = lane >> 3, col = c0 + s * kPer;
      O* to = first + (int64_t)r1 * ld + col;
      const char* from = staging + r1 * 128;
      // all of them are read before any is stored: the compiler does not know that the stores go elsewhere
      uint4 slice[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) slice[k] = *(const uint4*)(from + k * 512 + ((s ^ ((4 * k + r1) & 7)) << 4));
      const int rows_left = col < columns ? here - r1 : 0;
#pragma unroll
      for (int k = 0; k < 8; ++k, to += 4 * ld)
        if (4 * k < rows_left) *(uint4*)to = slice[k];
    } else if (ld * (int64_t)sizeof(O) % 8 == 0) {
      put_narrow_rows<O, uint2>(staging, lane, first + c0, ld, here, columns - c0);
    } else if (ld * (int64_t)sizeof(O) % 4 == 0) {
      put_narrow_rows<O, uint32_t>(staging, lane, first + c0, ld, here, columns - c0);
    } else if constexpr (sizeof(O) == 2) {
      put_narrow_rows<O, uint16_t>(staging, lane, first + c0, ld, here, columns - c0);
    }
    __syncwarp();
  }
}

// ---- the kernel ----------------------------------------------------------------------
// 151552 x 256 -> 256 bf16 in 16 groups, us: out 34, dx 35 (HBM: 24; products: 12), dw and db 45 (24; 12) and their join 11.5. Eight tiles a block,
// of which the first waits for the list and the weights and the last is brought out beside nothing: a third of the tensor cores' cycles and 36 to 45 per
// cent of the DRAM's are in use. 495616 x 1024 -> 256 f16 in 4 groups: 260 (194; 159), at 1.05 to 1.3 GHz under the power cap. 67584 x 128 -> 256 fp32 in
// 8 groups: out 40, dx 42, dw and db with their join 53 (HBM: 16, 16, 16; products: 16 each): six products of pieces read 208 KB of shared memory a stage, which bounds it.
// 61 rows in 64 groups, 1024 -> 1024 bf16: 25, the weights of the groups that have rows (13).
template <typename T, int MODE>
__global__ void __launch_bounds__(GroupedTraits<T, MODE>::kThreads, 1)
k_grouped(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ GroupedCall c) {
  using Tr = GroupedTraits<T, MODE>;
  constexpr int kBuffers = 2;
  constexpr bool kMends = MODE == kGradW && !Tr::kSplit;
  extern __shared__ char raw_shared[];
  __shared__ uint64_t full[kMaxStages], free_[kMaxStages], ready[kMaxStages], used[kMaxStages], acc_full[2], acc_free[2], kept_full, kept_free, drained, met;
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up_word, scan[33];
  volatile int* const gave_up = &gave_up_word;
  char* const shared = (char*)(((uintptr_t)raw_shared + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  const bool keep = MODE != kGradW && c.keep;
  // (products read 128 rows of a smaller tile too: what lies behind it in shared memory)
  const int copied_a = MODE == kGradW || Tr::kSplit ? Tr::copied(kTileM, Tr::kMnA) : c.halves * c.tile_m * 128, copied_b = Tr::copied(c.tile_n, Tr::kMnB);
  const int block_bytes = copied_a + (keep ? 0 : copied_b), copied_bytes = c.deep * block_bytes;
  const int piece_a = Tr::piece(kTileM, Tr::kMnA), piece_b = Tr::piece(c.tile_n, Tr::kMnB);
  const int piece_bytes = Tr::kSplit ? 3 * (piece_a + (keep ? 0 : piece_b)) : 0;
  const int kept_stages = keep ? (c.num_k + Tr::kBlock - 1) / Tr::kBlock : 0, kept_bytes = Tr::kSplit ? 3 * piece_b : copied_b;
  char* const copied = shared;
  char* const pieces = copied + (size_t)c.copied_stages * copied_bytes;
  char* const kept = pieces + (size_t)c.piece_stages * piece_bytes;
  char* const staging = kept + (size_t)kept_stages * kept_bytes;
  float* const bias = (float*)(staging + Tr::kOutWarps * 4096);      // of a tile in out; in dw the sums of db that several threads have
  int *const prefix = (int*)(bias + (MODE == kGradW ? 512 : 256)), *const begin = prefix + c.groups + 2;

  if (warp == 1) tmem_alloc(shared_addr(&tmem_slot), 512);
  if (threadIdx.x == 0) {
    for (int k = 0; k < kMaxStages; ++k) {
      barrier_init(shared_addr(full + k), 1);
      barrier_init(shared_addr(free_ + k), (Tr::kSplit ? 4 : 1) + (MODE == kGradW && c.grad_bias ? Tr::kOutWarps : 0));
      barrier_init(shared_addr(ready + k), Tr::kSplit ? 4 : 1);
      barrier_init(shared_addr(used + k), 1);
    }
    for (int k = 0; k < 2; ++k) barrier_init(shared_addr(acc_full + k), 1), barrier_init(shared_addr(acc_free + k), Tr::kOutWarps);
    barrier_init(shared_addr(&kept_full), Tr::kSplit ? 8 : 1);
    barrier_init(shared_addr(&kept_free), 1);
    barrier_init(shared_addr(&drained), 1);
    barrier_init(shared_addr(&met), Tr::kOutWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    gave_up_word = 0;
  }
  wait_for_previous();

  // The groups' first rows, and the tiles (stages) of the groups before each; none at all where the ends are no ends.
  int bad = 0;
  for (int g = threadIdx.x; g <= c.groups; g += Tr::kThreads) {
    const int64_t v = c.offsets[g];
    bad |= v < 0 || v > c.rows || (g == 0 && v != 0);
    begin[g] = (int)min(max(v, (int64_t)0), c.rows);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < c.groups; g += Tr::kThreads) bad |= begin[g + 1] < begin[g];
  bad = __syncthreads_or(bad);
  if (bad && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(c.status, APT_FLAG_BAD_OFFSETS);
  const int lists = MODE == kGradW ? c.groups : c.groups + 1, unit = MODE == kGradW ? Tr::kBlock : c.tile_m * c.halves;      // (the last one: rows of no group)
  int before = 0;
  for (int g0 = 0; g0 < lists; g0 += Tr::kThreads) {
    const int g = g0 + threadIdx.x;
    int total, n = 0;
    if (g < lists && !bad) n = ((g < c.groups ? begin[g + 1] : (int)c.rows) - begin[g] + unit - 1) / unit;
    if (MODE != kGradW && c.keep && n) n += kKeepChange;
    if (lists <= 32) {      // one warp's
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (g < lists) prefix[g + 1] = sum;
    } else {
      const int at = before + block_exclusive_scan(n, scan, &total);
      if (g < lists) prefix[g + 1] = at + n;
      before += total;
    }
  }
  if (threadIdx.x == 0) {
    prefix[0] = 0;
    if (MODE != kGradW) begin[lists] = (int)c.rows;
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = tmem_slot;
  GroupedWalk<T, MODE> walk(c, prefix, begin);
  if (MODE == kGradW && blockIdx.x == 0 && threadIdx.x == 0) c.plan[0] = walk.runs.units, c.plan[1] = walk.runs.runs;
  GroupedItem item;
  bool fine = true;
  if (warp == 0) {
    // ---- copies
    if (one_of_warp()) {
      int stage = 0, loaded = 0, kept_g = -1, kept_n = -1, kept_times = 0;
      uint32_t phase = 0;
      while (fine && walk.take(&item)) {
        const int boxes_a = MODE == kGradW ? (min(kTileM, c.num_m - item.m0) + Tr::kBox - 1) / Tr::kBox : 1;
        const int boxes_b = Tr::kMnB ? (min(c.tile_n, c.num_n - item.n0) + Tr::kBox - 1) / Tr::kBox : 1;
        constexpr int kBoxBytes = Tr::kBlock * 128;
        const uint32_t bytes_b = Tr::kMnB ? boxes_b * kBoxBytes : c.tile_n * 128;
        const int halves = MODE != kGradW && item.rows > c.tile_m ? 2 : 1, blocks = MODE == kGradW ? 0 : (c.num_k + Tr::kBlock - 1) / Tr::kBlock;
        const uint32_t bytes = (MODE == kGradW ? boxes_a * kBoxBytes : halves * c.tile_m * 128) + (keep ? 0 : bytes_b);
        const auto copy_weights = [&](uint32_t b, int k, uint32_t bar) {
          if constexpr (MODE == kOut) {
            copy_box(b, &map_b, k * Tr::kBlock, item.n0, item.g, bar);
          } else {
            for (int i = 0; i < boxes_b; ++i) copy_box(b + i * kBoxBytes, &map_b, item.n0 + i * Tr::kBox, k * Tr::kBlock, item.g, bar);
          }
        };
        if (keep && item.stages && (item.g != kept_g || item.n0 != kept_n)) {
          kept_g = item.g, kept_n = item.n0;
          if constexpr (Tr::kSplit) {      // by the ring, to be taken apart
            for (int k = 0; k < kept_stages; ++k) {
              if (!(fine = barrier_wait(shared_addr(free_ + stage), phase ^ 1, gave_up, c.polls))) break;
              barrier_expect(shared_addr(full + stage), bytes_b);
              copy_weights(shared_addr(copied + (size_t)stage * copied_bytes), k, shared_addr(full + stage));
              ++loaded;
              if (++stage == c.copied_stages) stage = 0, phase ^= 1;
            }
          } else if ((fine = barrier_wait(shared_addr(&kept_free), (kept_times & 1) ^ 1, gave_up, c.polls))) {
            barrier_expect(shared_addr(&kept_full), bytes_b * kept_stages);
            for (int k = 0; k < kept_stages; ++k) copy_weights(shared_addr(kept + (size_t)k * kept_bytes), k, shared_addr(&kept_full));
            ++kept_times;
          }
          if (!fine) break;
        }
        for (int k = 0; k < item.stages; ++k) {
          if (!(fine = barrier_wait(shared_addr(free_ + stage), phase ^ 1, gave_up, c.polls))) break;
          const uint32_t bar = shared_addr(full + stage);
          uint32_t a = shared_addr(copied + (size_t)stage * copied_bytes), b = a + copied_a;
          if constexpr (MODE == kGradW) {
            barrier_expect(bar, bytes);
            const int row = (int)item.row + k * Tr::kBlock;
            for (int i = 0; i < boxes_a; ++i) copy_box(a + i * kBoxBytes, &map_a, item.m0 + i * Tr::kBox, row, bar);
            for (int i = 0; i < boxes_b; ++i) copy_box(b + i * kBoxBytes, &map_b, item.n0 + i * Tr::kBox, row, bar);
          } else {
            const int first = (item.before + k) * c.deep, last = min(first + c.deep, blocks);
            barrier_expect(bar, bytes * (last - first));
            for (int l = first; l < last; ++l, a += block_bytes, b += block_bytes) {
              copy_box(a, &map_a, l * Tr::kBlock, (int)item.row, bar);
              if (halves == 2) copy_box(a + kTileM * 128, &map_a, l * Tr::kBlock, (int)item.row + kTileM, bar);
              if (!keep) copy_weights(b, l, bar);
            }
          }
          ++loaded;
          if (++stage == c.copied_stages) stage = 0, phase ^= 1;
        }
      }
      // copies on their way land before the block ends, also where somebody has given up, or will behind the last copy
      for (int k = max(0, loaded - c.copied_stages); k < loaded; ++k) barrier_settle(shared_addr(full + k % c.copied_stages), (k / c.copied_stages) & 1);
      if (kept_times) barrier_settle(shared_addr(&kept_full), (kept_times - 1) & 1);
    }
  } else if (warp == 1) {
    // ---- products
    if (one_of_warp()) {
      const int stages = Tr::kSplit ? c.piece_stages : c.copied_stages;
      const uint32_t what = product_descriptor(!std::is_same<T, __half>::value, Tr::kMnA, Tr::kMnB, kTileM, c.tile_n);
      const uint32_t start = shared_addr(Tr::kSplit ? pieces : copied), start_b = keep ? shared_addr(kept) : start + (Tr::kSplit ? 3 * piece_a : copied_a);
      const uint32_t stage_units = (Tr::kSplit ? piece_bytes : copied_bytes) >> 4;
      const uint64_t first_a = Tr::kMnA ? tile_descriptor(start, Tr::kBlock * 128, 1024, kSwizzle128)
                                        : tile_descriptor(start, 16, Tr::kBlock * 16, Tr::kSplit ? kSwizzle64 : kSwizzle128);
      const uint64_t first_b = Tr::kMnB ? tile_descriptor(start_b, Tr::kBlock * 128, 1024, kSwizzle128)
                                        : tile_descriptor(start_b, 16, Tr::kBlock * 16, Tr::kSplit ? kSwizzle64 : kSwizzle128);
      int stage = 0, kept_g = -1, kept_n = -1, kept_times = 0, buffer = kBuffers - 1;
      uint32_t phase = 0, mended = 0, turns = 0;      // turns: parity of each buffer's uses
      while (fine && walk.take(&item)) {
        if (!item.stages) continue;
        const int halves = MODE != kGradW && item.rows > c.tile_m ? 2 : 1;
        buffer = c.halves == 2 || buffer == kBuffers - 1 ? 0 : buffer + 1;
        if (!(fine = barrier_wait(shared_addr(acc_free + buffer), turns >> buffer & 1 ^ 1, gave_up, c.polls))) break;
        if (halves == 2 && !(fine = barrier_wait(shared_addr(acc_free + 1), turns >> 1 & 1 ^ 1, gave_up, c.polls))) break;
        turns ^= halves == 2 ? 3 : 1 << buffer;
        if (keep && (item.g != kept_g || item.n0 != kept_n)) {
          kept_g = item.g, kept_n = item.n0;
          if (kept_times) products_done(shared_addr(&kept_free));
          if (!(fine = barrier_wait(shared_addr(&kept_full), kept_times & 1, gave_up, c.polls))) break;
          ++kept_times;
        }
        const uint32_t acc = tmem + buffer * kAccColumns;
        for (int k = 0; k < item.stages; ++k) {
          if (!(fine = barrier_wait(shared_addr((Tr::kSplit ? ready : full) + stage), phase, gave_up, c.polls))) break;
          const int left = MODE == kGradW ? item.rows - k * Tr::kBlock : c.num_k - (item.before + k) * Tr::kBlock * c.deep, steps = (min(left, Tr::kBlock * c.deep) + 15) / 16;
          if (kMends && left < Tr::kBlock && left % 16) {
            barrier_arrive(shared_addr(ready));
            if (!(fine = barrier_wait(shared_addr(ready + 1), mended, gave_up, c.polls))) break;
            mended ^= 1;
          }
          tmem_fence_after();
          const uint64_t tile_a = first_a + (uint32_t)stage * stage_units, tile_b = keep ? first_b + (uint32_t)k * (uint32_t)(kept_bytes >> 4) : first_b + (uint32_t)stage * stage_units;
          const auto step = [&](uint64_t tile_a, uint64_t tile_b, int s, bool add) {
            const uint64_t da = tile_a + s * ((Tr::kMnA ? 2048 : 32) >> 4), db = tile_b + s * ((Tr::kMnB ? 2048 : 32) >> 4);
            tile_product(acc, da, db, what, add);
            if (!Tr::kSplit && MODE != kGradW && halves == 2) tile_product(acc + kAccColumns, da + (kTileM * 128 >> 4), db, what, add);
            if constexpr (Tr::kSplit) {
              const uint64_t pa = piece_a >> 4, pb = piece_b >> 4;
              const uint32_t small = acc + Tr::kMostN;
              tile_product(small, da, db + pb, what, add);
              tile_product(small, da + pa, db, what, true);
              tile_product(small, da + pa, db + pb, what, true);
              tile_product(small, da, db + 2 * pb, what, true);
              tile_product(small, da + 2 * pa, db, what, true);
            }
          };
          constexpr int kSteps = Tr::kBlock / 16;
          for (int l = 0; l < (Tr::kSplit || MODE == kGradW ? 1 : c.deep) && l * kSteps < steps; ++l) {
            const uint64_t at_a = tile_a + (uint32_t)l * (uint32_t)(block_bytes >> 4), at_b = tile_b + (uint32_t)l * (uint32_t)(block_bytes >> 4);
            if (steps >= (l + 1) * kSteps) {
#pragma unroll
              for (int s = 0; s < kSteps; ++s) step(at_a, at_b, s, k > 0 || l > 0 || s > 0);
            } else {
              for (int s = 0; s < steps - l * kSteps; ++s) step(at_a, at_b, s, k > 0 || l > 0 || s > 0);
            }
          }
          products_done(shared_addr((Tr::kSplit ? used : free_) + stage));
          if (k == item.stages - 1) {
            products_done(shared_addr(acc_full + buffer));
            if (halves == 2) products_done(shared_addr(acc_full + 1));
          }
          if (++stage == stages) stage = 0, phase ^= 1;
        }
      }
      products_done(shared_addr(&drained));      // (as the copies)
      barrier_settle(shared_addr(&drained), 0);
    }
  } else if (kMends && warp == 2) {
    // ---- rows of the next group in the last stage of a sum: zeros, in both operands, when the products get there and ask for it (ready[0], answered by
    // ready[1]: both sides count the same stages)
    int64_t before_item = 0;
    uint32_t mended = 0;
    while (fine && walk.take(&item)) {
      const int64_t last = before_item + item.stages - 1;
      before_item += item.stages;
      if (item.rows % 16 == 0) continue;
      const int stage = (int)(last % c.copied_stages), valid = item.rows - (item.stages - 1) * Tr::kBlock;
      if (!(fine = __all_sync(0xffffffffu, barrier_wait(shared_addr(ready), mended, gave_up, c.polls)))) break;
      mended ^= 1;
      char* const base = copied + (size_t)stage * copied_bytes;
      const int slices = ((valid + 15) / 16 * 16 - valid) * 8, blocks = copied_bytes / 8192;
      for (int i = lane; i < slices * blocks; i += 32) *(uint4*)(base + i / slices * 8192 + valid * 128 + i % slices * 16) = make_uint4(0u, 0u, 0u, 0u);
      fence_for_tensor_cores();
      __syncwarp();
      if (lane == 0) barrier_arrive(shared_addr(ready + 1));
    }
  } else if (warp >= 4 && (warp < 8 || !Tr::kSplit)) {
    // ---- finished tiles
    const int quarter = warp % 4, turn = warp >= 8, thread = turn * 128 + threadIdx.x % 128;
    constexpr int kTurns = Tr::kOutWarps / 4;
    char* const mine = staging + (turn * 4 + quarter) * 4096;
    int summed = 0;
    uint32_t summed_phase = 0;
    int bias_g = -1, bias_n = -1, buffer = kBuffers - 1;
    uint32_t turns = 0, meetings = 0;
    float sum[2] = {0.0f, 0.0f};      // of columns of dy
    float* const carry = Tr::kCuts ? c.carry + ((int64_t)blockIdx.x * 4 + quarter) * 32 * Tr::kMostN + lane * 4 : nullptr;
    const auto meet = [&] {      // of the warps here; false: somebody has given up
      __syncwarp();
      if (lane == 0) barrier_arrive(shared_addr(&met));
      const bool all = __all_sync(0xffffffffu, barrier_wait(shared_addr(&met), meetings, gave_up, c.polls));
      meetings ^= 1;
      return all;
    };
    while (fine && walk.take(&item)) {
      const bool empty = item.stages == 0;
      const int columns = min(c.tile_n, c.num_n - item.n0);
      if (MODE == kOut && c.bias && !empty && (item.g != bias_g || item.n0 != bias_n)) {
        bias_g = item.g, bias_n = item.n0;
        if (!(fine = meet())) break;      // the tile before is out
        for (int k = thread; k < 256; k += Tr::kOutWarps * 32)
          bias[k] = bias_n + k < c.num_n ? Elem<T>::to_f(((const T*)c.bias)[(int64_t)bias_g * c.num_n + bias_n + k]) : 0.0f;
        if (!(fine = meet())) break;
      }
      float column = 0.0f;      // of db
      if constexpr (MODE == kGradW) {
        if (c.grad_bias) {
          // the columns of dy, while the products are made of them: as products with ones they took a third of the time of a stage
          if (!item.before) sum[0] = sum[1] = 0.0f;
          for (int k = 0; k < item.stages; ++k) {
            if (!(fine = __all_sync(0xffffffffu, barrier_wait(shared_addr(full + summed), summed_phase, gave_up, c.polls)))) break;
            const int valid = item.rows - k * Tr::kBlock;
            if (item.n0 == 0) add_columns<T>(copied + (size_t)summed * copied_bytes, valid, thread, sum);
            __syncwarp();
            if (lane == 0) barrier_arrive(shared_addr(free_ + summed));
            if (++summed == c.copied_stages) summed = 0, summed_phase ^= 1;
          }
          if (!fine) break;
          column = sum[0];
          if constexpr (!Tr::kSplit) {      // four threads have a pair of columns
            if (item.n0 == 0 && !item.after) {
              if (!(fine = meet())) break;
              *(float2*)(bias + (thread >> 6) * 128 + (thread & 63) * 2) = make_float2(sum[0], sum[1]);
              if (!(fine = meet())) break;
              const int m = thread & 127;
              column = (bias[m] + bias[128 + m]) + (bias[256 + m] + bias[384 + m]);
            }
          }
        }
      }
      const int halves = MODE != kGradW && item.rows > c.tile_m ? 2 : 1;
      for (int half = 0; half < halves; ++half) {
        if (!empty) {
          buffer = c.halves == 2 ? half : buffer == kBuffers - 1 ? 0 : buffer + 1;
          fine = __all_sync(0xffffffffu, barrier_wait(shared_addr(acc_full + buffer), turns >> buffer & 1, gave_up, c.polls));
          if (!fine) break;
          turns ^= 1u << buffer;
          tmem_fence_after();
        }
        const uint32_t acc = tmem + buffer * kAccColumns;
        if constexpr (MODE == kGradW) {
          const int rows = min(kTileM, c.num_m - item.m0), m = quarter * 32 + lane;
          if (quarter * 32 < rows) {
            if (item.piece < 0 || item.after)
              store_tile<T, T, MODE>(acc, empty, mine, lane, quarter, turn, kTurns, (T*)c.out + ((int64_t)item.g * c.num_m + item.m0) * c.num_n + item.n0,
                                     (int64_t)c.num_n, rows, columns, nullptr, 0u, carry, item.before, item.after);
            else
              store_tile<T, float, MODE>(acc, empty, mine, lane, quarter, turn, kTurns, c.partial + item.piece * kTileM * c.tile_n, (int64_t)c.tile_n, rows,
                                         columns, nullptr, 0u, carry, item.before, item.after);
            if (c.grad_bias && item.n0 == 0 && turn == 0 && !item.after) {
              if (m < rows) {
                if (item.piece < 0) ((T*)c.grad_bias)[(int64_t)item.g * c.num_m + item.m0 + m] = Elem<T>::from_f(column);
                else c.partial_bias[item.piece * kTileM + m] = column;
              }
            }
          }
        }
        const int rows = item.rows - half * kTileM;
        const bool stores = MODE != kGradW && quarter * 32 < min(rows, c.tile_m) && turn * (128 / (int)sizeof(T)) < columns;
        if (stores)
          store_tile<T, T, MODE>(acc, empty, mine, lane, quarter, turn, kTurns, (T*)c.out + (item.row + half * kTileM) * c.num_n + item.n0, (int64_t)c.num_n,
                                 min(rows, c.tile_m), columns, MODE == kOut && c.bias && !empty ? bias : nullptr, shared_addr(acc_free + buffer), carry, item.before, item.after);
        if (!empty && !stores) {
          tmem_fence_before();
          __syncwarp();
          if (lane == 0) barrier_arrive(shared_addr(acc_free + buffer));
        }
      }
    }
  } else if (MODE == kGradW && warp == 3) {
    // ---- the plan of the block's run, which follows from the walk and waits for nothing: k_join_weights reads it whoever gives up
    if (lane == 0 && walk.take(&item)) {
      const int64_t run = blockIdx.x;
      int64_t* const to = c.plan + 2 + kPlanWords * run;
      to[0] = (int64_t)(item.m0 / kTileM * c.tiles_n + item.n0 / c.tile_n) * c.groups + item.g, to[1] = item.first;
      to[2] = walk.runs.begin(run), to[3] = run ? walk.runs.begin(run - 1) : 0, to[4] = walk.runs.of(item.last - 1);
    }
    // ---- groups without rows
    const int64_t per = (int64_t)c.num_m * c.num_n;
    const bool slices = per * sizeof(T) % 16 == 0;
    const int64_t from = (int64_t)blockIdx.x * 32 + lane, by = (int64_t)gridDim.x * 32;
    for (int g = 0; g < c.groups; ++g) {
      if (prefix[g + 1] > prefix[g]) continue;
      T* const out = (T*)c.out + g * per;
      if (slices)
        for (int64_t i = from; i < per * (int64_t)sizeof(T) / 16; i += by) *((uint4*)out + i) = make_uint4(0u, 0u, 0u, 0u);
      else
        for (int64_t i = from; i < per; i += by) out[i] = Elem<T>::from_f(0.0f);
      if (c.grad_bias)
        for (int64_t i = from; i < c.num_m; i += by) ((T*)c.grad_bias)[(int64_t)g * c.num_m + i] = Elem<T>::from_f(0.0f);
    }
  } else if (Tr::kSplit && warp >= 8) {
    // ---- fp32 taken apart, by two teams in turn: one's waits and fence are the other's work
    const int team = (warp - 8) / 4;
    int from = 0, kept_g = -1, kept_n = -1, kept_times = 0, turn = 0;
    uint32_t from_phase = 0, uses = 0;      // uses: parity of the team's stage of pieces
    const auto next_from = [&] {
      if (++from == c.copied_stages) from = 0, from_phase ^= 1;
    };
    while (fine && walk.take(&item)) {
      if (keep && item.stages && (item.g != kept_g || item.n0 != kept_n)) {
        kept_g = item.g, kept_n = item.n0;
        fine = __all_sync(0xffffffffu, barrier_wait(shared_addr(&kept_free), (kept_times & 1) ^ 1, gave_up, c.polls));
        ++kept_times;
        for (int k = 0; fine && k < kept_stages; ++k, next_from()) {
          // the other team's stages too: a wait for a phase is one only where the phase before is known to be over
          if (!(fine = __all_sync(0xffffffffu, barrier_wait(shared_addr(full + from), from_phase, gave_up, c.polls)))) break;
          if ((k & 1) != team) continue;
          take_stage_apart<Tr::kMnB, false>(copied + (size_t)from * copied_bytes, kept + (size_t)k * kept_bytes, c.tile_n, piece_b, Tr::kBlock);
          __syncwarp();
          if (lane == 0) barrier_arrive(shared_addr(free_ + from));
        }
        if (!fine) break;
        fence_for_tensor_cores();
        __syncwarp();
        if (lane == 0) barrier_arrive(shared_addr(&kept_full));
      }
      for (int k = 0; k < item.stages; ++k, turn ^= 1, next_from()) {
        if (turn != team) continue;      // each team has a stage of pieces of its own
        // first the products of the team's stage before: they came behind those of all earlier ones, so that what the ring's place held before
        // has arrived, and the wait for its next phase is one
        fine = __all_sync(0xffffffffu, barrier_wait(shared_addr(used + team), uses ^ 1, gave_up, c.polls) && barrier_wait(shared_addr(full + from), from_phase, gave_up, c.polls));
        if (!fine) break;
        const char* const in = copied + (size_t)from * copied_bytes;
        char* const out = pieces + (size_t)team * piece_bytes;
        const int valid = MODE == kGradW ? item.rows - k * Tr::kBlock : Tr::kBlock;
        if (MODE == kGradW && valid < Tr::kBlock) {
          take_stage_apart<Tr::kMnA, true>(in, out, kTileM, piece_a, valid);
          take_stage_apart<Tr::kMnB, true>(in + copied_a, out + 3 * piece_a, c.tile_n, piece_b, valid);
        } else {
          take_stage_apart<Tr::kMnA, false>(in, out, MODE == kGradW ? kTileM : c.tile_m, piece_a, valid);
          if (!keep) take_stage_apart<Tr::kMnB, false>(in + copied_a, out + 3 * piece_a, c.tile_n, piece_b, valid);
        }
        fence_for_tensor_cores();
        __syncwarp();
        if (lane == 0) {
          barrier_arrive(shared_addr(free_ + from));
          barrier_arrive(shared_addr(ready + team));
        }
        uses ^= 1;
      }
    }
  }
  tmem_fence_before();
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 512);
  if (threadIdx.x == 0 && *gave_up) atomicOr(c.status, APT_FLAG_COPY_TIMEOUT);
}

// The partial sums of dw and db that make up one, in the order of the rows. A run that begins within a sum says so in the plan; the first
// such run of a sum has it joined: blocks (part of the tile, run). 147 runs of 256 x 256: 11.5 us for 38 MB out of L2, of which half is the launch
// and the look at the plan.
template <typename T>
__global__ void __launch_bounds__(256)
k_join_weights(const __grid_constant__ GroupedCall c) {
  wait_for_previous();
  const int64_t v = blockIdx.y + 1;
  if (v >= c.plan[1]) return;
  const int64_t *const from = c.plan + 2 + kPlanWords * v, what = from[0], first = from[1], here = from[2], before = from[3], r1 = from[4];
  // a run that begins with a sum has nothing to join it to; an earlier run that begins within this sum does it
  if (here <= first || before > first) return;
  const int tile = (int)(what / c.groups), g = (int)(what - (int64_t)tile * c.groups), m0 = tile / c.tiles_n * kTileM, n0 = tile % c.tiles_n * c.tile_n;
  const int64_t piece = 2 * (v - 1) + (before < first);
  const int slices = c.tile_n / 4;
  const int64_t size = (int64_t)kTileM * c.tile_n;
  // a sixteenth of the rows, four slices a thread at once
  const int i1 = (blockIdx.x + 1) * (kTileM / kJoinParts) * slices;
  for (int i0 = blockIdx.x * (kTileM / kJoinParts) * slices + threadIdx.x; i0 < i1; i0 += 4 * 256) {
    float4 sum[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u * 256 < i1) sum[u] = *(const float4*)(c.partial + piece * size + (int64_t)(i0 + u * 256) * 4);
    for (int64_t r = v; r <= r1; ++r) {
      float4 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * 256 < i1) p[u] = *(const float4*)(c.partial + 2 * r * size + (int64_t)(i0 + u * 256) * 4);
#pragma unroll
      for (int u = 0; u < 4; ++u) sum[u].x += p[u].x, sum[u].y += p[u].y, sum[u].z += p[u].z, sum[u].w += p[u].w;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * 256, m = i / slices, n = i % slices * 4;
      if (i >= i1 || m0 + m >= c.num_m || n0 + n >= c.num_n) continue;
      T* const to = (T*)c.out + ((int64_t)g * c.num_m + m0 + m) * c.num_n + n0 + n;
      const float s[4] = {sum[u].x, sum[u].y, sum[u].z, sum[u].w};
      if (c.num_n % 4 == 0) {
        store_all<T, 4>(to, s);
      } else {
        for (int k = 0; k < 4; ++k)
          if (n0 + n + k < c.num_n) to[k] = Elem<T>::from_f(s[k]);
      }
    }
  }
  const int i = threadIdx.x;
  if (c.grad_bias && n0 == 0 && blockIdx.x == 0 && i < kTileM && m0 + i < c.num_m) {
    float sum = c.partial_bias[piece * kTileM + i];
    for (int64_t r = v; r <= r1; ++r) sum += c.partial_bias[2 * r * kTileM + i];
    ((T*)c.grad_bias)[(int64_t)g * c.num_m + m0 + i] = Elem<T>::from_f(sum);
  }
}

// db without dw: 32 columns of a group a block. 151552 x 256 bf16 in 16 groups 20 us (HBM: 12), 32 warps with eight rows each
// on their way; eight with one each took 97.
template <typename T>
__global__ void __launch_bounds__(1024)
k_bias_sums(const T* __restrict__ grad, int64_t rows, int64_t out_dim, const int64_t* __restrict__ offsets, T* __restrict__ grad_bias, int32_t* status) {
  wait_for_previous();
  __shared__ float part[32][33];
  const int g = blockIdx.y, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (threadIdx.x == 0 && blockIdx.x == 0 && bad_group(offsets, g, rows)) atomicOr(status, APT_FLAG_BAD_OFFSETS);
  const RowRange r = group_rows(offsets, g, rows);
  const int64_t n = (int64_t)blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (n < out_dim)
    for (int64_t row = r.begin + warp; row < r.end; row += 8 * 32) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = row + 32 * k < r.end ? Elem<T>::to_f(grad[(row + 32 * k) * out_dim + n]) : 0.0f;
      sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && n < out_dim) {
    for (int k = 1; k < 32; ++k) sum += part[k][lane];
    grad_bias[g * out_dim + n] = Elem<T>::from_f(sum);
  }
}

// ---- host side -----------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// A matrix of `rows` rows as the copies read it: in whole 16-byte slices, `pitch` elements apart.
struct Operand {
  const void* data;
  int64_t stack, rows, columns, pitch;
};
static int make_map(CUtensorMap* map, int dtype, const Operand& o, int box_columns, int box_rows) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) {
    set_error("grouped_linear: the driver has no cuTensorMapEncodeTiled");
    return APT_ERR_CUDA;
  }
  const size_t size = dtype == APT_F32 ? 4 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)o.columns, (cuuint64_t)o.rows, (cuuint64_t)o.stack};
  const cuuint64_t strides[2] = {(cuuint64_t)(o.pitch * size), (cuuint64_t)(o.rows * o.pitch * size)};
  const cuuint32_t box[3] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows, 1}, ones[3] = {1, 1, 1};
  const auto made = [&] {
    return encode(map, dtype == APT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == APT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                  o.stack ? 3 : 2, (void*)o.data, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = made();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {      // a thread (the autograd engine's, say) that has not called the runtime yet
    int device;
    APT_CUDA(cudaGetDevice(&device));
    APT_CUDA(cudaSetDevice(device));
    r = made();
  }
  if (r != CUDA_SUCCESS) {
    set_error("grouped_linear: cuTensorMapEncodeTiled -> %d (%lld x %lld, pitch %lld)", (int)r, (long long)o.rows, (long long)o.columns, (long long)o.pitch);
    return APT_ERR_CUDA;
  }
  return APT_OK;
}

static int64_t pitch_of(int64_t columns, size_t size) { return widened_dim(columns, size); }
static size_t room_of(int64_t rows, int64_t columns, size_t size) {
  const int64_t pitch = pitch_of(columns, size);
  return pitch == columns ? 0 : align_up((size_t)rows * pitch * size, 256);
}
// The matrix, or a copy of it in whole slices in front of *room.
static int laid_out(const void* data, int64_t stack, int64_t rows, int64_t columns, size_t size, char** room, Operand* o, cudaStream_t s) {
  *o = {data, stack, rows, columns, pitch_of(columns, size)};
  if (o->pitch == columns) return APT_OK;
  const int64_t all = rows * std::max<int64_t>(stack, 1);
  if (const int e = widen_rows(data, all, columns * size, *room, s)) return e;
  o->data = *room;
  *room += room_of(all, columns, size);
  return APT_OK;
}

// Columns of a tile: as few tiles as can be, of the same width.
static int tile_columns(int64_t n, int most) { return (int)(ceil_div(ceil_div(n, ceil_div(n, most)), 16) * 16); }

// Runs of stages that dw is cut into at most, one for every block, and partial sums that come of it.
struct WeightPlan {
  int tile_n, tiles_m, tiles_n;
  int64_t ranges, pieces;
};
template <typename T>
static WeightPlan weight_plan(int64_t rows, int64_t dim, int64_t out_dim, int64_t groups) {
  using Tr = GroupedTraits<T, kGradW>;
  WeightPlan p;
  p.tile_n = tile_columns(dim, Tr::kMostN);
  p.tiles_m = (int)ceil_div(out_dim, kTileM);
  p.tiles_n = (int)ceil_div(dim, p.tile_n);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n, most = (ceil_div(rows, Tr::kBlock) + groups) * tiles;
  p.ranges = grouped_runs(most, kNumSMs).runs;
  p.pieces = 2 * p.ranges;
  return p;
}

// The blocks' tiles of sums that are brought out in parts.
template <typename T>
static size_t carry_room(int64_t rows, int64_t dim, int64_t out_dim, bool backward) {
  using Tr = GroupedTraits<T, kGradW>;
  const int64_t terms = (int64_t)Tr::kCut * Tr::kBlock;
  const bool cut = backward ? rows > terms || (Tr::kSplit && out_dim > terms) : Tr::kSplit && dim > terms;
  return cut ? (size_t)kNumSMs * kTileM * Tr::kMostN * 4 : 0;
}

template <typename T, int MODE>
static int launch_grouped(GroupedCall c, const CUtensorMap& a, const CUtensorMap& b, int64_t items, cudaStream_t s) {
  using Tr = GroupedTraits<T, MODE>;
  const int lists = 1024 + (MODE == kGradW ? 2048 : 1024) + (int)align_up((size_t)(c.groups + 2) * 8, 16);
  const int room = kMostShared - lists - Tr::kOutWarps * 4096;
  int copied = MODE == kGradW || Tr::kSplit ? Tr::copied(kTileM, Tr::kMnA) : c.tile_m * 128, pieces = Tr::kSplit ? 3 * Tr::piece(kTileM, Tr::kMnA) : 0, kept = 0;
  const int copied_b = Tr::copied(c.tile_n, Tr::kMnB), pieces_b = Tr::kSplit ? 3 * Tr::piece(c.tile_n, Tr::kMnB) : 0;
  // Weights are kept where they leave room for four stages of rows and a block has several tiles of them: what the copies bring from L2, which
  // gives 10 to 12 TB/s, is then the rows alone.
  if (MODE != kGradW) {
    const int64_t bytes = ceil_div(c.num_k, Tr::kBlock) * (Tr::kSplit ? pieces_b : copied_b), least = Tr::kSplit ? 2 * pieces + 3 * copied : 4 * copied;
    c.keep = bytes + least <= room && items >= 3 * kNumSMs && items >= 3 * (int64_t)c.groups * c.tiles_n;
    if (c.keep) kept = (int)bytes;
  }
  c.halves = c.deep = 1, c.polls = bulk_wait_polls();
  if (MODE != kGradW && !Tr::kSplit && !c.keep) {
    // Two tiles of rows share the weights of a stage where groups are long and the contraction is: the weights come half as often, and bringing
    // tiles out beside the products, which both halves of tensor memory are taken from, is what a long contraction needs least.
    if (c.tile_m == kTileM && c.num_k >= 512 && c.rows >= (int64_t)c.groups * 4 * kTileM && items >= 4 * kNumSMs) c.halves = 2, items /= 2;
    // Small stages are two blocks of the contraction deep: a stage costs its waits whatever it holds.
    else if (c.num_k > Tr::kBlock && 2 * (copied + copied_b) <= 48 * 1024) c.deep = 2;
  }
  if (!c.keep) copied += copied_b, pieces += pieces_b;
  if (c.halves == 2) copied += kTileM * 128;
  copied *= c.deep;
  c.piece_stages = Tr::kSplit ? 2 : 0;
  c.copied_stages = std::min(kMaxStages, (room - kept - c.piece_stages * pieces) / copied);
  const int bytes = lists + Tr::kOutWarps * 4096 + kept + c.copied_stages * copied + c.piece_stages * pieces;
  static bool sized[64] = {};
  int dev = 0;
  APT_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !sized[dev]) {
    APT_CUDA(cudaFuncSetAttribute(k_grouped<T, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
    if (dev < 64) sized[dev] = true;
  }
  // over half of an SM's shared memory, so that no two blocks share one: each takes all of its tensor memory
  APT_FOLLOW((k_grouped<T, MODE>), std::min<int64_t>(items, kNumSMs), Tr::kThreads, std::max(bytes, 116 * 1024), s, a, b, c);
  return APT_OK;
}

template <typename T>
static int code_of() { return sizeof(T) == 4 ? APT_F32 : std::is_same<T, __half>::value ? APT_F16 : APT_BF16; }

// Rows against weights: out (contraction along w's rows) or dx (across them).
template <typename T, int MODE>
static int rows_product(const Operand& rows, const Operand& weight, int64_t num_n, const void* bias, const int64_t* offsets, int groups, void* out,
                        char* carry, int32_t* status, cudaStream_t s) {
  using Tr = GroupedTraits<T, MODE>;
  GroupedCall c = {};
  c.offsets = offsets, c.rows = rows.rows, c.groups = groups;
  c.num_n = (int)num_n, c.num_k = (int)rows.columns;
  // Tiles of 128 rows, or as many as a mean group has twice over, are made smaller, down to 16 rows and 64 columns, while every tile is still
  // another SM's (or two of them are one's, where rows are few and the time is that of reading the weights). The products are of 128 rows
  // always: rows that are not copied are not written either, so that only copies and conversions get fewer.
  int64_t most = Tr::kMostN;
  const auto tiles = [&](int64_t m, int64_t n) { return (ceil_div(rows.rows, m) + std::min<int64_t>(groups, rows.rows) / 2) * ceil_div(num_n, n); };
  c.tile_m = kTileM;
  while (c.tile_m > 16 && c.tile_m >= 2 * ceil_div(rows.rows, groups)) c.tile_m /= 2;
  const int64_t enough = c.tile_m < 64 ? 2 * kNumSMs : kNumSMs;
  for (;;) {
    const bool columns = most > 64 && (most >= 2 * c.tile_m || c.tile_m == 16);
    const int64_t m = columns ? c.tile_m : c.tile_m / 2, n = columns ? most / 2 : most;
    if (m < 16 || tiles(m, n) > enough) break;
    c.tile_m = (int)m, most = n;
  }
  c.tile_n = tile_columns(num_n, (int)most), c.tiles_n = (int)ceil_div(num_n, c.tile_n);
  c.a = rows.data, c.b = weight.data, c.pitch_a = rows.pitch, c.pitch_b = weight.pitch;
  c.bias = bias, c.out = out, c.carry = (float*)carry, c.status = status;
  CUtensorMap a, b;
  if (const int e = make_map(&a, code_of<T>(), rows, Tr::kBox, c.tile_m)) return e;
  if (const int e = make_map(&b, code_of<T>(), weight, Tr::kBox, MODE == kOut ? c.tile_n : Tr::kBlock)) return e;
  return launch_grouped<T, MODE>(c, a, b, (ceil_div(rows.rows, c.tile_m) + groups + 1) * c.tiles_n, s);
}

template <typename T>
static int linear_forward(const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t out_dim, const int64_t* offsets, int groups,
                          void* out, char* room, int32_t* status, cudaStream_t s) {
  char* const carry = room;
  room += carry_room<T>(rows, dim, out_dim, false);
  Operand a, w;
  if (const int e = laid_out(x, 0, rows, dim, sizeof(T), &room, &a, s)) return e;
  if (const int e = laid_out(weight, groups, out_dim, dim, sizeof(T), &room, &w, s)) return e;
  return rows_product<T, kOut>(a, w, out_dim, bias, offsets, groups, out, carry, status, s);
}

template <typename T>
static size_t linear_room(int64_t rows, int64_t dim, int64_t out_dim, int64_t groups, bool backward) {
  size_t bytes = carry_room<T>(rows, dim, out_dim, backward) + room_of(rows, dim, sizeof(T)) + room_of(groups * out_dim, dim, sizeof(T));
  if (backward) {
    const WeightPlan p = weight_plan<T>(rows, dim, out_dim, groups);
    bytes += room_of(rows, out_dim, sizeof(T)) + align_up((size_t)(2 + kPlanWords * p.ranges) * 8, 256) + (size_t)p.pieces * kTileM * (p.tile_n + 1) * 4;
  }
  return bytes;
}

template <typename T>
static int linear_backward(const void* x, int64_t rows, int64_t dim, const void* weight, int64_t out_dim, const int64_t* offsets, int groups,
                           const void* grad, void* grad_x, void* grad_weight, void* grad_bias, char* room, int32_t* status, cudaStream_t s) {
  if (grad_bias && !grad_weight) {
    const dim3 grid((unsigned)ceil_div(out_dim, 32), (unsigned)groups);
    APT_FOLLOW((k_bias_sums<T>), grid, 1024, 0, s, (const T*)grad, rows, out_dim, offsets, (T*)grad_bias, status);
  }
  if (rows == 0) {
    if (grad_weight) APT_CUDA(cudaMemsetAsync(grad_weight, 0, (size_t)groups * out_dim * dim * sizeof(T), s));
    if (grad_weight && grad_bias) APT_CUDA(cudaMemsetAsync(grad_bias, 0, (size_t)groups * out_dim * sizeof(T), s));
    return look_at_ends(offsets, groups, 0, status, s);
  }
  if (!grad_x && !grad_weight) return APT_OK;
  char* const carry = room;
  room += carry_room<T>(rows, dim, out_dim, true);
  Operand dy;
  if (const int e = laid_out(grad, 0, rows, out_dim, sizeof(T), &room, &dy, s)) return e;
  if (grad_x) {
    Operand w;
    if (const int e = laid_out(weight, groups, out_dim, dim, sizeof(T), &room, &w, s)) return e;
    if (const int e = rows_product<T, kGradX>(dy, w, dim, nullptr, offsets, groups, grad_x, carry, status, s)) return e;
  }
  if (grad_weight) {
    using Tr = GroupedTraits<T, kGradW>;
    Operand in;
    if (const int e = laid_out(x, 0, rows, dim, sizeof(T), &room, &in, s)) return e;
    const WeightPlan p = weight_plan<T>(rows, dim, out_dim, groups);
    GroupedCall c = {};
    c.offsets = offsets, c.rows = rows, c.groups = groups;
    c.num_m = (int)out_dim, c.num_n = (int)dim;
    c.tile_n = p.tile_n, c.tiles_m = p.tiles_m, c.tiles_n = p.tiles_n, c.ranges = p.ranges;
    c.a = dy.data, c.b = in.data, c.pitch_a = dy.pitch, c.pitch_b = in.pitch;
    c.out = grad_weight, c.grad_bias = grad_bias, c.carry = (float*)carry, c.status = status;
    c.plan = (int64_t*)room;
    c.partial = (float*)(room + align_up((size_t)(2 + kPlanWords * p.ranges) * 8, 256));
    c.partial_bias = c.partial + (size_t)p.pieces * kTileM * p.tile_n;
    CUtensorMap a, b;
    if (const int e = make_map(&a, code_of<T>(), dy, Tr::kBox, Tr::kBlock)) return e;
    if (const int e = make_map(&b, code_of<T>(), in, Tr::kBox, Tr::kBlock)) return e;
    if (const int e = launch_grouped<T, kGradW>(c, a, b, p.ranges, s)) return e;
    if (p.ranges > 1) {
      const dim3 grid(kJoinParts, (unsigned)(p.ranges - 1));
      APT_FOLLOW((k_join_weights<T>), grid, 256, 0, s, c);
    }
  }
  return APT_OK;
}

static int linear_check(const char* who, int dtype, int64_t rows, int64_t dim, int64_t out_dim, int64_t groups, const void* workspace, size_t workspace_bytes,
                        int backward) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(rows >= 0 && rows < (1ll << 31) - (1 << 20) && dim > 0 && out_dim > 0 && dim <= APT_GROUPED_LINEAR_MAX_DIM && out_dim <= APT_GROUPED_LINEAR_MAX_DIM,
                "%s: %lld rows of %lld by %lld (1 to %d are possible)", who, (long long)rows, (long long)dim, (long long)out_dim, APT_GROUPED_LINEAR_MAX_DIM);
  APT_CHECK_ARG(groups > 0 && groups <= APT_GROUPED_LINEAR_MAX_GROUPS, "%s: %lld groups (1 to %d are possible)", who, (long long)groups,
                APT_GROUPED_LINEAR_MAX_GROUPS);
  APT_CHECK_ARG(rows == 0 || workspace_bytes >= apt_grouped_linear_workspace_bytes(dtype, rows, dim, out_dim, groups, backward), "%s: workspace too small", who);
  APT_CHECK_ARG((uintptr_t)workspace % 16 == 0, "%s: workspace not aligned to 16 bytes", who);
  return APT_OK;
}

}  // namespace apt

extern "C" size_t apt_grouped_linear_workspace_bytes(int dtype, int64_t rows, int64_t dim, int64_t out_dim, int64_t groups, int backward) {
  if (rows <= 0 || dim <= 0 || out_dim <= 0 || groups <= 0) return 0;
  return dtype == APT_F32 ? apt::linear_room<float>(rows, dim, out_dim, groups, backward) : apt::linear_room<__half>(rows, dim, out_dim, groups, backward);
}

extern "C" int apt_grouped_linear_forward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t out_dim,
                                          const int64_t* offsets, int64_t groups, void* out, void* workspace, size_t workspace_bytes,
                                          int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = linear_check("apt_grouped_linear_forward", dtype, rows, dim, out_dim, groups, workspace, workspace_bytes, 0)) return e;
  if (rows == 0) return look_at_ends(offsets, groups, 0, status_word, (cudaStream_t)stream);
  APT_CHECK_ARG(x && weight && offsets && out && status_word, "apt_grouped_linear_forward: null buffer");
  APT_CHECK_ARG(((uintptr_t)x | (uintptr_t)weight | (uintptr_t)out) % 16 == 0, "apt_grouped_linear_forward: buffers not aligned to 16 bytes");
  const cudaStream_t s = (cudaStream_t)stream;
  char* const room = (char*)workspace;
  if (dtype == APT_F32) return linear_forward<float>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, room, status_word, s);
  if (dtype == APT_BF16) return linear_forward<__nv_bfloat16>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, room, status_word, s);
  return linear_forward<__half>(x, rows, dim, weight, bias, out_dim, offsets, (int)groups, out, room, status_word, s);
}

extern "C" int apt_grouped_linear_backward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, int64_t out_dim,
                                           const int64_t* offsets, int64_t groups, const void* grad_out, void* grad_x, void* grad_weight,
                                           void* grad_bias, void* workspace, size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  if (const int e = linear_check("apt_grouped_linear_backward", dtype, rows, dim, out_dim, groups, workspace, workspace_bytes, 1)) return e;
  APT_CHECK_ARG(offsets && status_word && (rows == 0 || grad_out) && (!grad_x || rows == 0 || weight) && (!grad_weight || rows == 0 || x),
                "apt_grouped_linear_backward: null buffer");
  APT_CHECK_ARG(((uintptr_t)x | (uintptr_t)weight | (uintptr_t)grad_out | (uintptr_t)grad_x | (uintptr_t)grad_weight) % 16 == 0,
                "apt_grouped_linear_backward: buffers not aligned to 16 bytes");
  const cudaStream_t s = (cudaStream_t)stream;
  const int g = (int)groups;
  char* const room = (char*)workspace;
  if (dtype == APT_F32) return linear_backward<float>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, room, status_word, s);
  if (dtype == APT_BF16)
    return linear_backward<__nv_bfloat16>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, room, status_word, s);
  return linear_backward<__half>(x, rows, dim, weight, out_dim, offsets, g, grad_out, grad_x, grad_weight, grad_bias, room, status_word, s);
}
