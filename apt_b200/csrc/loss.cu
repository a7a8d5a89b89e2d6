// Softmax cross entropy behind the last layer's product, whose logits are never kept.
//
//   z = x W^T + b,   loss_r = log sum_v exp(z_rv) - z_r,label,   dz_rv = g_r (exp(z_rv) / sum_v exp(z_rv) - [v = label])
//   dx = dz W,   dW = dz^T x,   db_v = sum_r dz_rv
//
// Forward: products of rows and classes tile by tile on the tensor cores (k_grouped, kStats), of which a tile leaves each row's largest
// logit and sum of exponentials; k_loss_rows puts those of all tiles together. Backward: the products once more, from which the slopes dz of
// some classes follow at once (kSlopes), rounded to x's type, and from those the two products dW (kSumW) and dx (kSumX). The classes are taken
// in pieces, so that slopes of at most kMostSlopes bytes are there at a time; a piece finishes its rows of dW and adds to dx, which is held in
// fp32 until the last one.
//
// The slopes' factors g_r are kept out of them as far as they are common to all rows, and multiplied to the sums of dx and dW: in 16 bits the
// label's slope, p - 1, is then next to a power of two, and f16 has them times 2^14, so that probabilities down to 4e-9 are numbers and not
// steps of its smallest. Fewer than 2^-11 (f16; bf16 2^-8) of a slope are lost to its rounding. Where every row has a gradient of its own they are in the
// slopes, next to the largest. f16 has not the range for those of less than 2^-8 of it: then dx goes by slopes without them, and is multiplied by its row's,
// and dW and db by slopes that are made once more, where a row adds what is more than 2^-39 of the largest gradient.
#include "grouped.cuh"

namespace apt {

constexpr size_t kMostSlopes = 512ull << 20, kMostParts = 128ull << 20;
constexpr int kPieceUnit = 256;
constexpr float kWide = 0x1p-8f;
constexpr float kLn2 = 0.69314718055994531f;

struct RowsCall {
  const float2* parts;
  int num_parts;
  int64_t pitch;
  float2* stats;                // of the pieces so far, in the end of all classes; the sum -1: the row does not count
  const float* picked;
  const int64_t* labels;
  int64_t rows, classes, ignore;
  int first, last;
  float* losses;                // null: not wanted row by row
  float2* sums;                 // [blocks]: losses and rows that count
  int *turn, *dirty;            // blocks that have theirs there; 1: rows that do not count have logits that are no numbers
  int mean;
  float *loss, *count;          // of all rows; loss null: not wanted
  int32_t* status;
};

// 32 rows a block, eight warps that have every eighth part.
__global__ void __launch_bounds__(256) k_loss_rows(const __grid_constant__ RowsCall c) {
  wait_for_previous();
  __shared__ float2 shared[8][32];
  __shared__ double total[2][8];
  __shared__ int is_last;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t row = (int64_t)blockIdx.x * 32 + lane;
  const bool there = row < c.rows;
  float2 s = make_float2(-INFINITY, 0.0f);
  if (there) {
    if (warp == 0 && !c.first) s = c.stats[row];
    const float2* const from = c.parts + row;
    int p = warp;
    for (; p + 24 < c.num_parts; p += 32) {
      float2 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = from[(p + 8 * u) * c.pitch];
#pragma unroll
      for (int u = 0; u < 4; ++u) join_statistics(&s, v[u]);
    }
    for (; p < c.num_parts; p += 8) join_statistics(&s, from[p * c.pitch]);
  }
  shared[warp][lane] = s;
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) join_statistics(&s, shared[w][lane]);
    float loss = 0.0f, counts = 0.0f;
    if (there && c.last) {
      const int64_t label = c.labels[row];
      const bool known = label >= 0 && label < c.classes;
      if (label != c.ignore && !known) atomicOr(c.status, APT_FLAG_ID_OUT_OF_RANGE);
      if (label != c.ignore && known) {
        // against the same number that the sum's exponents refer to, so that a row that is all but sure of its label keeps its digits
        loss = (log2f(s.y) - fmaf(c.picked[row], kLog2e, -s.x)) * kLn2, counts = 1.0f;
      } else {
        if (!(fabsf(s.x) < INFINITY && s.y < INFINITY)) *c.dirty = 1;
        s.y = -1.0f;
      }
      if (c.losses) c.losses[row] = loss;
    }
    if (there) c.stats[row] = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o), counts += __shfl_xor_sync(0xffffffffu, counts, o);
    if (lane == 0 && c.last) {
      c.sums[blockIdx.x] = make_float2(loss, counts);
      __threadfence();
      is_last = atomicAdd(c.turn, 1) == (int)gridDim.x - 1;
    }
  }
  if (!c.last) return;
  __syncthreads();
  if (!is_last) return;
  // The last block adds up what all have left, in their order: the sum, or the mean over the rows that count (0 where none does), and their number.
  __threadfence();
  double a = 0.0, b = 0.0;
  const volatile float2* const sums = c.sums;
  for (int64_t i = threadIdx.x; i < gridDim.x; i += 256) a += sums[i].x, b += sums[i].y;
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o), b += __shfl_xor_sync(0xffffffffu, b, o);
  if (lane == 0) total[0][warp] = a, total[1][warp] = b;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 8; ++w) a += total[0][w], b += total[1][w];
  *c.count = (float)b;
  if (c.loss) *c.loss = (float)(c.mean ? a / fmax(b, 1.0) : a);
}

// Rows' own gradients go into their slopes, less the largest of those that are numbers (one that is none is its own row's matter). scale[0]: what they
// are multiplied by there, scale[1]: what the sums over slopes are. wide: some that are not zero are less than 2^-8 of the largest. One block.
__global__ void __launch_bounds__(1024) k_loss_scale(const float* __restrict__ grad, int64_t rows, const float2* __restrict__ stats, float range, float* scale, int* wide) {
  wait_for_previous();
  __shared__ float part[2][32];
  float m = 0.0f, least = INFINITY;
  // (nothing is asked between the loads of eight rows: a million rows take 155 us, and 630 with a question between the two loads of each)
  constexpr int kAtOnce = 8;
  for (int64_t i0 = threadIdx.x; i0 < rows; i0 += kAtOnce * 1024) {
    float g[kAtOnce], y[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int64_t i = min(i0 + u * 1024, rows - 1);
      g[u] = fabsf(grad[i]), y[u] = stats[i].y;
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float v = !(y[u] < 0.0f) && g[u] < INFINITY ? g[u] : 0.0f;
      m = fmaxf(m, v), least = fminf(least, v > 0.0f ? v : INFINITY);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o)), least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  if (threadIdx.x % 32 == 0) part[0][threadIdx.x / 32] = m, part[1][threadIdx.x / 32] = least;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 0; w < 32; ++w) m = fmaxf(m, part[0][w]), least = fminf(least, part[1][w]);
  *wide = least < kWide * m;
  m = m > 0.0f ? fmaxf(m, 1e-30f) : 1.0f;
  scale[0] = range / m, scale[1] = m / range;
}

// dx from its parts: 32 rows and 64 columns a block, 16 warps, or twice as many that have every other part. WHOLE: rows are whole slices of 8 elements.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(1024) k_loss_grad_rows(const __grid_constant__ GroupedCall c, T* out, int splits) {
  wait_for_previous();
  constexpr int kMostN = GroupedTraits<T, kSumX>::kMostN;
  __shared__ float tile[2][32][68];
  const int lane = threadIdx.x % 32, quad = threadIdx.x / 32 % 16, team = threadIdx.x / 512, teams = blockDim.x / 512;
  const int64_t row0 = (int64_t)blockIdx.x * 32;
  const int col0 = blockIdx.y * 64;
  const int tall = c.tile_m * c.halves;
  const int64_t row = row0 + lane;
  const int t = (int)(row / tall), in = (int)(row - (int64_t)t * tall), half = in / kTileM, quarter = in % kTileM / 32;
  const int64_t apart = (int64_t)c.tiles_m * c.tiles_n * c.halves * kTileM * kMostN;
  const int col = col0 + quad * 4, n = col / c.tile_n;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (row < c.rows && col < c.num_n) {
    const float* const from = c.carry + ((((int64_t)t * c.tiles_n + n) * c.halves + half) * 4 + quarter) * 32 * kMostN + (col - n * c.tile_n) * 32 + in % 32 * 4;
#pragma unroll 8
    for (int s = team; s < splits; s += teams) {
      const float4 p = *(const float4*)(from + s * apart);
      sum.x += p.x, sum.y += p.y, sum.z += p.z, sum.w += p.w;
    }
  }
  *(float4*)&tile[team][lane][quad * 4] = sum;
  __syncthreads();
  if constexpr (WHOLE) {
    if (threadIdx.x >= 256) return;
    const int r = threadIdx.x / 8, at = threadIdx.x % 8 * 8;
    if (row0 + r < c.rows && col0 + at < c.num_n) {
      const float scale = row_scale(c.loss, row0 + r);
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = (tile[0][r][at + q] + (teams > 1 ? tile[1][r][at + q] : 0.0f)) * scale;
      T* const to = out + (row0 + r) * c.num_n + col0 + at;
      if constexpr (sizeof(T) == 2) *(uint4*)to = rounded_slice<T>(v);
      else *(uint4*)to = rounded_slice<T>(v), *(uint4*)(to + 4) = rounded_slice<T>(v + 4);
    }
  } else {
    for (int i = threadIdx.x; i < 32 * 64; i += blockDim.x) {
      const int64_t r = row0 + i / 64;
      const int at = i % 64;
      if (r < c.rows && col0 + at < c.num_n) out[r * c.num_n + col0 + at] = Elem<T>::from_f((tile[0][i / 64][at] + (teams > 1 ? tile[1][i / 64][at] : 0.0f)) * row_scale(c.loss, r));
    }
  }
}

// The rows for dW, zeros for those that do not count, where some of these hold what is no number (0 times it would be none either). Nothing is done where
// none does. Rows of whole 16-byte slices.
__global__ void __launch_bounds__(256) k_loss_clean(const uint4* __restrict__ x, int64_t rows, int slices, const float2* __restrict__ stats, const int* __restrict__ unclean,
                                                    uint4* out) {
  wait_for_previous();
  if (!*unclean) return;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * slices; i += (int64_t)gridDim.x * 256)
    out[i] = stats[i / slices].y < 0.0f ? make_uint4(0u, 0u, 0u, 0u) : x[i];
}

// db without dW.
template <typename T>
__global__ void __launch_bounds__(1024) k_loss_grad_bias(const T* __restrict__ slopes, int64_t rows, int64_t pitch, int classes, const __grid_constant__ LossCall loss, T* out) {
  wait_for_previous();
  __shared__ float part[32][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, v = blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (v < classes)
    for (int64_t r = warp; r < rows; r += 32) sum += Elem<T>::to_f(slopes[r * pitch + v]);
  part[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && v < classes) {
    for (int k = 1; k < 32; ++k) sum += part[k][lane];
    out[v] = Elem<T>::from_f(sum * sum_scale(loss));
  }
}

// ---- host side -----------------------------------------------------------------------
// A workspace's parts, one behind the other; without a workspace their sizes.
struct Arena {
  char* base;
  size_t used = 0;
  template <typename V>
  V* take(size_t count) {
    char* const p = base + used;
    used += align_up(count * sizeof(V), 256);
    return base ? (V*)p : nullptr;
  }
};
static Operand in_arena(Arena* a, const void* data, int64_t stack, int64_t rows, int64_t columns, size_t size, bool* copied) {
  Operand o = {data, stack, rows, columns, pitch_of(columns, size)};
  *copied = o.pitch != columns;
  if (*copied) o.data = a->take<char>((size_t)rows * o.pitch * size);
  return o;
}

// Tiles, what is kept and how the work is cut, of rows against classes (n of them, k the rows' length) and of dx (n its columns, k classes).
template <typename T, int MODE>
static GroupedCall listed_call(int64_t rows, int64_t n, int64_t k) {
  using Tr = GroupedTraits<T, MODE>;
  GroupedCall c = {};
  c.rows = rows, c.groups = 1, c.num_n = (int)n, c.num_k = (int)k, c.halves = c.deep = c.splits = 1;
  c.tile_m = kTileM;
  while (c.tile_m > 16 && c.tile_m >= 2 * rows) c.tile_m /= 2;
  int64_t most = Tr::kMostN;
  if (Tr::kClasses) {
    // narrower tiles while there are blocks without one, or shorter ones (the products are of 128 rows always: copies and conversions get fewer)
    while (most > 64 && ceil_div(rows, c.tile_m) * ceil_div(n, most) < kNumSMs) most /= 2;
    while (c.tile_m > 16 && 2 * ceil_div(rows, c.tile_m) * ceil_div(n, most) <= kNumSMs) c.tile_m /= 2;
  }
  int64_t tiles_m = ceil_div(rows, c.tile_m);
  c.tile_n = tile_columns(n, (int)most), c.tiles_n = (int)ceil_div(n, c.tile_n);
  const int room = kMostShared - grouped_lists<T, MODE>(1) - Tr::kOutWarps * Tr::kStaging;
  const int copied = Tr::kSplit ? Tr::copied(kTileM, Tr::kMnA) : c.tile_m * 128, pieces = Tr::kSplit ? 3 * Tr::piece(kTileM, Tr::kMnA) : 0;
  const int copied_b = Tr::copied(c.tile_n, Tr::kMnB), pieces_b = Tr::kSplit ? 3 * Tr::piece(c.tile_n, Tr::kMnB) : 0;
  if (Tr::kClasses) {
    const int64_t bytes = ceil_div(k, Tr::kBlock) * (Tr::kSplit ? pieces_b : copied_b), least = (Tr::kSplit ? 2 * pieces : 0) + 3 * copied;
    c.keep = bytes + least <= room && tiles_m >= 3 && tiles_m * c.tiles_n >= 3 * kNumSMs;
  }
  if (!Tr::kSplit && !c.keep) {
    if (rows > kTileM && (MODE == kSumX || (k >= 512 && tiles_m * c.tiles_n >= 4 * kNumSMs))) c.halves = 2;
    else if (k > Tr::kBlock && 2 * (copied + copied_b) <= 48 * 1024) c.deep = 2;
  }
  tiles_m = ceil_div(rows, (int64_t)c.tile_m * c.halves);
  c.tiles_m = (int)tiles_m;
  // a band's rows: a quarter of L2
  c.band = c.keep ? c.tiles_m : (int)std::max<int64_t>(1, std::min<int64_t>(tiles_m, (32ll << 20) / ((int64_t)c.tile_m * c.halves * k * (int64_t)sizeof(T))));
  if (MODE == kSumX) {
    // Few tiles share the contraction among as many blocks as make it shortest: the longest one's stages, six stages' time for bringing a part
    // out, and a part's way to memory and back (a stage's time for 256 KB).
    const int64_t stages = ceil_div(k, Tr::kBlock * c.deep), tiles = tiles_m * c.tiles_n, bytes = (int64_t)c.halves * kTileM * c.tile_n * 4;
    int64_t best = 0, cost = 0;
    for (int64_t s = 1; s <= std::max<int64_t>(1, std::min(stages / 4, 4 * kNumSMs / tiles)); ++s) {
      const int64_t here = ceil_div(tiles * s, kNumSMs) * (ceil_div(stages, s) + 6) + 2 * tiles * s * bytes / (1 << 20);
      if (!best || here < cost) best = s, cost = here;
    }
    c.split_stages = (int)ceil_div(stages, best), c.splits = (int)ceil_div(stages, c.split_stages);
  }
  return c;
}
template <typename T, int MODE>
static int run_listed(const GroupedCall& c, const Operand& rows, const Operand& weight, cudaStream_t s) {
  using Tr = GroupedTraits<T, MODE>;
  CUtensorMap a, b;
  if (const int e = make_map(&a, code_of<T>(), rows, Tr::kBox, c.tile_m)) return e;
  if (const int e = make_map(&b, code_of<T>(), weight, Tr::kBox, Tr::kMnB ? Tr::kBlock : c.tile_n)) return e;
  return run_grouped<T, MODE>(c, a, b, (int64_t)c.tiles_m * c.tiles_n * c.splits, s);
}

// dW in whole sums where that leaves no more than two fifths of the blocks without one: 256 classes a tile, nothing to join. 32768 classes of 256
// and 8192 rows, bf16: 111 us; in runs that begin and end within sums 135, and their join 17.
template <typename T>
static bool tall_weights(int64_t dim, int64_t classes) {
  if (sizeof(T) == 4) return false;
  const int64_t tiles = ceil_div(classes, 2 * kTileM) * ceil_div(dim, GroupedTraits<T, kTallW>::kMostN);
  return 5 * tiles >= 3 * ceil_div(tiles, kNumSMs) * kNumSMs;
}

// Classes of a piece, of which a row takes so many bytes each: whole tiles, and pieces as long as one another.
static int64_t piece_of(int64_t classes, double bytes_a_class, size_t most) {
  const int64_t fit = std::max<int64_t>(1, (int64_t)(most / bytes_a_class) / kPieceUnit), units = ceil_div(classes, kPieceUnit);
  return ceil_div(units, ceil_div(units, fit)) * kPieceUnit;
}
// The rows [v0, v0 + n) of a matrix.
static Operand some_rows(const Operand& o, int64_t v0, int64_t n, size_t size) { return {(const char*)o.data + v0 * o.pitch * size, 1, n, o.columns, o.pitch}; }

struct LossProblem {
  const void* x;
  int64_t rows, dim;
  const void *weight, *bias;
  int64_t classes;
  const int64_t* labels;
  int64_t ignore;
  int reduction;
  int32_t* status;
};
// fp32: contractions that are brought out in parts take a tile a block.
template <typename T>
static float* carry_of(Arena* a, int64_t terms) {
  using Tr = GroupedTraits<T, kStats>;
  return Tr::kCuts && terms > (int64_t)Tr::kCut * Tr::kBlock ? a->take<float>((size_t)kNumSMs * kTileM * Tr::kMostN) : nullptr;
}

// Both passes take their workspace as they go; with `run` false that is all.
template <typename T>
static int loss_forward(const LossProblem& q, float* loss, float* saved, Arena* arena, bool run, cudaStream_t s) {
  using Tr = GroupedTraits<T, kStats>;
  bool copy_x, copy_w;
  const Operand x = in_arena(arena, q.x, 0, q.rows, q.dim, sizeof(T), &copy_x), w = in_arena(arena, q.weight, 1, q.classes, q.dim, sizeof(T), &copy_w);
  const int64_t pitch = align_up(q.rows, 32), blocks = ceil_div(q.rows, 32);
  // (tiles of 64 columns at the least; in narrower ones than the widest there are few)
  const int64_t piece = piece_of(q.classes, (double)pitch * 8 / Tr::kMostN, kMostParts);
  int64_t most_parts = 0;
  for (const int64_t n : {std::min(piece, q.classes), q.classes - (ceil_div(q.classes, piece) - 1) * piece})
    most_parts = std::max<int64_t>(most_parts, listed_call<T, kStats>(q.rows, n, q.dim).tiles_n);
  float2* const parts = arena->take<float2>(most_parts * pitch);
  float* const picked = arena->take<float>(q.rows);
  float2* const sums = arena->take<float2>(blocks);
  int* const turn = arena->take<int>(1);
  float* const carry = carry_of<T>(arena, q.dim);
  if (!run) return APT_OK;
  if (copy_x)
    if (const int e = widen_rows(q.x, q.rows, q.dim * sizeof(T), (void*)x.data, s)) return e;
  if (copy_w)
    if (const int e = widen_rows(q.weight, q.classes, q.dim * sizeof(T), (void*)w.data, s)) return e;
  for (int64_t v0 = 0; v0 < q.classes; v0 += piece) {
    const int64_t n = std::min(piece, q.classes - v0);
    GroupedCall c = listed_call<T, kStats>(q.rows, n, q.dim);
    c.bias = q.bias ? (const T*)q.bias + v0 : nullptr, c.carry = carry, c.status = q.status;
    c.loss.labels = q.labels, c.loss.class0 = v0, c.loss.pitch = pitch, c.loss.parts = parts, c.loss.picked = picked, c.loss.turn = turn, c.loss.dirty = (int*)saved + 2 * q.rows + 1;
    if (const int e = run_listed<T, kStats>(c, x, some_rows(w, v0, n, sizeof(T)), s)) return e;
    RowsCall r = {};
    r.parts = parts, r.num_parts = c.tiles_n, r.pitch = pitch, r.stats = (float2*)saved, r.picked = picked, r.labels = q.labels;
    r.rows = q.rows, r.classes = q.classes, r.ignore = q.ignore, r.first = v0 == 0, r.last = v0 + n == q.classes;
    r.losses = q.reduction == APT_LOSS_NONE ? loss : nullptr, r.sums = sums, r.turn = turn, r.dirty = (int*)saved + 2 * q.rows + 1, r.status = q.status;
    r.mean = q.reduction == APT_LOSS_MEAN, r.loss = q.reduction == APT_LOSS_NONE ? nullptr : loss, r.count = saved + 2 * q.rows;
    APT_FOLLOW(k_loss_rows, blocks, 256, 0, s, r);
  }
  return APT_OK;
}

template <typename T>
static int loss_backward(const LossProblem& q, const float* saved, const float* grad, void* grad_x, void* grad_weight, void* grad_bias, Arena* arena, bool run,
                         cudaStream_t s) {
  bool copy_x, copy_w;
  const Operand x = in_arena(arena, q.x, 0, q.rows, q.dim, sizeof(T), &copy_x), w = in_arena(arena, q.weight, 1, q.classes, q.dim, sizeof(T), &copy_w);
  const int64_t piece = piece_of(q.classes, (double)q.rows * sizeof(T), kMostSlopes), most = std::min(piece, q.classes);
  const int64_t pitch = align_up(most, 64);
  T* const slopes = arena->take<T>(q.rows * pitch);
  float* const scale = arena->take<float>(2);
  int* const wide = arena->take<int>(1);
  float* const carry = carry_of<T>(arena, q.dim);
  void* const clean = arena->take<char>((size_t)q.rows * x.pitch * sizeof(T));
  GroupedCall sum_x = listed_call<T, kSumX>(q.rows, q.dim, most);
  const int splits = sum_x.splits;
  // dx in whole sums: all classes at once, in one part of the contraction
  const bool whole_x = splits == 1 && most == q.classes && most <= (int64_t)GroupedTraits<T, kSumX>::kCut * GroupedTraits<T, kSumX>::kBlock;
  if (!whole_x) sum_x.carry = arena->take<float>((size_t)splits * sum_x.tiles_m * sum_x.tiles_n * sum_x.halves * kTileM * GroupedTraits<T, kSumX>::kMostN);
  const WeightPlan p = weight_plan<T>(q.rows, q.dim, most, 1);
  int64_t* const plan = arena->take<int64_t>(2 + kPlanWords * p.ranges);
  float* const partial = arena->take<float>((size_t)p.pieces * kTileM * p.tile_n);
  float* const partial_bias = arena->take<float>((size_t)p.pieces * kTileM);
  float* const weight_carry = (float*)arena->take<char>((tall_weights<T>(q.dim, most) ? 2 : 1) * carry_room<T>(q.rows, q.dim, most, true));
  if (!run) return APT_OK;
  if (copy_x)
    if (const int e = widen_rows(q.x, q.rows, q.dim * sizeof(T), (void*)x.data, s)) return e;
  if (copy_w)
    if (const int e = widen_rows(q.weight, q.classes, q.dim * sizeof(T), (void*)w.data, s)) return e;
  const bool each = q.reduction == APT_LOSS_NONE;
  const float range = std::is_same<T, __half>::value ? 16384.0f : 1.0f;
  // a single row's own gradient is the common one
  LossCall call = {};
  if (grad_weight) {
    call.unclean = (const int*)saved + 2 * q.rows + 1;
    const int slices = (int)(x.pitch * sizeof(T) / 16);
    APT_FOLLOW(k_loss_clean, wave_grid(ceil_div(q.rows * slices, 256), 8, 1), 256, 0, s, (const uint4*)x.data, q.rows, slices, (const float2*)saved, call.unclean,
               (uint4*)clean);
    Operand o = x;
    o.data = clean;
    if (const int e = make_map(&call.clean, code_of<T>(), o, GroupedTraits<T, kSumW>::kBox, GroupedTraits<T, kSumW>::kBlock)) return e;
  }
  call.labels = q.labels, call.pitch = pitch, call.stats = (const float2*)saved, call.range = range;
  if (each && q.rows > 1) {
    call.grad = grad, call.scale = scale;
    APT_FOLLOW(k_loss_scale, 1, 1024, 0, s, grad, q.rows, (const float2*)saved, range, scale, wide);
  } else {
    call.common = grad, call.count = q.reduction == APT_LOSS_MEAN ? saved + 2 * q.rows : nullptr;
  }
  // dx by its rows' own gradients (where they are wide), and slopes for dW and db by themselves then
  LossCall call_x = call;
  if (std::is_same<T, __half>::value && call.scale && grad_x) call_x.wide = wide, call_x.own = 1;
  for (int64_t v0 = 0; v0 < q.classes; v0 += piece) {
    const int64_t n = std::min(piece, q.classes - v0);
    const Operand some = some_rows(w, v0, n, sizeof(T));
    GroupedCall c = listed_call<T, kSlopes>(q.rows, n, q.dim);
    c.bias = q.bias ? (const T*)q.bias + v0 : nullptr, c.carry = carry, c.out = slopes, c.status = q.status;
    c.loss = call_x, c.loss.class0 = v0;
    if (const int e = run_listed<T, kSlopes>(c, x, some, s)) return e;
    const Operand dz = {slopes, 0, q.rows, n, pitch};
    if (grad_x) {
      GroupedCall d = sum_x;
      d.num_k = (int)n, d.splits = (int)ceil_div(ceil_div(n, GroupedTraits<T, kSumX>::kBlock * d.deep), d.split_stages);
      d.status = q.status, d.loss = call_x, d.loss.more = v0 > 0, d.out = whole_x ? grad_x : nullptr;
      if (const int e = run_listed<T, kSumX>(d, dz, some, s)) return e;
    }
    if (call_x.own && (grad_weight || grad_bias)) {
      c.loss = call, c.loss.class0 = v0, c.loss.wide = wide, c.loss.again = 1;
      if (const int e = run_listed<T, kSlopes>(c, x, some, s)) return e;
    }
    if (grad_weight && tall_weights<T>(q.dim, most)) {
      if constexpr (sizeof(T) == 2) {
        using Tr = GroupedTraits<T, kTallW>;
        GroupedCall d = {};
        d.rows = q.rows, d.groups = 1, d.num_m = (int)n, d.num_n = (int)q.dim, d.halves = 2, d.deep = 1;
        d.tile_n = tile_columns(q.dim, Tr::kMostN), d.tiles_m = (int)ceil_div(n, 2 * kTileM), d.tiles_n = (int)ceil_div(q.dim, d.tile_n);
        d.out = (T*)grad_weight + v0 * q.dim, d.grad_bias = grad_bias ? (T*)grad_bias + v0 : nullptr, d.carry = weight_carry, d.status = q.status;
        d.loss = call;
        CUtensorMap a, b;
        if (const int e = make_map(&a, code_of<T>(), dz, Tr::kBox, Tr::kBlock)) return e;
        if (const int e = make_map(&b, code_of<T>(), x, Tr::kBox, Tr::kBlock)) return e;
        if (const int e = run_grouped<T, kTallW>(d, a, b, (int64_t)d.tiles_m * d.tiles_n, s)) return e;
      }
    } else if (grad_weight) {
      const WeightPlan p = weight_plan<T>(q.rows, q.dim, n, 1);
      GroupedCall d = {};
      d.rows = q.rows, d.groups = 1, d.num_m = (int)n, d.num_n = (int)q.dim;
      d.tile_n = p.tile_n, d.tiles_m = p.tiles_m, d.tiles_n = p.tiles_n, d.ranges = p.ranges;
      d.out = (T*)grad_weight + v0 * q.dim, d.grad_bias = grad_bias ? (T*)grad_bias + v0 : nullptr, d.carry = weight_carry, d.status = q.status;
      d.plan = plan, d.partial = partial, d.partial_bias = partial_bias, d.loss = call;
      using Tr = GroupedTraits<T, kSumW>;
      CUtensorMap a, b;
      if (const int e = make_map(&a, code_of<T>(), dz, Tr::kBox, Tr::kBlock)) return e;
      if (const int e = make_map(&b, code_of<T>(), x, Tr::kBox, Tr::kBlock)) return e;
      if (const int e = launch_grouped<T, kSumW>(d, a, b, p.ranges, s)) return e;
      if (p.ranges > 1) {
        const dim3 grid(kJoinParts, (unsigned)(p.ranges - 1));
        APT_FOLLOW((k_join_weights<T>), grid, 256, 0, s, d);
      }
    } else if (grad_bias) {
      APT_FOLLOW((k_loss_grad_bias<T>), ceil_div(n, 32), 1024, 0, s, (const T*)slopes, q.rows, pitch, (int)n, call, (T*)grad_bias + v0);
    }
  }
  if (grad_x && !whole_x) {
    sum_x.loss = call_x;
    const dim3 grid((unsigned)ceil_div(q.rows, 32), (unsigned)ceil_div(q.dim, 64));
    if (q.dim % 8 == 0) APT_FOLLOW((k_loss_grad_rows<T, true>), grid, splits >= 16 ? 1024 : 512, 0, s, sum_x, (T*)grad_x, splits);
    else APT_FOLLOW((k_loss_grad_rows<T, false>), grid, splits >= 16 ? 1024 : 512, 0, s, sum_x, (T*)grad_x, splits);
  }
  return APT_OK;
}

static int loss_check(const char* who, int dtype, int64_t rows, int64_t dim, int64_t classes, int reduction) {
  APT_CHECK_ARG(dtype == APT_F32 || dtype == APT_BF16 || dtype == APT_F16, "%s: unsupported dtype %d", who, dtype);
  APT_CHECK_ARG(rows >= 0 && rows < (1ll << 31) - (1 << 20) && classes >= 1 && classes < (1ll << 31) - (1 << 20), "%s: %lld rows, %lld classes", who, (long long)rows,
                (long long)classes);
  APT_CHECK_ARG(dim >= 1 && dim <= APT_GROUPED_LINEAR_MAX_DIM, "%s: rows of %lld (1 to %d are possible)", who, (long long)dim, APT_GROUPED_LINEAR_MAX_DIM);
  APT_CHECK_ARG(reduction == APT_LOSS_NONE || reduction == APT_LOSS_SUM || reduction == APT_LOSS_MEAN, "%s: unknown reduction %d", who, reduction);
  return APT_OK;
}
template <typename T>
static size_t loss_room(const LossProblem& q, int backward) {
  Arena a = {nullptr};
  if (backward) loss_backward<T>(q, nullptr, nullptr, nullptr, nullptr, nullptr, &a, false, nullptr);
  else loss_forward<T>(q, nullptr, nullptr, &a, false, nullptr);
  return a.used;
}

}  // namespace apt

extern "C" size_t apt_linear_cross_entropy_workspace_bytes(int dtype, int64_t rows, int64_t dim, int64_t classes, int backward) {
  using namespace apt;
  if (rows <= 0 || dim <= 0 || classes <= 0) return 0;
  LossProblem q = {};
  q.rows = rows, q.dim = dim, q.classes = classes;
  return dtype == APT_F32 ? loss_room<float>(q, backward) : loss_room<__half>(q, backward);
}

extern "C" int apt_linear_cross_entropy_forward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t classes,
                                                const int64_t* labels, int64_t ignore, int reduction, float* loss, float* saved, void* workspace,
                                                size_t workspace_bytes, int32_t* status_word, void* stream) {
  using namespace apt;
  const char* const who = "apt_linear_cross_entropy_forward";
  if (const int e = loss_check(who, dtype, rows, dim, classes, reduction)) return e;
  APT_CHECK_ARG((loss || (rows == 0 && reduction == APT_LOSS_NONE)) && saved, "%s: null buffer", who);
  const cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    APT_CUDA(cudaMemsetAsync(saved, 0, 8, s));
    if (reduction != APT_LOSS_NONE) APT_CUDA(cudaMemsetAsync(loss, 0, 4, s));
    return APT_OK;
  }
  APT_CHECK_ARG(x && weight && labels && status_word && workspace, "%s: null buffer", who);
  APT_CHECK_ARG(((uintptr_t)x | (uintptr_t)weight) % 16 == 0 && (uintptr_t)saved % 8 == 0, "%s: buffers not aligned to 16 bytes", who);
  APT_CHECK_ARG(workspace_bytes >= apt_linear_cross_entropy_workspace_bytes(dtype, rows, dim, classes, 0) && (uintptr_t)workspace % 256 == 0, "%s: workspace too small", who);
  const LossProblem q = {x, rows, dim, weight, bias, classes, labels, ignore, reduction, status_word};
  Arena a = {(char*)workspace};
  if (dtype == APT_F32) return loss_forward<float>(q, loss, saved, &a, true, s);
  if (dtype == APT_BF16) return loss_forward<__nv_bfloat16>(q, loss, saved, &a, true, s);
  return loss_forward<__half>(q, loss, saved, &a, true, s);
}

extern "C" int apt_linear_cross_entropy_backward(int dtype, const void* x, int64_t rows, int64_t dim, const void* weight, const void* bias, int64_t classes,
                                                 const int64_t* labels, int reduction, const float* saved, const float* grad_loss, void* grad_x,
                                                 void* grad_weight, void* grad_bias, void* workspace, size_t workspace_bytes, int32_t* status_word,
                                                 void* stream) {
  using namespace apt;
  const char* const who = "apt_linear_cross_entropy_backward";
  if (const int e = loss_check(who, dtype, rows, dim, classes, reduction)) return e;
  const cudaStream_t s = (cudaStream_t)stream;
  if (!grad_x && !grad_weight && !grad_bias) return APT_OK;
  const size_t size = dtype == APT_F32 ? 4 : 2;
  if (rows == 0) {
    if (grad_weight) APT_CUDA(cudaMemsetAsync(grad_weight, 0, (size_t)classes * dim * size, s));
    if (grad_bias) APT_CUDA(cudaMemsetAsync(grad_bias, 0, (size_t)classes * size, s));
    return APT_OK;
  }
  APT_CHECK_ARG(x && weight && labels && saved && grad_loss && status_word && workspace, "%s: null buffer", who);
  APT_CHECK_ARG(((uintptr_t)x | (uintptr_t)weight | (uintptr_t)grad_x | (uintptr_t)grad_weight) % 16 == 0 && (uintptr_t)saved % 8 == 0, "%s: buffers not aligned to 16 bytes",
                who);
  APT_CHECK_ARG(workspace_bytes >= apt_linear_cross_entropy_workspace_bytes(dtype, rows, dim, classes, 1) && (uintptr_t)workspace % 256 == 0, "%s: workspace too small", who);
  const LossProblem q = {x, rows, dim, weight, bias, classes, labels, 0, reduction, status_word};
  Arena a = {(char*)workspace};
  if (dtype == APT_F32) return loss_backward<float>(q, saved, grad_loss, grad_x, grad_weight, grad_bias, &a, true, s);
  if (dtype == APT_BF16) return loss_backward<__nv_bfloat16>(q, saved, grad_loss, grad_x, grad_weight, grad_bias, &a, true, s);
  return loss_backward<__half>(q, saved, grad_loss, grad_x, grad_weight, grad_bias, &a, true, s);
}
