// qe_op_page_weigh: the softmax weight that each cached position gets from new tokens, added up per
// sequence and KV head. No reference counterpart.
//
//   mass[s][h][j] += sum over rows t, q heads g of KV head h of w_tg(j),
//   w_tg(j) = exp(x_tg(j) - m_tg) / sum_i exp(x_tg(i) - m_tg),  x_tg(j) = q[t][g] . k_j / sqrt(128)
//
// A weight needs its row's sum over all positions. Up to 16 rows (tokens x q heads) of a sequence and KV head:
// k_weigh_few leaves the scores, 4 bytes a row and position where K has 128 or 256 for all rows, and k_weigh_kept makes
// weights of them. More rows: the scores are computed twice. k_weigh<kStats> leaves each row's maximum and sum over
// each block of positions, k_weigh_rows joins them, and k_weigh<kSums> adds up the weights; where tables hold no more than
// a block, k_weigh<kBoth> does all of it.
//
// Those two passes hold K still: a workgroup has 256 positions of a sequence and KV head, 64 a wave, as operand
// A of v_mfma_f32_32x32x16_bf16 in registers, and passes the rows by, 32 at a time through LDS. So K is read
// once a pass and a position's sum belongs to one wave: nothing is added in an order that changes. Where the
// positions make few workgroups the rows are split among several, whose sums k_weigh_add adds in order.
// f32 rows as three bf16 parts that add up exactly.
//
// Measured: the last 32 rows of each of 4 sequences of up to 16,000 positions, 16 over 8 heads, bf16 (82 MB of K), 48
// us: two passes of 21 and 24, bound by K (4 and 3.4 TB/s), and 5 the join. Up to 1024 f32 rows of 3 sequences over up to
// 4096 positions, 223: two passes of 114, 900 of the 1239 TFLOP/s that a large library product reaches, with
// exponentials, sums and the parts of f32 rows on the vector unit as long as the products. Up to 88 f32 rows of each of 19
// sequences over up to 112 positions, 24 over 8 heads, by k_weigh<kBoth> 24 us, by the passes 41.
#include "pages.h"

#include "device_common.h"
#include "status.h"

#include <cmath>

namespace qe {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kSpan = 256;   // positions of a workgroup
constexpr uint32_t kTile = 32;    // rows that pass by together
constexpr uint32_t kFewRows = 16;

struct WeighArgs {
  PagePlan p;
  PageStore st;
  const uint8_t* q;
  uint64_t q_stride;
  float* mass;
  uint64_t mass_stride;
  float2* parts;  // [n_rows][heads][blocks]: maximum, sum over a block; few rows: [n_seqs][n_kv][few][blocks]
  float2* rows;   // [n_rows][heads]: maximum, 1 / sum
  float* sums;    // [splits][n_seqs][n_kv][blocks][kSpan], where splits > 1
  float* scores;  // few rows: [n_seqs][n_kv][few][blocks * span], -inf where a row does not attend
  uint32_t n_rows, group, blocks, splits;
  uint32_t few, span;  // rows of a sequence and KV head that scores are kept of (0: none); positions of a workgroup
  float c;  // log2(e) / sqrt(128)
};

// The rows of a sequence: (token, q head) pairs of a KV head, token first.
struct Span {
  int64_t first;        // position of its first token
  uint32_t row0, rows;  // first packed row; tokens * group
  uint32_t end;         // positions that any of them attends: 0 .. end - 1
};
__device__ __forceinline__ Span span_of(const WeighArgs& a, uint32_t s) {
  const int64_t b = a.p.starts[s], e = a.p.starts[s + 1], lo = b < 0 ? 0 : b, hi = e < a.n_rows ? e : a.n_rows;
  Span q;
  q.first = int64_t(a.p.lens[s]) - (e - lo);
  q.row0 = uint32_t(lo);
  const int64_t n = hi > lo ? hi - lo : 0;
  q.rows = uint32_t(n) * a.group;
  q.end = uint32_t(max(min(q.first + n, capacity_of(a.p)), int64_t(0)));
  if (n == 0) q.end = 0;
  return q;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rebase(float from, float to) { return from == to ? 1.f : exp2_fast(from - to); }
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sums of 32 values over the 32 lanes of each half of the wave, value i to lane i: each step adds two values'
// halves up, one for the lanes whose bit is clear and one for the others.
template <int CTRL, int N>
__device__ __forceinline__ void halve(float (&v)[32], bool upper) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float keep = upper ? v[i + N] : v[i], send = upper ? v[i] : v[i + N];
    v[i] = keep + dpp<CTRL>(send);
  }
}
__device__ __forceinline__ float sums_of_halves(float (&v)[32]) {
  const uint32_t lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 16]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  halve<0x128, 8>(v, lane & 8);  // with lane ^ 8 of its row
  halve<0x141, 4>(v, lane & 4);  // 7 - lane of its 8
  halve<0x4E, 2>(v, lane & 2);   // lane ^ 2
  halve<0xB1, 1>(v, lane & 1);   // lane ^ 1
  return v[0];
}

// 8 e4m3 values (two words) as bf16 times a power of two
__device__ __forceinline__ bf16x8 fp8_bf16(uint32_t a, uint32_t b, float scale) {
  u32x4 u;
  u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false));
  u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true));
  u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false));
  u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true));
  return __builtin_bit_cast(bf16x8, u);
}

// 8 floats as three bf16 parts that add up to them: 8 + 8 + 8 of f32's 24 bits, so nothing is lost
__device__ __forceinline__ void cut_f32(const u32x4 (&x)[2], u32x4 (&part)[3]) {
#pragma unroll
  for (int k = 0; k < 4; k++) {
    uint32_t w[2][3];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const float v = __uint_as_float(x[k / 2][2 * (k & 1) + e]);
      w[e][0] = __float_as_uint(v);
      const float rest = v - __uint_as_float(w[e][0] & 0xFFFF0000u);
      w[e][1] = __float_as_uint(rest);
      w[e][2] = __float_as_uint(rest - __uint_as_float(w[e][1] & 0xFFFF0000u));
    }
#pragma unroll
    for (int n = 0; n < 3; n++) part[n][k] = __builtin_amdgcn_perm(w[1][n], w[0][n], 0x07060302u);  // upper halves
  }
}

// What passes by: a tile of rows of q in LDS, each of NS bf16 parts; the 16-byte piece c of row r at place
// c ^ (r & 15), so that the 32 rows that are read at once lie in different banks.
template <bool BF16_ROWS>
struct RowTile {
  static constexpr int NS = BF16_ROWS ? 1 : 3, LOADS = BF16_ROWS ? 2 : 4;
  u32x4 raw[LOADS];
  // thread: 16 dims of row tid / 8 (rows behind the last are read as that one)
  __device__ __forceinline__ void load(const WeighArgs& a, const Span& q, uint32_t head, uint32_t r0) {
    const uint32_t r = min(r0 + threadIdx.x / 8, q.rows - 1), t = r / a.group;
    const uint64_t e = (uint64_t(q.row0) + t) * a.q_stride + (head * a.group + (r - t * a.group)) * kPageDim + (threadIdx.x & 7) * 16;
    const u32x4* p = reinterpret_cast<const u32x4*>(a.q + e * (BF16_ROWS ? 2 : 4));
#pragma unroll
    for (int i = 0; i < LOADS; i++) raw[i] = p[i];
  }
  __device__ __forceinline__ void store(uint8_t (*buf)[kTile * 256]) const {
    const uint32_t r = threadIdx.x / 8;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t at = r * 256 + (((threadIdx.x & 7) * 2 + i) ^ (r & 15)) * 16;
      if constexpr (BF16_ROWS) {
        *reinterpret_cast<u32x4*>(buf[0] + at) = raw[i];
      } else {
        u32x4 part[3];
        const u32x4 two[2] = {raw[2 * i], raw[2 * i + 1]};
        cut_f32(two, part);
#pragma unroll
        for (int n = 0; n < 3; n++) *reinterpret_cast<u32x4*>(buf[n] + at) = part[n];
      }
    }
  }
};

// What a pass does: the rows' maxima and sums over the block (kStats), the weights by them (kSums), or both, where one
// block holds all positions (kBoth: the scores are still there when the four waves know a row's sum).
enum Pass { kStats, kSums, kBoth };

template <bool FP8, bool BF16_ROWS, Pass PASS>
__global__ __launch_bounds__(256, 2) void k_weigh(WeighArgs a) {
  constexpr int NS = BF16_ROWS ? 1 : 3, EL = FP8 ? 1 : 2;
  constexpr bool STATS = PASS != kSums, SUMS = PASS != kStats;
  __shared__ __align__(16) uint8_t buf[2][NS][kTile * 256];
  __shared__ float2 stat[STATS ? 2 : 1][STATS ? 4 : 1][STATS ? kTile : 1];
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t at = blockIdx.x;
  const uint32_t head = at % a.p.n_kv;
  at /= a.p.n_kv;
  const uint32_t split = at % a.splits;
  at /= a.splits;
  const uint32_t block = at % a.blocks, s = at / a.blocks;
  const Span q = span_of(a, s);
  if (block * kSpan >= q.end) return;
  // the tiles of rows that attend any of the positions, and of them this workgroup's
  const uint32_t tiles = (q.rows + kTile - 1) / kTile;
  const int64_t token0 = int64_t(block * kSpan) - q.first;
  const uint32_t tile0 = token0 > 0 ? uint32_t(token0) * a.group / kTile : 0;
  const uint32_t from = tile0 + uint32_t(uint64_t(tiles - tile0) * split / a.splits);
  const uint32_t to = tile0 + uint32_t(uint64_t(tiles - tile0) * (split + 1) / a.splits);
  const uint32_t x = block * kSpan + 64 * wave;  // this wave's positions
  RowTile<BF16_ROWS> rows;
  if (from < to) rows.load(a, q, head, from * kTile);

  // K, 32 positions at a time: operand A's lane has row `col` and, of dims in 8 steps, 8 a step
  const int32_t* const table = a.p.table + size_t(s) * a.p.table_stride;
  const uint32_t mask = (1u << a.p.page_shift) - 1;
  int32_t page[4];
  uint32_t there = 0;  // which of the four runs of 16 positions have a page
#pragma unroll
  for (int i = 0; i < 4; i++) {
    page[i] = table[min((x + 16 * i) >> a.p.page_shift, a.p.table_stride - 1)];
    if (uint32_t(page[i]) < a.p.n_pages) there |= 1u << i;
    else page[i] = 0;  // read as page 0, and what comes of it is masked
  }
  bf16x8 k[2][8];
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int32_t one = page[2 * u], two = page[2 * u + 1];
    const size_t row = page_row(a.p, col < 16 ? one : two, head, (x + 32 * u + col) & mask);
    if constexpr (FP8) {
      u32x4 raw[4];
#pragma unroll
      for (int i = 0; i < 4; i++) raw[i] = *reinterpret_cast<const u32x4*>(a.st.k + row * kPageDim + 32 * i + 16 * half);
      const float scale = exp_scale(a.st.k_exp[row]);
#pragma unroll
      for (int j = 0; j < 8; j++) k[u][j] = fp8_bf16(raw[j / 2][2 * (j & 1)], raw[j / 2][2 * (j & 1) + 1], scale);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        k[u][j] = *reinterpret_cast<const bf16x8*>(a.st.k + (row * kPageDim + 16 * j + 8 * half) * EL);
    }
  }

  f32x16 sum[2];
  sum[0] = 0.f;
  sum[1] = 0.f;
  if (from < to) {
    rows.store(buf[from & 1]);
    if (from + 1 < to) rows.load(a, q, head, (from + 1) * kTile);
  }
  __syncthreads();
  for (uint32_t i = from; i < to; i++) {
    const uint32_t r = i * kTile + col, token = r / a.group;  // this lane's row
    const bool real = r < q.rows;
    const int32_t last = real ? int32_t(max(min(q.first + token, capacity_of(a.p) - 1), int64_t(-1))) : -1;  // the last position it attends
    const uint64_t stat_at = (uint64_t(q.row0) + token) * a.group * a.p.n_kv + head * a.group + (r - token * a.group);
    float2 rs = make_float2(0.f, 0.f);
    if constexpr (PASS == kSums)
      if (real) rs = a.rows[stat_at];
    f32x16 v[2];
    v[0] = 0.f;
    v[1] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      // dims of step j: bf16 16 j + 8 half .., e4m3 32 (j / 2) + 16 half + 8 (j & 1) ..
      const uint32_t piece = FP8 ? 4 * (j / 2) + 2 * half + (j & 1) : 2 * j + half;
#pragma unroll
      for (int n = NS - 1; n >= 0; n--) {
        const bf16x8 f = *reinterpret_cast<const bf16x8*>(buf[i & 1][n] + col * 256 + ((piece ^ (col & 15)) * 16));
#pragma unroll
        for (int u = 0; u < 2; u++) v[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[u][j], f, v[u], 0, 0, 0);
      }
    }
    // element e of tile u: position x + 32 u + 8 (e / 4) + 4 half + e % 4
    const int64_t free_to = q.first + i * kTile / a.group;  // the least position that any of the tile's rows attends
    const bool masked = int64_t(x) + 63 > min(free_to, capacity_of(a.p) - 1) || (i + 1) * kTile > q.rows || there != 15;
    auto hidden = [&](int u, int e) __attribute__((always_inline)) {
      const uint32_t in = 32 * u + 8 * (e / 4) + (e & 3);
      return int32_t(x + in + 4 * half) > last || !(there >> (2 * u + e / 8) & 1);
    };
    if constexpr (STATS) {
      if (masked) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (hidden(u, e)) v[u][e] = -INFINITY;
      }
      float m = v[0][0], l = 0.f;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 16; e++) m = fmaxf(m, v[u][e]);
      m = max_halves(m) * a.c;
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 16; e++) l += exp2_fast(fmaf(v[u][e], a.c, -ref));
      l = add_halves(l);
      if (half == 0) stat[i & 1][wave][col] = make_float2(m, l);
    }
    // a row's maximum and sum over the block, of the four waves'
    auto of_block = [&] __attribute__((always_inline)) {
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; w++) m = fmaxf(m, stat[i & 1][w][col].x);
#pragma unroll
      for (int w = 0; w < 4; w++) l = fmaf(stat[i & 1][w][col].y, rebase(stat[i & 1][w][col].x, m), l);
      return make_float2(m, l);
    };
    if constexpr (PASS == kBoth) {
      __syncthreads();
      rs = of_block();
      rs.y = rs.y == 0.f ? 0.f : 1.f / rs.y;
    }
    if constexpr (SUMS) {
      const float ref = rs.x == -INFINITY ? 0.f : rs.x;
      if (masked) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 16; e++) {
            const float w = exp2_fast(fmaf(v[u][e], a.c, -ref)) * rs.y;
            sum[u][e] += hidden(u, e) ? 0.f : w;
          }
      } else {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 16; e++) sum[u][e] = fmaf(exp2_fast(fmaf(v[u][e], a.c, -ref)), rs.y, sum[u][e]);
      }
    }
    if (i + 1 < to) {
      rows.store(buf[(i + 1) & 1]);
      if (i + 2 < to) rows.load(a, q, head, (i + 2) * kTile);
    }
    __syncthreads();
    if constexpr (PASS == kStats)
      if (tid < kTile && real) a.parts[stat_at * a.blocks + block] = of_block();  // (wave 0, whose lane has this row)
  }
  if constexpr (SUMS) {
    float all[32];
#pragma unroll
    for (int i = 0; i < 32; i++) all[i] = sum[i / 16][i % 16];
    const float v = sums_of_halves(all);  // of element lane % 16 of tile lane / 16 % 2
    const uint32_t in = 64 * wave + 32 * (lane >> 4 & 1) + 8 * (lane >> 2 & 3) + 4 * half + (lane & 3), j = block * kSpan + in;
    const uint64_t item = uint64_t(s) * a.p.n_kv + head;
    if (a.splits > 1) a.sums[((uint64_t(split) * a.p.n_seqs * a.p.n_kv + item) * a.blocks + block) * kSpan + in] = v;
    else if (j < q.end && !(v == 0.f)) a.mass[item * a.mass_stride + j] += v;
  }
}

// ---- few rows: up to 16 of a sequence and KV head ----
// K goes by once, in steps of 64 positions a wave, against the rows in registers (operand B of
// v_mfma_f32_16x16x32_bf16), and the scores are kept, which is less than a second read of K. A
// step's loads are issued a step ahead. Bound by the bytes of K and of the scores: a row of each of 40 sequences of up
// to 4097 positions, 32 over 8 heads, e4m3 (99 MB of K, 13 MB of scores), 31 us, 25 without the stores; with the
// weights (8 us) 38. The same by the passes for more rows, which read K twice, 77.
template <bool FP8>
struct KStep {
  u32x4 k[FP8 ? 8 : 16];
  u32x4 exp;      // e4m3: of the run that the lane's rows of K lie in
  uint32_t there;  // which of the four runs of 16 positions have a page
};

template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256, 2) void k_weigh_few(WeighArgs a) {
  constexpr int NS = BF16_ROWS ? 1 : 3, EL = FP8 ? 1 : 2;
  __shared__ float2 stat[4][kFewRows];
  __shared__ __align__(16) float out[4][kFewRows][68];  // each wave's own
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t head = blockIdx.x % a.p.n_kv, block = blockIdx.x / a.p.n_kv % a.blocks, s = blockIdx.x / a.p.n_kv / a.blocks;
  const Span q = span_of(a, s);
  const uint32_t x0 = block * a.span, x1 = min(x0 + a.span, q.end);
  if (x0 >= q.end || q.rows > a.few) return;  // (more rows than there was room for: k_weigh_kept sees to them)
  const int32_t* const table = a.p.table + size_t(s) * a.p.table_stride;
  const uint32_t mask = (1u << a.p.page_shift) - 1;
  // K of positions x .. x + 63: operand A's row `col` of tile t is position 16 (col / 4) + 4 t + col % 4, so that a
  // lane's results of the four tiles are those of the 16 positions from 16 g; and of dims a lane has 8 in each of
  // 4 steps: bf16 32 j + 8 g .., e4m3 64 (j / 2) + 16 g + 8 (j & 1) ..
  auto fetch = [&](KStep<FP8>& d, uint32_t x) __attribute__((always_inline)) {
    int32_t page[4];
    d.there = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      page[i] = table[min((x + 16 * i) >> a.p.page_shift, a.p.table_stride - 1)];
      if (uint32_t(page[i]) < a.p.n_pages) d.there |= 1u << i;
      else page[i] = 0;  // read as page 0, and what comes of it is masked
    }
    const int32_t p0 = page[0], p1 = page[1], p2 = page[2], p3 = page[3];
    const int32_t mine = col & 8 ? (col & 4 ? p3 : p2) : (col & 4 ? p1 : p0);
    const size_t run = page_row(a.p, mine, head, (x + 16 * (col >> 2)) & mask);
    const uint8_t* p = a.st.k + (run + (col & 3)) * kPageDim * EL + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int i = 0; i < (FP8 ? 2 : 4); i++)
        d.k[(FP8 ? 2 : 4) * t + i] = *reinterpret_cast<const u32x4*>(p + 4 * t * kPageDim * EL + 64 * i);
    if constexpr (FP8) d.exp = *reinterpret_cast<const u32x4*>(a.st.k_exp + run);
  };
  const uint32_t r = min(col, q.rows - 1), token = r / a.group;
  const int32_t last = col < q.rows ? int32_t(max(min(q.first + token, capacity_of(a.p) - 1), int64_t(-1))) : -1;
  const int32_t free_to = int32_t(max(min(q.first, capacity_of(a.p) - 1), int64_t(-1)));
  const uint64_t e0 = (uint64_t(q.row0) + token) * a.q_stride + (head * a.group + (r - token * a.group)) * kPageDim;
  bf16x8 f[4][NS];
  u32x4 raw[4][BF16_ROWS ? 1 : 2];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t d = FP8 ? 64 * (j / 2) + 16 * g + 8 * (j & 1) : 32 * j + 8 * g;
#pragma unroll
    for (int i = 0; i < (BF16_ROWS ? 1 : 2); i++)
      raw[j][i] = *reinterpret_cast<const u32x4*>(a.q + (e0 + d) * (BF16_ROWS ? 2 : 4) + 16 * i);
  }
  KStep<FP8> d0, d1;
  uint32_t x = x0 + 64 * wave;
  fetch(d0, x);
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if constexpr (BF16_ROWS) {
      f[j][0] = __builtin_bit_cast(bf16x8, raw[j][0]);
    } else {
      u32x4 part[3];
      cut_f32(raw[j], part);
#pragma unroll
      for (int n = 0; n < 3; n++) f[j][n] = __builtin_bit_cast(bf16x8, part[n]);
    }
  }
  const uint64_t stride = uint64_t(a.blocks) * a.span;
  float* const kept = a.scores + (uint64_t(s) * a.p.n_kv + head) * a.few * stride;
  float m = -INFINITY, l = 0.f;
  auto step = [&](const KStep<FP8>& d, uint32_t x) __attribute__((always_inline)) {
    f32x4 v[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      v[t] = 0.f;
      float scale = 1.f;
      if constexpr (FP8) scale = exp_scale(d.exp[t] >> (8 * (col & 3)) & 0xFFu);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        bf16x8 k;
        if constexpr (FP8) k = fp8_bf16(d.k[2 * t + j / 2][2 * (j & 1)], d.k[2 * t + j / 2][2 * (j & 1) + 1], scale);
        else k = __builtin_bit_cast(bf16x8, d.k[4 * t + j]);
#pragma unroll
        for (int n = NS - 1; n >= 0; n--) v[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, f[j][n], v[t], 0, 0, 0);
      }
    }
    if (int32_t(x + 63) > free_to || d.there != 15) {
      const bool there = d.there >> g & 1;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (int32_t(x + 16 * g + 4 * t + e) > last || !there) v[t][e] = -INFINITY;
    }
    // through LDS, so that each store instruction writes whole rows of 64 positions
    if (col < q.rows)
#pragma unroll
      for (int t = 0; t < 4; t++) *reinterpret_cast<f32x4*>(&out[wave][col][16 * g + 4 * t]) = v[t];
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses keep their order)
    for (uint32_t i = lane >> 4; i < q.rows; i += 4)
      *reinterpret_cast<f32x4*>(kept + i * stride + x + 4 * col) = *reinterpret_cast<const f32x4*>(&out[wave][i][4 * col]);
    float top = v[0][0];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) top = fmaxf(top, v[t][e]);
    top = fmaxf(m, top * a.c);
    const float ref = top == -INFINITY ? 0.f : top;
    l *= rebase(m, top);
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) l += exp2_fast(fmaf(v[t][e], a.c, -ref));
    m = top;
  };
  while (x < x1) {
    fetch(d1, min(x + 256, x1 - 1) & ~63u);  // (past the end: positions that are there, unused)
    step(d0, x);
    x += 256;
    if (x >= x1) break;
    fetch(d0, min(x + 256, x1 - 1) & ~63u);
    step(d1, x);
    x += 256;
  }
  // the four groups of lanes, then the four waves
#pragma unroll
  for (int d = 16; d < 64; d *= 2) {
    const float om = __shfl_xor(m, d), ol = __shfl_xor(l, d), top = fmaxf(m, om);
    l = l * rebase(m, top) + ol * rebase(om, top);
    m = top;
  }
  if (g == 0) stat[wave][col] = make_float2(m, l);
  __syncthreads();
  if (tid < q.rows) {
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) m = fmaxf(m, stat[w][tid].x);
#pragma unroll
    for (int w = 0; w < 4; w++) l = fmaf(stat[w][tid].y, rebase(stat[w][tid].x, m), l);
    a.parts[((uint64_t(s) * a.p.n_kv + head) * a.few + tid) * a.blocks + block] = make_float2(m, l);
  }
}

// The weight of the rows' kept scores, 1024 positions a workgroup: the rows' maxima and sums first, 16 lanes a row.
template <bool FP8, bool BF16_ROWS>
__global__ __launch_bounds__(256) void k_weigh_kept(WeighArgs a, uint32_t blocks) {
  __shared__ float2 stat[kFewRows];
  const uint32_t tid = threadIdx.x, head = blockIdx.x % a.p.n_kv, s = blockIdx.x / a.p.n_kv / blocks;
  const uint32_t item = s * a.p.n_kv + head;
  const Span q = span_of(a, s);
  const uint32_t x0 = blockIdx.x / a.p.n_kv % blocks * 1024, j = x0 + 4 * tid;
  if (x0 >= q.end) return;
  float* const mass = a.mass + uint64_t(item) * a.mass_stride;
  if (q.rows > a.few) {
    // more rows than max_new says: a row after another, its maximum, its sum, its weights, by plain sums
    __shared__ float2 part[256];
    const int32_t* const table = a.p.table + size_t(s) * a.p.table_stride;
    float sum[4] = {};
    for (uint32_t r = 0; r < q.rows; r++) {
      const uint32_t token = r / a.group;
      const uint64_t e = (uint64_t(q.row0) + token) * a.q_stride + (head * a.group + (r - token * a.group)) * kPageDim;
      const uint32_t end = uint32_t(max(min(q.first + token + 1, capacity_of(a.p)), int64_t(0)));
      auto score = [&](uint32_t p) {
        const int32_t page = p < end ? table[p >> a.p.page_shift] : -1;
        if (uint32_t(page) >= a.p.n_pages) return -INFINITY;
        const size_t row = page_row(a.p, page, head, p & ((1u << a.p.page_shift) - 1));
        float v = 0.f;
        for (uint32_t d = 0; d < kPageDim; d++) {
          const float x = BF16_ROWS ? bf16f(reinterpret_cast<const uint16_t*>(a.q)[e + d]) : reinterpret_cast<const float*>(a.q)[e + d];
          const float k = FP8 ? __builtin_amdgcn_cvt_f32_fp8(a.st.k[row * kPageDim + d], 0)
                              : bf16f(reinterpret_cast<const uint16_t*>(a.st.k)[row * kPageDim + d]);
          v = fmaf(x, k, v);
        }
        return (FP8 ? v * exp_scale(a.st.k_exp[row]) : v) * a.c;
      };
      float m = -INFINITY, l = 0.f;
      for (uint32_t p = tid; p < end; p += 256) {
        const float v = score(p), top = fmaxf(m, v);
        l = l * rebase(m, top) + (v == -INFINITY ? 0.f : exp2_fast(v - top));
        m = top;
      }
      __syncthreads();
      part[tid] = make_float2(m, l);
      __syncthreads();
      m = -INFINITY, l = 0.f;
      for (int i = 0; i < 256; i++) m = fmaxf(m, part[i].x);
      for (int i = 0; i < 256; i++) l = fmaf(part[i].y, rebase(part[i].x, m), l);
      for (int i = 0; i < 4; i++) {
        const float v = j + i < end ? score(j + i) : -INFINITY;
        if (v != -INFINITY) sum[i] += exp2_fast(v - m) / l;
      }
    }
    for (int i = 0; i < 4; i++)
      if (j + i < q.end && !(sum[i] == 0.f)) mass[j + i] += sum[i];
    return;
  }
  const uint64_t stride = uint64_t(a.blocks) * a.span;
  const float* kept = a.scores + uint64_t(item) * a.few * stride + j;
  constexpr uint32_t AT = 4;  // rows whose scores are loaded together, the first of them before the sums are joined
  f32x4 v[AT];
  auto load = [&](uint32_t r0) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < AT; i++)
      if (r0 + i < q.rows && j < q.end) v[i] = *reinterpret_cast<const f32x4*>(kept + (r0 + i) * stride);
  };
  load(0);
  {
    const uint32_t r = tid / 16, lane = tid & 15;
    float m = -INFINITY, l = 0.f;
    if (r < q.rows) {
      const int64_t last = min(q.first + r / a.group, capacity_of(a.p) - 1);
      const uint32_t n = last < 0 ? 0 : uint32_t(last) / a.span + 1;
      const float2* parts = a.parts + (uint64_t(item) * a.few + r) * a.blocks;
      for (uint32_t i = lane; i < n; i += 16) {
        const float2 p = parts[i];
        const float top = fmaxf(m, p.x);
        l = l * rebase(m, top) + p.y * rebase(p.x, top);
        m = top;
      }
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
      const float om = __shfl_xor(m, d), ol = __shfl_xor(l, d), top = fmaxf(m, om);
      l = l * rebase(m, top) + ol * rebase(om, top);
      m = top;
    }
    if (lane == 0) stat[r] = make_float2(m, l == 0.f ? 0.f : 1.f / l);
  }
  __syncthreads();
  if (j >= q.end) return;
  float sum[4] = {};
  for (uint32_t r0 = 0; r0 < q.rows; r0 += AT) {
#pragma unroll
    for (uint32_t n = 0; n < AT; n++) {
      if (r0 + n >= q.rows) break;
      const float2 rs = stat[r0 + n];
#pragma unroll
      for (int i = 0; i < 4; i++) sum[i] += v[n][i] == -INFINITY ? 0.f : exp2_fast(fmaf(v[n][i], a.c, -rs.x)) * rs.y;
    }
    load(r0 + AT);
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (j + i < q.end && !(sum[i] == 0.f)) mass[j + i] += sum[i];
}

// ---- more rows ----
// Joins a row's maxima and sums over its blocks, 16 lanes a row.
__global__ __launch_bounds__(256) void k_weigh_rows(WeighArgs a) {
  const uint32_t heads = a.group * a.p.n_kv, lane = threadIdx.x & 15;
  const uint64_t r = uint64_t(blockIdx.x) * 16 + threadIdx.x / 16;
  const uint32_t t = uint32_t(r / heads);
  if (t >= a.n_rows) return;
  uint32_t lo = 0, hi = a.p.n_seqs;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.p.starts[mid] <= int32_t(t)) lo = mid;
    else hi = mid;
  }
  const Span q = span_of(a, lo);
  if (t < q.row0 || t - q.row0 >= q.rows / a.group) return;
  const int64_t last = min(q.first + (t - q.row0), capacity_of(a.p) - 1);
  const uint32_t n = last < 0 ? 0 : uint32_t(last) / kSpan + 1;
  const float2* parts = a.parts + r * a.blocks;
  float m = -INFINITY, l = 0.f;
  for (uint32_t i = lane; i < n; i += 16) {
    const float2 p = parts[i];
    const float top = fmaxf(m, p.x);
    l = l * rebase(m, top) + p.y * rebase(p.x, top);
    m = top;
  }
#pragma unroll
  for (int d = 1; d < 16; d *= 2) {
    const float om = __shfl_xor(m, d), ol = __shfl_xor(l, d), top = fmaxf(m, om);
    l = l * rebase(m, top) + ol * rebase(om, top);
    m = top;
  }
  if (lane == 0) a.rows[r] = make_float2(m, l == 0.f ? 0.f : 1.f / l);
}

// Adds the sums of the splits to mass, in order.
__global__ __launch_bounds__(256) void k_weigh_add(WeighArgs a) {
  const uint32_t item = blockIdx.x / a.blocks, block = blockIdx.x - item * a.blocks, s = item / a.p.n_kv;
  const uint32_t j = block * kSpan + threadIdx.x;
  const Span q = span_of(a, s);
  if (j >= q.end) return;
  float v = 0.f;
  for (uint32_t i = 0; i < a.splits; i++)
    v += a.sums[((uint64_t(i) * a.p.n_seqs * a.p.n_kv + item) * a.blocks + block) * kSpan + threadIdx.x];
  if (!(v == 0.f)) a.mass[uint64_t(item) * a.mass_stride + j] += v;
}

// How a call is cut up, and what its work holds.
struct WeighCut {
  uint64_t few, span, blocks, splits, parts, rows, sums, scores;  // the last four in bytes
  uint64_t bytes() const { return parts + rows + sums + scores; }
};
WeighCut weigh_cut(uint64_t n_rows, uint64_t n_heads, uint64_t n_kv, uint64_t n_seqs, uint64_t positions, uint64_t max_new) {
  WeighCut c{};
  const uint64_t most = max_new && max_new < n_rows ? max_new : n_rows, items = n_seqs * n_kv;
  const uint64_t rows = max_new ? most * (n_heads / n_kv) : ~0ull;
  if (rows <= kFewRows) {
    c.few = rows ? rows : 1;
    c.span = 1024;
    while (c.span > kSpan && items * ((positions + c.span - 1) / c.span) < 512) c.span /= 2;
  } else {
    c.span = kSpan;
  }
  c.blocks = (positions + c.span - 1) / c.span;
  c.splits = 1;
  if (c.few) {
    c.parts = (items * c.few * c.blocks * sizeof(float2) + 15) / 16 * 16;
    c.scores = items * c.few * c.blocks * c.span * sizeof(float);
    return c;
  }
  // rows are split where the positions alone make fewer than four workgroups a CU, into parts of at least four tiles (3
  // x up to 1024 rows over 4096 positions, both passes: for 512 workgroups 253 us, 1024 231, 2048 229, 4096 239)
  const uint64_t tiles = (most * (n_heads / n_kv) + kTile - 1) / kTile;
  c.splits = (1024 + items * c.blocks - 1) / (items * c.blocks);
  if (c.splits > tiles / 4) c.splits = tiles / 4;
  if (c.splits < 1) c.splits = 1;
  c.parts = (n_rows * n_heads * c.blocks * sizeof(float2) + 15) / 16 * 16;
  c.rows = (n_rows * n_heads * sizeof(float2) + 15) / 16 * 16;
  c.sums = c.splits > 1 ? c.splits * items * c.blocks * kSpan * sizeof(float) : 0;
  return c;
}

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_op_page_weigh_work_bytes(uint64_t n_rows, uint64_t n_heads, uint64_t n_kv_heads, uint64_t n_seqs,
                                     uint64_t positions, uint64_t max_new) {
  if (!n_kv_heads || !n_heads || n_heads % n_kv_heads || !n_seqs || !positions || n_seqs > 65536 || n_kv_heads > 1024 ||
      n_heads > 65536 || positions > 0x7FFFFFFFull || n_rows >= (1ull << 28) / n_heads)
    return 0;
  return qe::weigh_cut(n_rows, n_heads, n_kv_heads, n_seqs, positions, max_new).bytes();
}

int qe_op_page_weigh(const qe_pages* pages, const void* q, uint64_t n_rows, uint64_t n_heads, uint64_t q_stride,
                     uint64_t max_new, int dtype, float* mass, uint64_t mass_stride, void* work, uint64_t work_bytes,
                     void* stream) {
  qe::WeighArgs a{};
  if (int rc = qe::check_pages(pages, &a.p, &a.st)) return rc;
  if (dtype != QE_KV_F32 && dtype != QE_KV_BF16) return qe::set_error(QE_ERR_ARG, "rows are QE_KV_F32 or QE_KV_BF16");
  if (n_heads == 0 || n_heads % a.p.n_kv || n_heads > 65536)
    return qe::set_error(QE_ERR_ARG, "n_heads must be a multiple of n_kv_heads, at most 65536");
  if (n_rows == 0) return QE_OK;
  if (!q || !mass || !work) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_rows >= (1ull << 28) / n_heads) return qe::set_error(QE_ERR_ARG, "need n_rows * n_heads < 2^28");
  const uint64_t el = dtype == QE_KV_F32 ? 4 : 2, capacity = pages->table_stride * pages->page_size;
  if (q_stride < n_heads * qe::kPageDim || q_stride > 0xFFFFFFFFull || q_stride * el % 16)
    return qe::set_error(QE_ERR_ARG, "q_stride must be at least n_heads * 128 elements and a multiple of 16 bytes");
  if (mass_stride < capacity || mass_stride > 0x7FFFFFFFull)
    return qe::set_error(QE_ERR_ARG, "mass_stride must be at least table_stride * page_size, and below 2^31");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(work)) % 16 || reinterpret_cast<uintptr_t>(mass) % 4)
    return qe::set_error(QE_ERR_ARG, "q and work must be 16-byte aligned, mass 4-byte");
  const qe::WeighCut cut = qe::weigh_cut(n_rows, n_heads, a.p.n_kv, a.p.n_seqs, capacity, max_new);
  const uint64_t items = uint64_t(a.p.n_seqs) * a.p.n_kv * cut.blocks;
  if (items * cut.splits >= 1u << 24)
    return qe::set_error(QE_ERR_ARG, "need n_seqs * n_kv_heads * (positions of a table's row / 256) < 2^24");
  if (work_bytes < cut.bytes())
    return qe::set_error(QE_ERR_ARG, "work holds %llu bytes, fewer than qe_op_page_weigh_work_bytes gives",
                         (unsigned long long)work_bytes);
  const qe::Bytes to{mass, 4 * mass_stride * a.p.n_seqs * a.p.n_kv};
  const uint64_t page_bytes = qe_page_bytes(pages->n_pages, pages->page_size, pages->n_kv_heads, pages->kv_dtype);
  const bool fp8 = pages->kv_dtype == QE_KV_FP8;
  if (to.meets({q, ((n_rows - 1) * q_stride + n_heads * qe::kPageDim) * el}) || to.meets({pages->k, page_bytes}) ||
      to.meets({pages->v, page_bytes}) || to.meets({work, work_bytes}) ||
      (fp8 && (to.meets({pages->k_exp, page_bytes / qe::kPageDim}) || to.meets({pages->v_exp, page_bytes / qe::kPageDim}))))
    return qe::set_error(QE_ERR_ARG, "mass must not overlap q, the pages or work");
  a.q = static_cast<const uint8_t*>(q);
  a.q_stride = q_stride;
  a.mass = mass;
  a.mass_stride = mass_stride;
  uint8_t* const base = static_cast<uint8_t*>(work);
  a.parts = reinterpret_cast<float2*>(base);
  a.rows = reinterpret_cast<float2*>(base + cut.parts);
  a.sums = reinterpret_cast<float*>(base + cut.parts + cut.rows);
  a.scores = a.sums;
  a.n_rows = uint32_t(n_rows);
  a.group = uint32_t(n_heads / a.p.n_kv);
  a.blocks = uint32_t(cut.blocks);
  a.splits = uint32_t(cut.splits);
  a.few = uint32_t(cut.few);
  a.span = uint32_t(cut.span);
  a.c = 1.44269504f / sqrtf(float(qe::kPageDim));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const uint32_t grid = uint32_t(items * cut.splits);
  auto go = [&](auto* few, auto* kept, auto* first, auto* second, auto* both) {
    if (a.few) {
      const uint32_t blocks = uint32_t((capacity + 1023) / 1024);
      few<<<grid, 256, 0, st>>>(a);
      kept<<<blocks * a.p.n_seqs * a.p.n_kv, 256, 0, st>>>(a, blocks);
      return;
    }
    if (a.blocks == 1) {
      both<<<grid, 256, 0, st>>>(a);
    } else {
      first<<<grid, 256, 0, st>>>(a);
      qe::k_weigh_rows<<<uint32_t((n_rows * n_heads + 15) / 16), 256, 0, st>>>(a);
      second<<<grid, 256, 0, st>>>(a);
    }
    if (a.splits > 1) qe::k_weigh_add<<<uint32_t(items), 256, 0, st>>>(a);
  };
#define QE_WEIGH(F, B)                                                                                              \
  go(qe::k_weigh_few<F, B>, qe::k_weigh_kept<F, B>, qe::k_weigh<F, B, qe::kStats>, qe::k_weigh<F, B, qe::kSums>, \
     qe::k_weigh<F, B, qe::kBoth>)
  const bool bf16 = dtype == QE_KV_BF16;
  if (fp8 && bf16) QE_WEIGH(true, true);
  else if (fp8) QE_WEIGH(true, false);
  else if (bf16) QE_WEIGH(false, true);
  else QE_WEIGH(false, false);
#undef QE_WEIGH
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "page weigh launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
