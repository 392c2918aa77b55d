// qe_op_page_attention: causal GQA attention of packed new tokens over the paged K/V cache. No
// reference counterpart (its attention reads one sequence's contiguous cache, one token at a time:
// cpu_inference.rs:144-162).
//
//   out[t][h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(q[t][h] . k_j / sqrt(128)),  j = 0 .. pos(t),
//
// over the positions j whose page is there; a row that has none gives zeros.
//
// How the work is cut. The rows of a sequence and KV head are (token, q head) pairs, token first; an
// item is one tile of them (16 to 256 rows) with its positions in blocks of 64, up to the last
// position that any of its rows attends. The blocks of all items, in order (sequence, head, tile),
// are dealt to a fixed number of workgroups in equal contiguous parts, whatever the lengths: the
// lengths are device data, so the host cannot choose a split by them, and a batch of ragged lengths
// keeps every CU busy to the end. A workgroup that holds all blocks of an item writes its rows out;
// one that holds a part leaves the part's unnormalised sums, maxima and weight sums in `work`, and
// k_page_join adds the parts of an item in order. (Short items are dealt out whole: find_part.) The
// cut depends on the plan alone, so results are the same every time.
#include "pages.h"

#include "device_common.h"
#include "dma.h"
#include "status.h"

#include <type_traits>

namespace qe {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kBlock = 64;    // positions
// Weights are 2^(score - m) with m the largest score so far, or up to kSlack below it: sums are only put
// on a new m when a score exceeds it by that much (in some row of 32 one is a little larger in most blocks).
// So a weight is up to 2^8, and sums over up to 2^31 positions hold V up to 2^88 in f32.
constexpr float kSlack = 8.f;
constexpr uint32_t kWholeBlocks = 32, kSpare = 1, kSpareCut = 3, kFewTiles = 4;  // see find_part
constexpr uint32_t kNowhere = 0xFFFFFFFFu;
constexpr uint32_t kPartRow = 130; // floats of a part's row: 128 sums, then (apart) the maximum and the weight sum

struct AttnArgs {
  PagePlan p;
  PageStore st;
  const uint8_t* q;
  uint8_t* out;
  uint64_t q_stride, out_stride;  // elements
  float* parts;                   // [workgroup][2][rows of a tile][kPartRow]
  struct Joint* joints;           // [workgroup]
  uint32_t n_rows, group;
  uint32_t group_magic, group_shift;  // r / group = (2 r * magic >> 32) >> shift for r < 2^31
  uint32_t whole_items;           // 1: an item counts as one block and is never cut (a call without a join says
                                  // so; else each workgroup finds out by the lengths)
  uint32_t join;                  // a join follows
  float c;                        // log2(e) / sqrt(128)
};

// An item whose first part is the last one of a workgroup: parts of `n` workgroups from there (0: none). And the
// workgroup of the first part of the item that this one's first part goes on with, where it helps to join it
// (else kNowhere).
struct Joint {
  uint32_t n, rows, head, first;  // rows of the tile; the first of them among its sequence's rows
  int32_t row0;                   // first packed row of the sequence
  uint32_t from;
};

__device__ __forceinline__ uint32_t token_of(const AttnArgs& a, uint32_t r) {  // r / group
  return __umulhi(2 * r, a.group_magic) >> a.group_shift;
}

// ---- the plan of a sequence: its rows and how far each tile's positions go ----
struct Seq {
  int32_t first;   // position of its first row (may be negative: such rows attend nothing)
  int32_t row0;    // first packed row
  uint32_t rows;   // new tokens * group
  __device__ uint32_t tiles(uint32_t R) const { return (rows + R - 1) / R; }
};

__device__ __forceinline__ Seq read_seq(const AttnArgs& a, uint32_t s) {
  const int64_t b = a.p.starts[s], e = a.p.starts[s + 1];
  const int64_t lo = b < 0 ? 0 : b, hi = e < int64_t(a.n_rows) ? e : int64_t(a.n_rows);
  Seq q;
  q.row0 = int32_t(lo);
  q.rows = hi > lo ? uint32_t(hi - lo) * a.group : 0;
  // its last row is at lens[s] - 1 < 2^31; below -2^31 every row is at a negative position
  const int64_t first = int64_t(a.p.lens[s]) - (e - lo);
  q.first = int32_t(first > -0x80000000ll ? first : -0x80000000ll);
  return q;
}

// The last position that row r of a sequence's rows attends: its own, or the table's last where it lies behind
// that (what a step or block holds past the table is masked by it, like any later position); negative: none.
__device__ __forceinline__ int32_t row_position(const AttnArgs& a, const Seq& q, uint32_t r) {
  return min(q.first + int32_t(token_of(a, r)), int32_t((a.p.table_stride << a.p.page_shift) - 1));
}
// Positions that rows up to r attend: 0 .. limit - 1.
__device__ __forceinline__ uint32_t row_limit(const AttnArgs& a, const Seq& q, uint32_t r) {
  const int32_t pos = row_position(a, q, r);
  return pos < 0 ? 0 : uint32_t(pos) + 1;
}
__device__ __forceinline__ uint32_t tile_limit(const AttnArgs& a, const Seq& q, uint32_t tile, uint32_t R) {
  return row_limit(a, q, min((tile + 1) * R, q.rows) - 1);
}
// A tile that attends nothing still counts one block: its rows are zeros that someone writes.
__device__ __forceinline__ uint32_t tile_blocks(const AttnArgs& a, const Seq& q, uint32_t tile, uint32_t R) {
  return a.whole_items ? 1 : max((tile_limit(a, q, tile, R) + kBlock - 1) / kBlock, 1u);
}
__device__ uint64_t seq_blocks(const AttnArgs& a, const Seq& q, uint32_t R) {
  uint64_t n = 0;
  const uint32_t t = q.tiles(R);
  if (a.whole_items) return t;
  for (uint32_t i = 0; i < t; i++) n += tile_blocks(a, q, i, R);
  return n;
}

// Where a workgroup is in the list of all blocks.
struct Cursor {
  Seq q;
  uint32_t seq, head, tile, block, blocks;  // block of the tile's `blocks`
};

struct PlanShared {
  uint64_t sum[512];
  Cursor at;
};

// The next tile with rows after `cu`'s (false: there is none).
__device__ __forceinline__ bool next_tile(const AttnArgs& a, Cursor& cu, uint32_t R) {
  cu.block = 0;
  if (++cu.tile >= cu.q.tiles(R)) {
    cu.tile = 0;
    if (++cu.head >= a.p.n_kv) {
      cu.head = 0;
      do {
        if (++cu.seq >= a.p.n_seqs) return false;
        cu.q = read_seq(a, cu.seq);
      } while (cu.q.rows == 0);
    }
  }
  cu.blocks = tile_blocks(a, cu.q, cu.tile, R);
  return true;
}

// The block `at` blocks into the list of sequence s's.
__device__ __forceinline__ Cursor cursor_in(const AttnArgs& a, uint32_t s, const Seq& q, uint64_t one, uint64_t at, uint32_t R) {
  Cursor cu;
  cu.q = q;
  cu.seq = s;
  cu.head = uint32_t(at / one);
  uint64_t rest = at % one;
  cu.tile = 0;
  while (rest >= (cu.blocks = tile_blocks(a, q, cu.tile, R))) {
    rest -= cu.blocks;
    cu.tile++;
  }
  cu.block = uint32_t(rest);
  return cu;
}

// A value that all lanes hold, in a scalar register: what comes out of LDS would stay in vector
// registers, and everything worked out from it with it.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ Cursor uniform(const Cursor& c) {
  Cursor u;
  u.q.first = int32_t(uniform(uint32_t(c.q.first)));
  u.q.row0 = int32_t(uniform(uint32_t(c.q.row0)));
  u.q.rows = uniform(c.q.rows);
  u.seq = uniform(c.seq);
  u.head = uniform(c.head);
  u.tile = uniform(c.tile);
  u.block = uniform(c.block);
  u.blocks = uniform(c.blocks);
  return u;
}

// The cursor of the lane that has `here`, to all lanes.
__device__ __forceinline__ void take_from(Cursor& cu, bool here) {
  const uint32_t owner = uniform(uint32_t(__builtin_ctzll(__ballot(here))));
  auto from = [&](uint32_t v) { return from_lane(v, int(owner)); };
  cu.q.first = int32_t(from(uint32_t(cu.q.first)));
  cu.q.row0 = int32_t(from(uint32_t(cu.q.row0)));
  cu.q.rows = from(cu.q.rows);
  cu.seq = from(cu.seq);
  cu.head = from(cu.head);
  cu.tile = from(cu.tile);
  cu.block = from(cu.block);
  cu.blocks = from(cu.blocks);
}

// How many parts of q blocks b blocks make. (b + q - 1/2) / q is at least 1/2q from a whole number, which f32's
// rounding of it cannot reach for b up to 2^20 and q up to 2^20.
__device__ __forceinline__ uint32_t parts_of(uint32_t b, uint32_t q) {
  return uint32_t((float(b + q) - 0.5f) * __builtin_amdgcn_rcpf(float(q)));
}

// Workgroup w's part of the list, of W parts of `per` blocks: where it begins and how many blocks it has
// (0: none). (A part is far below 2^32 blocks: that many are 70 TB of K and V.) A wave finds it alone where a
// lane can have a sequence each; else each thread sums a contiguous range of sequences, and the one whose
// range holds the block walks it. W is a power of two.
//
// A second piece costs a workgroup some 5 us (its q, its first loads, its sums through LDS and the join), so
// parts keep to the items in three cases (times in a graph; f32 rows over bf16 pages, 16 over 8 heads, where not
// said otherwise):
// - Items that are short and about as many as the workgroups are not cut but dealt out whole: the longest up to
//   32 blocks and up to twice a workgroup's share. bf16 rows over e4m3 pages, 32 over 8 heads: 32 sequences of up
//   to 1000 positions 24 us cut, so 15; up to 2000 34 and 24; 4 of up to 2000 (13 times the share) 12 cut, 21
//   whole; 64 of up to 4000 60 cut, 63 whole.
// - Few items are cut into equally many parts each, where the longest part is at most a block over the even
//   share: a chunk of 512 over 2048 positions 42.8 us dealt evenly, so 38.3 (bf16 rows 33.0 and 30.1); one row
//   over 4225 positions 13.9 and 12.1; 3 chunks of up to 300, whose parts would be 2 to 4 blocks over, 41 and 46.
// - Else few items (of few tiles a sequence, so that counting is quick) are cut into parts of equally many blocks,
//   with the last of an item shorter, where up to 3 blocks over the even share give no more parts than
//   workgroups: 16 x 8 of up to 2048 positions, 5 rows each, e4m3 21.9 us dealt evenly, so 18.9 (12 rows 33.7 and
//   30.0; bf16 pages 26.6 and 26.4); 10 x 8 of up to 3000, one row 23.2 and 21.7.
__device__ __forceinline__ uint32_t find_part(AttnArgs& a, uint32_t w, uint32_t W, uint32_t R, PlanShared& sh,
                                              uint32_t& per_out, Cursor& cu) {
  const uint32_t tid = threadIdx.x, log_w = 31 - __builtin_clz(W);
  auto split = [&](uint64_t total) { return (total + W - 1) >> log_w; };
  auto longest_whole = [&](uint64_t total) { return min(uint64_t(kWholeBlocks), 2 * split(total)); };
  if (a.p.n_seqs <= 64) {
    const uint32_t lane = tid & 63;
    Seq q{};
    uint64_t one = 0;
    uint32_t longest = 0, tiles = 0;
    if (lane < a.p.n_seqs) {
      q = read_seq(a, lane);
      one = seq_blocks(a, q, R);
      tiles = q.tiles(R);
      if (tiles) longest = tile_blocks(a, q, tiles - 1, R);
    }
    const uint64_t mine = one * a.p.n_kv;
    const uint32_t my_items = tiles * a.p.n_kv;
    const uint64_t up_to = wave_scan(mine), total = from_lane(up_to, 63);  // blocks of the sequences up to the lane's
    const uint32_t up_items = wave_scan(my_items), items = from_lane(up_items, 63);
    uint64_t per = split(total), at = w * per;
    uint32_t each = 0;  // parts of every item
    if (!a.whole_items) {
      if (!__any(longest > longest_whole(total))) a.whole_items = 1;
      else if (items <= W) {
        each = W / items;
        if (__any(longest > each * (per + kSpare))) each = 0;
      }
    }
    uint32_t most = 0, parts = 0;  // blocks of a part at most; parts of a head of the lane's sequence
    if (!a.whole_items && !each && items <= W && !__any(tiles > kFewTiles || longest > 1u << 20)) {
      uint32_t cut[kSpareCut + 1] = {};
      for (uint32_t i = 0; i < tiles; i++) {
        const uint32_t b = tile_blocks(a, q, i, R);
#pragma unroll
        for (uint32_t c = 0; c <= kSpareCut; c++) cut[c] += parts_of(b, uint32_t(per) + c);
      }
#pragma unroll
      for (int c = kSpareCut; c >= 0; c--) {
        if (from_lane(wave_scan(cut[c] * a.p.n_kv), 63) <= W) {
          most = uint32_t(per) + c;
          parts = cut[c];
        }
      }
      if (most) {
        const uint32_t up_parts = wave_scan(parts * a.p.n_kv);
        const bool here = w < up_parts && w >= up_parts - parts * a.p.n_kv;
        if (w >= from_lane(up_parts, 63)) return 0;
        if (here) {
          uint32_t in = w - (up_parts - parts * a.p.n_kv), n;
          cu.q = q;
          cu.seq = lane;
          cu.head = in / parts;
          in -= cu.head * parts;
          cu.tile = 0;
          while (in >= (n = parts_of(cu.blocks = tile_blocks(a, q, cu.tile, R), most))) {
            in -= n;
            cu.tile++;
          }
          cu.block = in * most;
        }
        per_out = uniform(most);
        take_from(cu, here);
        return uniform(min(most, cu.blocks - cu.block));
      }
    }
    const bool by_items = each || a.whole_items;
    if (by_items) {
      per = each ? 1 : split(items);
      at = each ? w / each : w * per;
    }
    const uint64_t end = by_items ? items : total;
    per_out = uniform(uint32_t(per));
    if (at >= end) return 0;
    const uint64_t to = by_items ? up_items : up_to, from_here = by_items ? my_items : mine;
    const bool here = at < to && at >= to - from_here;
    if (here) {
      if (by_items) {
        const uint32_t in = uint32_t(at - (to - from_here));
        cu.q = q;
        cu.seq = lane;
        cu.head = in / tiles;
        cu.tile = in - cu.head * tiles;
        cu.block = 0;
        cu.blocks = 1;
      } else {
        cu = cursor_in(a, lane, q, one, at - (to - from_here), R);
      }
    }
    take_from(cu, here);
    if (each) {
      cu.blocks = tile_blocks(a, cu.q, cu.tile, R);
      per_out = uniform((cu.blocks + each - 1) / each);
      cu.block = uniform((w % each) * per_out);
      return cu.block < cu.blocks ? uniform(min(per_out, cu.blocks - cu.block)) : 0;
    }
    return uniform(uint32_t(per < end - at ? per : end - at));
  }
  const uint32_t T = blockDim.x, each = (a.p.n_seqs + T - 1) / T;
  const uint32_t s0 = min(tid * each, a.p.n_seqs), s1 = min(s0 + each, a.p.n_seqs);
  uint64_t mine = 0;
  uint32_t longest = 0;
  auto sum = [&]() __attribute__((always_inline)) {
    mine = 0;
    for (uint32_t s = s0; s < s1; s++) {
      const Seq q = read_seq(a, s);
      mine += seq_blocks(a, q, R);
      if (q.rows) longest = max(longest, tile_blocks(a, q, q.tiles(R) - 1, R));
    }
    mine *= a.p.n_kv;
    sh.sum[tid] = mine;
    __syncthreads();
    for (uint32_t d = 1; d < T; d *= 2) {
      const uint64_t v = tid >= d ? sh.sum[tid - d] : 0;
      __syncthreads();
      sh.sum[tid] += v;
      __syncthreads();
    }
    return sh.sum[T - 1];
  };
  uint64_t total = sum();
  if (!a.whole_items && !__syncthreads_or(longest > longest_whole(total))) {
    a.whole_items = 1;
    total = sum();
  }
  const uint64_t per = split(total), at = w * per;
  uint64_t before = sh.sum[tid] - mine;
  if (at >= before && at < sh.sum[tid]) {
    for (uint32_t s = s0; s < s1; s++) {
      const Seq q = read_seq(a, s);
      const uint64_t one = seq_blocks(a, q, R);
      if (at < before + one * a.p.n_kv) {
        sh.at = cursor_in(a, s, q, one, at - before, R);
        break;
      }
      before += one * a.p.n_kv;
    }
  }
  __syncthreads();
  per_out = uniform(uint32_t(per));
  if (at >= total) return 0;
  cu = uniform(sh.at);
  return uniform(uint32_t(per < total - at ? per : total - at));
}

// How many of the workgroups of an item's n parts join it: more than one where a row's 16 threads would have more
// than two rounds of parts. Small tiles: they share the rows; large ones (R >= 128): the dims, a power of two of them.
__device__ __forceinline__ uint32_t joiners(uint32_t n, uint32_t rows, uint32_t R) {
  if (R < 128) return n * min(rows, 16u) > 128 ? min(n, 16u) : 1;
  return n > 64 ? 16 : n > 32 ? 8 : n > 16 ? 4 : 1;
}

// The joint of workgroup w before it has begun an item of its own: its first part is at cu, if it has one (`left`).
__device__ __forceinline__ void goes_on(Joint& j, uint32_t w, uint32_t left, uint32_t per, const Cursor& cu, uint32_t R) {
  j.n = 0;
  j.from = kNowhere;
  if (left && cu.block) {
    const uint32_t before = (cu.block + per - 1) / per, n = before + (cu.blocks - cu.block + per - 1) / per;
    if (joiners(n, min(cu.q.rows - cu.tile * R, R), R) > 1) j.from = w - before;
  }
}
// the item at cu begins a joint of n workgroups (`from` stays)
__device__ __forceinline__ void begin_joint(Joint& j, uint32_t n, const Cursor& cu, uint32_t R) {
  j.n = n;
  j.rows = min(cu.q.rows - cu.tile * R, R);
  j.head = cu.head;
  j.first = cu.tile * R;
  j.row0 = cu.q.row0;
}

// a workgroup's place in the list: consecutive parts on one XCD (workgroups go to the 8 XCDs in turn)
__device__ __forceinline__ uint32_t part_index() {
  const uint32_t n = gridDim.x;
  return n % 8 ? blockIdx.x : (blockIdx.x % 8) * (n / 8) + blockIdx.x / 8;
}

// v, of which the compiler does not know that it is the same in every round of a loop: what is worked out
// from it once an item then does not stay in registers over the loop on blocks.
__device__ __forceinline__ uint32_t afresh(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// ---- arithmetic ----
// maximum over the four groups of 16 lanes, to all of them
__device__ __forceinline__ float max_groups(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_groups(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// the same over the two halves of a wave
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 2^x by the hardware (1 ulp; results below 2^-126 are 0, which a weight relative to the largest may be)
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// the factor from sums relative to maximum `from` to sums relative to `to` >= from
__device__ __forceinline__ float rebase(float from, float to) { return from == to ? 1.f : exp2_fast(from - to); }

// 8 floats as NS bf16 parts that add up to them: 1 rounded to nearest, or 3 cut (8 + 8 + 8 of f32's 24
// bits: nothing is lost), so that NS matrix products against bf16 values keep f32's precision. bf16 rows take
// their weights as 1: each is off by at most 2^-8 of itself, as every value of their q and out is, and a second
// part would double the products of P V. Against 64 bits the result is off by 0.0023 (relative, 64 chats of up to
// 8192 positions); f32 weights with the same rounding of out leave 0.0017.
template <int NS>
__device__ __forceinline__ void split_bf16(const float (&x)[8], bf16x8 (&o)[NS]) {
  if constexpr (NS == 1) {
    u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; i++)
      u[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), bf16x2));
    o[0] = __builtin_bit_cast(bf16x8, u);
  } else {
    static_assert(NS == 3, "1 or 3");
    u32x4 h, m, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t a[3], b[3];
      auto cut = [](float v, uint32_t (&w)[3]) {
        w[0] = __float_as_uint(v);
        const float r = v - __uint_as_float(w[0] & 0xFFFF0000u);
        w[1] = __float_as_uint(r);
        w[2] = __float_as_uint(r - __uint_as_float(w[1] & 0xFFFF0000u));
      };
      cut(x[2 * i], a);
      cut(x[2 * i + 1], b);
      // the upper halves of b and a
      h[i] = __builtin_amdgcn_perm(b[0], a[0], 0x07060302u);
      m[i] = __builtin_amdgcn_perm(b[1], a[1], 0x07060302u);
      l[i] = __builtin_amdgcn_perm(b[2], a[2], 0x07060302u);
    }
    o[0] = __builtin_bit_cast(bf16x8, l);
    o[1] = __builtin_bit_cast(bf16x8, m);
    o[2] = __builtin_bit_cast(bf16x8, h);
  }
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
__device__ __forceinline__ float byte_scale(uint32_t w, int i) {  // 2^(e - 127) of byte i of w
  return __uint_as_float((i == 3 ? w >> 1 : w << (23 - 8 * i)) & 0x7F800000u);
}

// Clears the values of two bf16 (e4m3: four) that are not finite and says whether there were any.
template <bool FP8>
__device__ __forceinline__ uint32_t clear_foul(uint32_t& u) {
  uint32_t bad;
  if constexpr (FP8) {
    bad = (((u & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;  // bytes 0x7F and 0xFF, as 1 each
    u &= ~(bad * 0xFFu);
  } else {
    bad = ((u & 0x7F80u) == 0x7F80u ? 1u : 0u) | ((u & 0x7F800000u) == 0x7F800000u ? 0x10000u : 0u);
    u &= ~(bad * 0xFFFFu);
  }
  return bad;
}
// Element i of V as a float (without its scale).
template <bool FP8>
__device__ __forceinline__ float v_value(const uint8_t* v, size_t i) {
  if constexpr (FP8) return __builtin_amdgcn_cvt_f32_fp8(v[i], 0);
  else return bf16f(reinterpret_cast<const uint16_t*>(v)[i]);
}

// 8 values of a row of q as floats
template <bool BF16_ROWS>
__device__ __forceinline__ void load_q8(const uint8_t* q, uint64_t element, float (&x)[8]) {
  if constexpr (BF16_ROWS) {
    const u32x4 u = *reinterpret_cast<const u32x4*>(q + element * 2);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  } else {
    const f32x4 u = *reinterpret_cast<const f32x4*>(q + element * 4);
    const f32x4 v = *reinterpret_cast<const f32x4*>(q + element * 4 + 16);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[i] = u[i];
      x[i + 4] = v[i];
    }
  }
}
template <bool BF16_ROWS>
__device__ __forceinline__ void store_out8(uint8_t* out, uint64_t element, const float (&x)[8]) {
  if constexpr (BF16_ROWS) {
    bf16x8 o[1];
    split_bf16<1>(x, o);
    *reinterpret_cast<bf16x8*>(out + element * 2) = o[0];
  } else {
    *reinterpret_cast<f32x4*>(out + element * 4) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(out + element * 4 + 16) = f32x4{x[4], x[5], x[6], x[7]};
  }
}
// element of row r of a tile's item in rows of `stride` elements
__device__ __forceinline__ uint64_t row_element(const AttnArgs& a, const Seq& q, uint32_t head, uint32_t r,
                                                uint64_t stride) {
  const uint32_t t = token_of(a, r);
  return (uint64_t(q.row0) + t) * stride + (head * a.group + (r - t * a.group)) * kPageDim;
}

// ---------------------------------------------------------------------------------------------
// Few rows: tiles of 16 NQ rows, the positions of a part dealt to the workgroup's four waves in steps
// of 32 (bf16) or 64 (e4m3) positions, 16 KB of K and V a step.
//
// Bound by the K/V bytes, so the layout serves the loads. Scores are computed transposed, S^T = K Q^T
// with v_mfma_f32_16x16x32_bf16: operand A's lane l holds row l % 16 of K, which may be any position,
// and result lane l holds column (row of q) l % 16 and, of group g = l / 16, rows 4 g .. 4 g + 3.
// Out^T = V^T P^T wants in lane l of operand B the weights of q row l % 16 at 8 positions, in A the
// same positions of dim l % 16. With K's rows taken in the order below, a lane's results of two (e4m3:
// four) score tiles are the weights of consecutive positions from 8 g (16 g), that is B as it stands,
// and A is 16 bytes of one line of the transposed V page. So K and V go from memory to registers to
// the matrix cores, with no LDS, no exchange between lanes but the maximum, and no barrier until a
// part's end. The loads of a step are issued a step ahead (the page numbers two).
//
// Measured: a row of each of 64 chats of up to 8192 positions, 32 over 8 heads, e4m3 (587 MB): 106 us, 5.5
// TB/s, with the join 112 (a large copy reads and writes 4.9; V without non-temporal loads 10 more); 5 rows of each of 16 chats of 2048, 16 over 8 heads, bf16 (95 MB):
// 26 us; one row over 197 positions: 7.3 us, a launch and four load latencies (plan, page numbers, K and V, out).
// ---------------------------------------------------------------------------------------------
template <bool FP8>
struct StepData {
  u32x4 k[8], v[8];
  u32x4 ke, ve;     // e4m3: exponents of the 16 positions of the lane's K rows, and of its V
  bool there;       // the page of the lane's V (and scores) is
};

template <bool FP8, bool BF16_ROWS, int NQ>
__global__ __launch_bounds__(256, BF16_ROWS && NQ == 1 ? 2 : 1) void k_page_attn_rows(AttnArgs a) {
  constexpr int NS = BF16_ROWS ? 1 : 3, R = 16 * NQ, KEYS = FP8 ? 64 : 32, NT = KEYS / 16, EL = FP8 ? 1 : 2;
  constexpr int LDO = 132;  // floats of a row's sums in LDS
  __shared__ PlanShared sh;
  __shared__ __align__(16) float sums[4][R][LDO];
  __shared__ float top[4][R], mass[4][R];
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t w = part_index();
  Cursor cu;
  uint32_t per;
  uint32_t left = uniform(find_part(a, w, gridDim.x, R, sh, per, cu));
  cu = uniform(cu);
  per = uniform(per);
  a.whole_items = uniform(a.whole_items);
  if (tid == 0 && a.join) goes_on(a.joints[w], w, left, per, cu, R);
  if (left == 0) return;
  const uint32_t whole_part = left;
  const uint32_t ps_mask = (1u << a.p.page_shift) - 1;
  float* const my_parts = a.parts + size_t(w) * 2 * R * kPartRow;

  while (true) {
    const uint32_t take = min(cu.blocks - cu.block, left);
    const uint32_t limit = tile_limit(a, cu.q, cu.tile, R);
    const uint32_t rows = min(cu.q.rows - cu.tile * R, uint32_t(R));
    // the positions of this part, in steps
    const uint32_t first = cu.block * kBlock, last = a.whole_items ? limit : min((cu.block + take) * kBlock, limit);
    const uint32_t head = cu.head;
    // the least position any row attends up to: below it no score is masked
    const int32_t free_to = row_position(a, cu.q, cu.tile * R);
    const bool one_token = token_of(a, cu.tile * R) == token_of(a, cu.tile * R + rows - 1);
    int32_t row_pos[NQ];
    bf16x8 qf[NQ][4][NS];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      const uint32_t lane = afresh(tid & 63), col = lane & 15, g = lane >> 4;
      const uint32_t r = cu.tile * R + 16 * n + col;
      const bool real = r < cu.q.rows;
      row_pos[n] = real ? row_position(a, cu.q, r) : -1;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t d = FP8 ? 64 * (j / 2) + 16 * g + 8 * (j & 1) : 32 * j + 8 * g;
        float x[8] = {};
        if (real) load_q8<BF16_ROWS>(a.q, row_element(a, cu.q, head, r, a.q_stride) + d, x);
        split_bf16<NS>(x, qf[n][j]);
      }
    }
    f32x4 acc[NQ][8];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // the 16 positions a lane's K rows and its V lie in, counted from the step's start
    const uint32_t k16 = FP8 ? (col >> 2) * 16 : (col >> 3) * 16, v16 = FP8 ? g * 16 : (g >> 1) * 16;
    const uint32_t k_in = (FP8 ? (col & 3) : 8 * ((col >> 2) & 1) + (col & 3)) * kPageDim * EL + 16 * g;
    const uint32_t v_in = col * 16 * EL + (FP8 ? 0 : 16 * (g & 1));
    const int32_t* const table = a.p.table + size_t(cu.seq) * a.p.table_stride;
    auto look_up = [&](uint32_t x, int32_t& kp, int32_t& vp) __attribute__((always_inline)) {
      kp = table[min((x + k16) >> a.p.page_shift, a.p.table_stride - 1)];
      vp = table[min((x + v16) >> a.p.page_shift, a.p.table_stride - 1)];
    };
    auto load = [&](StepData<FP8>& d, uint32_t x, int32_t kp, int32_t vp) __attribute__((always_inline)) {
      // a page that is not there is read as page 0, and what comes of it is masked
      d.there = uint32_t(vp) < a.p.n_pages;
      const size_t kr = page_row(a.p, uint32_t(kp) < a.p.n_pages ? kp : 0, head, (x + k16) & ps_mask);
      const size_t vr = page_row(a.p, d.there ? vp : 0, head, (x + v16) & ps_mask);
      const uint8_t* ka = a.st.k + kr * kPageDim * EL + k_in;
      const uint8_t* va = a.st.v + vr * kPageDim * EL + v_in;
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int j = 0; j < 8 / NT; j++)
          d.k[t * (8 / NT) + j] = *reinterpret_cast<const u32x4*>(ka + t * 4 * kPageDim * EL + 64 * j);
#pragma unroll
      for (int i = 0; i < 8; i++) d.v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(va + i * 256 * EL));
      if constexpr (FP8) {
        d.ke = *reinterpret_cast<const u32x4*>(a.st.k_exp + kr);
        d.ve = *reinterpret_cast<const u32x4*>(a.st.v_exp + vr);
      }
    };
    uint32_t foul_from = kNowhere;  // the first step that cleared something
    // one step of positions x .. x + KEYS - 1
    auto step = [&](StepData<FP8>& d, uint32_t x) __attribute__((always_inline)) {
      f32x4 s[NQ][NT];
#pragma unroll
      for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int t = 0; t < NT; t++) s[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float ks = 1.f;
        if constexpr (FP8) ks = __uint_as_float(((d.ke[t] >> (8 * (col & 3))) & 0xFFu) << 23);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          bf16x8 kf;
          if constexpr (FP8) kf = fp8_bf16(d.k[2 * t + j / 2][2 * (j & 1)], d.k[2 * t + j / 2][2 * (j & 1) + 1], ks);
          else kf = __builtin_bit_cast(bf16x8, d.k[4 * t + j]);
#pragma unroll
          for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int i = 0; i < NS; i++)
              s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][j][i], s[n][t], 0, 0, 0);
        }
      }
      // positions of this lane's scores and V: base .. base + 4 NT - 1
      const uint32_t base = x + g * (KEYS / 4);
      const bool masked = int32_t(x + KEYS - 1) > free_to || !__all(d.there);
      uint32_t foul = 0;  // V is not finite at a position that only some rows of the tile attend
      if (masked) {
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (int32_t(base + 4 * t + i) > row_pos[n] || !d.there) s[n][t][i] = -INFINITY;
        // V at positions no row attends may hold anything: 0 x NaN is NaN
        const uint32_t ok = d.there && limit > base ? min(limit - base, uint32_t(KEYS / 4)) : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          constexpr uint32_t PER = 4 / EL;
          const uint32_t have = ok > i * PER ? min(ok - i * PER, PER) : 0;
          const uint32_t bits = have == PER ? ~0u : (1u << (8 * EL * have)) - 1;
#pragma unroll
          for (int t = 0; t < 8; t++) d.v[t][i] &= bits;
          if constexpr (FP8) d.ve[i] &= bits;
        }
        if (!one_token) {
#pragma unroll
          for (int t = 0; t < 8; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              uint32_t u = d.v[t][i];
              foul |= clear_foul<FP8>(u);
              d.v[t][i] = u;
            }
        }
      }
      bf16x8 pf[NQ][NT / 2][NS];
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        float mx = s[n][0][0];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[n][t][i]);
        mx = fmaxf(m[n], max_groups(mx) * a.c);
        if (__any(mx > m[n] + kSlack)) {
          const float f = rebase(m[n], mx);
          l[n] *= f;
#pragma unroll
          for (int i = 0; i < 8; i++) acc[n][i] *= f;
          m[n] = mx;
        }
        const float ref = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
        for (int u = 0; u < NT / 2; u++) {
          float e[8];
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float y = exp2_fast(fmaf(s[n][2 * u + i / 4][i & 3], a.c, -ref));
            l[n] += y;
            e[i] = y;
            if constexpr (FP8) e[i] = y == 0.f ? 0.f : y * byte_scale(d.ve[2 * u + i / 4], i & 3);
          }
          split_bf16<NS>(e, pf[n][u]);
        }
      }
#pragma unroll
      for (int t = 0; t < 8; t++)
#pragma unroll
        for (int u = 0; u < NT / 2; u++) {
          bf16x8 vf;
          if constexpr (FP8) vf = fp8_bf16(d.v[t][2 * u], d.v[t][2 * u + 1], 1.f);
          else vf = __builtin_bit_cast(bf16x8, d.v[t]);
#pragma unroll
          for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int i = 0; i < NS; i++)
              acc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n][u][i], acc[n][t], 0, 0, 0);
        }
      if (foul_from == kNowhere && __any(foul != 0)) foul_from = x;
    };

    uint32_t x = first + wave * KEYS;
    if (x < last) {
      StepData<FP8> d0, d1;
      int32_t kp, vp;
      look_up(x, kp, vp);
      load(d0, x, kp, vp);
      look_up(x + 4 * KEYS, kp, vp);
      while (true) {
        // (past the end the loads of a step are of pages that are there, and unused)
        load(d1, x + 4 * KEYS, kp, vp);
        look_up(x + 8 * KEYS, kp, vp);
        step(d0, x);
        x += 4 * KEYS;
        if (x >= last) break;
        load(d0, x + 4 * KEYS, kp, vp);
        look_up(x + 8 * KEYS, kp, vp);
        step(d1, x);
        x += 4 * KEYS;
        if (x >= last) break;
      }
    }

    // what was cleared, to the rows that attend it: infinity and NaN stay what they are under a weight
    for (uint32_t y = foul_from; y < last; y += 4 * KEYS) {
      for (uint32_t j = y; j < min(y + KEYS, limit); j++) {
        const int32_t page = table[j >> a.p.page_shift];
        if (uint32_t(page) >= a.p.n_pages) continue;
        const size_t e = v_element(a.p, page, head, j & ps_mask);
#pragma unroll
        for (int t = 0; t < 8; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float v = v_value<FP8>(a.st.v, e + 16 * (16 * t + 4 * g + i));
            if (!(fabsf(v) < INFINITY))
#pragma unroll
              for (int n = 0; n < NQ; n++)
                if (int32_t(j) <= row_pos[n]) acc[n][t][i] += v;
          }
      }
    }

    {
      const uint32_t tid = afresh(threadIdx.x), lane = tid & 63, col = lane & 15, g = lane >> 4;
      // the four waves' sums meet in LDS, in wave order
      __syncthreads();  // the part before has been read
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        const float s = add_groups(l[n]);
        if (g == 0) {
          top[wave][16 * n + col] = m[n];
          mass[wave][16 * n + col] = s;
        }
#pragma unroll
        for (int t = 0; t < 8; t++) *reinterpret_cast<f32x4*>(&sums[wave][16 * n + col][16 * t + 4 * g]) = acc[n][t];
      }
      __syncthreads();
      const bool whole = cu.block == 0 && take == cu.blocks;
      float* const part = my_parts + (cu.block == 0 ? size_t(R) * kPartRow : 0);  // slot 1 begins an item, 0 goes on with one
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        const uint32_t r = 16 * n + tid / 16, d = (tid % 16) * 8;
        if (r < rows) {
          float mx = top[0][r];
          for (int i = 1; i < 4; i++) mx = fmaxf(mx, top[i][r]);
          float o[8] = {}, sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float f = rebase(top[i][r], mx);
            sum = fmaf(mass[i][r], f, sum);
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = fmaf(sums[i][r][d + e], f, o[e]);
          }
          if (whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] *= inv;
            store_out8<BF16_ROWS>(a.out, row_element(a, cu.q, head, cu.tile * R + r, a.out_stride) + d, o);
          } else {
            *reinterpret_cast<f32x4*>(part + r * kPageDim + d) = f32x4{o[0], o[1], o[2], o[3]};
            *reinterpret_cast<f32x4*>(part + r * kPageDim + d + 4) = f32x4{o[4], o[5], o[6], o[7]};
            if (d == 0) {
              part[R * kPageDim + r] = mx;
              part[R * kPageDim + R + r] = sum;
            }
          }
        }
      }
      if (!whole && cu.block == 0 && tid == 0)  // the item's last block is in the part (...) / per after this one
        begin_joint(a.joints[w], (whole_part - left + cu.blocks - 1) / per + 1, cu, R);
    }
    left -= take;
    if (left == 0 || !next_tile(a, cu, R)) break;
  }
}

// ---------------------------------------------------------------------------------------------
// Many rows: tiles of 32 rows (f32: 16) for each of the workgroup's waves, which share blocks of 64 positions
// of K and V through LDS: while one is multiplied the next (two, where LDS has room) are on their way.
//
// Bound by the matrix cores and the vector unit, which hardly work at the same time (a 32x32x16 product takes
// 36 cycles of a SIMD, of which 4 vector operations of its other wave hide behind it; each further one costs
// 2.8). bf16 rows: v_mfma_f32_32x32x16_bf16, transposed as above (a lane's 16 results of a score tile are the
// weights of 8 consecutive positions in two groups of 16, operand B of Out^T = V^T P^T as they stand): 32
// products and some 240 vector operations a block and wave. They go in tiles of 256 where there are so many:
// with 128 every CU pulls 32 KB from L2 for 2 MFLOP, and with all of them loading L2 gives some 50 B/ns each,
// less than the products take. f32 rows take three products for one, and 32 rows of their parts fill the
// registers of a SIMD: 16 rows by v_mfma_f32_16x16x32_bf16 (as in k_page_attn_rows) leave room for two waves
// on each (32 rows and one wave 1696 us, 16 and two 1455, for 8 chunks of up to 2048 over 4096 positions).
// Measured: those chunks, 32 over 8 heads, bf16 rows 680 to 705 us (e4m3 pages) and 650 to 675 (bf16), 850 to 920 TFLOP/s of
// 1225 that a large library product reaches; matrix cores busy 38% of the time, vector unit 50%. A chunk of
// 512 f32 rows over 2048 positions, 16 over 8 heads: 34.0 us, of which the plan takes 2, the first loads 3 to 4,
// the products of 8 blocks 20 and the join 5.
// LDS: K [64][128] with the 16-byte piece c of row r at place c ^ swap(r), V as it lies in memory
// ([4][128][16]), for 32-row waves with the two pieces of every second 8 dims exchanged: the lanes that a
// 16-byte read serves at once (0-3, 12-15, 20-23 and 24-27, and so on) find different banks. bf16 pages are
// loaded straight into it; e4m3 pages go through registers and are widened once for all rows (K with its
// scale, V's scale is put on the weights). A wave loads positions of one run of 16, which lie in one page.
// ---------------------------------------------------------------------------------------------
template <bool FP8, bool BF16_ROWS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void k_page_attn_tiles(AttnArgs a) {
  static_assert(BF16_ROWS || WAVES == 8, "f32 rows: 8 waves of 16");
  constexpr int NS = BF16_ROWS ? 1 : 3, WR = BF16_ROWS ? 32 : 16, R = WR * WAVES;
  constexpr int NJ = BF16_ROWS ? 8 : 4, NSUM = BF16_ROWS ? 16 : 8;  // fragments of a row of q; 4 dims of the sums each
  typedef typename std::conditional<BF16_ROWS, f32x16, f32x4>::type Acc;
  constexpr int PARTS = WAVES / 4, LOADS = 4 / PARTS;  // waves that share a run; 1 KB loads of K (and V) of each
  constexpr int STAGES = !FP8 && WAVES == 8 ? 3 : 2;  // LDS of one workgroup on a CU holds 3
  constexpr uint32_t TILE = kBlock * kPageDim * 2;  // bytes of K, and of V
  __shared__ __align__(16) uint8_t buf[STAGES][2 * TILE];
  __shared__ __align__(16) float vscale[2][FP8 ? kBlock : 4];
  __shared__ uint32_t foul[STAGES];
  __shared__ PlanShared sh;
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & (WR - 1), grp = lane / WR;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t w = part_index();
  Cursor cu;
  uint32_t per;
  uint32_t left = uniform(find_part(a, w, gridDim.x, R, sh, per, cu));
  cu = uniform(cu);
  per = uniform(per);
  a.whole_items = uniform(a.whole_items);
  if (tid == 0 && a.join) goes_on(a.joints[w], w, left, per, cu, R);
  if (left == 0) return;
  const uint32_t whole_part = left;
  const uint32_t ps_mask = (1u << a.p.page_shift) - 1;
  float* const my_parts = a.parts + size_t(w) * 2 * R * kPartRow;

  while (true) {
    const uint32_t take = min(cu.blocks - cu.block, left);
    const uint32_t limit = tile_limit(a, cu.q, cu.tile, R);
    const uint32_t first = cu.block * kBlock, last = a.whole_items ? limit : min((cu.block + take) * kBlock, limit);
    const uint32_t head = cu.head;
    // this wave's rows, and the positions that all of them (free_to) and some of them (end) attend
    const uint32_t wr0 = cu.tile * R + WR * wave;
    const uint32_t wrows = cu.q.rows > wr0 ? min(cu.q.rows - wr0, uint32_t(WR)) : 0;
    const int32_t free_to = row_position(a, cu.q, wr0);
    const uint32_t end = wrows ? row_limit(a, cu.q, wr0 + wrows - 1) : 0;
    const int32_t tile_free = row_position(a, cu.q, cu.tile * R);  // all rows of the tile attend up to it
    const uint32_t fresh = afresh(tid & 63), r = wr0 + (fresh & (WR - 1));
    const bool real = (fresh & (WR - 1)) < wrows;
    const int32_t row_pos = real ? row_position(a, cu.q, r) : -1;
    bf16x8 qf[NJ][NS];
    // sums of 4 dims each: n-th of them, and the first of its dims (of lane group g)
    constexpr int NACC = BF16_ROWS ? 4 : 8, PER = NSUM / NACC;
    Acc acc[NACC];
    auto dim_of = [](int n, uint32_t g) __attribute__((always_inline)) {
      return BF16_ROWS ? 32 * (n / 4) + 8 * (n % 4) + 4 * g : 16 * n + 4 * g;
    };
    auto sum_of = [&](int n) __attribute__((always_inline)) {
      const Acc& v = acc[n / PER];
      const int i = 4 * (n % PER);
      return f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    };
#pragma unroll
    for (int t = 0; t < NACC; t++) acc[t] = 0.f;
    float m = -INFINITY, l = 0.f;

    const int32_t* const table = a.p.table + size_t(cu.seq) * a.p.table_stride;
    // page of the 16 positions from x on, by a scalar load (the plan does not change while a call runs)
    auto page_at = [&](uint32_t x) __attribute__((always_inline)) {
      const uint32_t i = min(x >> a.p.page_shift, a.p.table_stride - 1);
      return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(table))[i];
    };
    auto is_page = [&](int32_t page) __attribute__((always_inline)) { return uint32_t(page) < a.p.n_pages; };
    const uint32_t run = wave / PARTS, part_of = wave % PARTS;
    u32x4 rk[FP8 ? 2 / PARTS : 1], rv[FP8 ? 2 / PARTS : 1];  // e4m3: 16 bytes of K rows, the 16 positions of V's dims
    uint32_t ke[FP8 ? 2 / PARTS : 1] = {}, ve = 0;
    // which place the 16-byte piece c of row p of K takes: c ^ swap(p), different for 16 rows that are read at once
    auto swap = [](uint32_t p) __attribute__((always_inline)) { return BF16_ROWS ? p & 15 : (p & 3) | (p >> 1 & 12); };
    // whether the two pieces of dim d of a run of V change places
    auto swap_v = [](uint32_t d) __attribute__((always_inline)) { return BF16_ROWS ? d >> 3 & 1 : 0; };
    // starts the loads of this wave's part of the block at x (a page that is not there is read as page 0,
    // and what comes of it is masked)
    auto fetch = [&](uint32_t x, uint32_t b, int32_t page) __attribute__((always_inline)) {
      const size_t row = page_row(a.p, is_page(page) ? page : 0, head, (x + 16 * run) & ps_mask);
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < 2 / PARTS; i++) {
          const uint32_t kr = 8 * (2 / PARTS * part_of + i) + (lane >> 3), d = 64 * (2 / PARTS * part_of + i) + lane;
          rk[i] = *reinterpret_cast<const u32x4*>(a.st.k + (row + kr) * kPageDim + 16 * (lane & 7));
          rv[i] = *reinterpret_cast<const u32x4*>(a.st.v + row * kPageDim + 16 * d);
          ke[i] = a.st.k_exp[row + kr];
        }
        ve = a.st.v_exp[row + (lane & 15)];
      } else {
        const uint32_t dst = lds_address(buf[b]) + run * 4096 + part_of * LOADS * 1024;
        const uint8_t *k = a.st.k + row * kPageDim * 2, *v = a.st.v + row * kPageDim * 2 + part_of * LOADS * 1024;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          const uint32_t kr = 4 * (part_of * LOADS + i) + (lane >> 4), c = (lane & 15) ^ swap(16 * run + kr);  // row, piece of the row
          dma16(dst + i * 1024, k + kr * kPageDim * 2 + c * 16);
        }
#pragma unroll
        for (int i = 0; i < LOADS; i++)
          dma16(dst + TILE + i * 1024, v + i * 1024 + (lane ^ swap_v(lane >> 1)) * 16);
      }
    };
    // e4m3: what fetch loaded, widened, into LDS
    auto widen = [&](uint32_t b) __attribute__((always_inline)) {
      if constexpr (FP8) {
#pragma unroll
        for (int i = 0; i < 2 / PARTS; i++) {
          const uint32_t kr = 8 * (2 / PARTS * part_of + i) + (lane >> 3), d = 64 * (2 / PARTS * part_of + i) + lane;
          uint8_t* k = buf[b] + run * 4096 + kr * 256;
          uint8_t* v = buf[b] + TILE + run * 4096 + d * 32;
          const float ks = __uint_as_float(ke[i] << 23);
#pragma unroll
          for (int e = 0; e < 2; e++) {
            *reinterpret_cast<bf16x8*>(k + (((2 * (lane & 7) + e) ^ swap(16 * run + kr)) * 16)) = fp8_bf16(rk[i][2 * e], rk[i][2 * e + 1], ks);
            *reinterpret_cast<bf16x8*>(v + ((e ^ swap_v(d)) * 16)) = fp8_bf16(rv[i][2 * e], rv[i][2 * e + 1], 1.f);
          }
        }
        if (part_of == 0 && lane < 16) vscale[b][16 * run + lane] = __uint_as_float(ve << 23);
      }
    };
    // V of positions 16 u + 8 (grp % 2) .., operand A of dims 32 t + col, or 16 t + col of positions 32 u + 8 grp ..
    auto v_part = [&](uint32_t b, int t, int u) __attribute__((always_inline)) {
      const uint32_t run = BF16_ROWS ? u : 2 * u + (grp >> 1), d = WR * t + col;
      return *reinterpret_cast<const bf16x8*>(buf[b] + TILE + run * 4096 + d * 32 + ((grp & 1) ^ swap_v(col)) * 16);
    };
    // V of the block in buffer b as every row may multiply it: zeros at positions that no row of the tile
    // attends, which may hold anything (0 x NaN is NaN), and where it is not finite at one that only some
    // attend (`foul`: those rows get it at the end). Each wave clears what it loaded.
    auto clear = [&](uint32_t x, uint32_t b, bool page) __attribute__((always_inline)) {
      // lane: 8 of the 16 positions at dims lane / 2, lane / 2 + 32, ... of its part
      const uint32_t base = x + 16 * run + 8 * ((lane & 1) ^ swap_v(lane >> 1)), ok = page && limit > base ? limit - base : 0;
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < LOADS; i++) {
        u32x4* v = reinterpret_cast<u32x4*>(buf[b] + TILE + run * 4096 + (part_of * LOADS + i) * 1024 + lane * 16);
        u32x4 u = *v;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          uint32_t z = u[k] & (ok >= 2u * k + 2 ? ~0u : ok > 2u * k ? 0xFFFFu : 0u);
          any |= clear_foul<false>(z);
          u[k] = z;
        }
        *v = u;
      }
      if (any) foul[b] = 1;
      // (scales behind the last position may be anything too)
      if constexpr (FP8)
        if (part_of == 0 && lane < 16 && !(page && x + 16 * run + lane < limit)) vscale[b][16 * run + lane] = 0.f;
    };
    uint32_t foul_from = kNowhere;  // the first block that `clear` cleared something of
    // this wave's rows against the block at x in buffer b; there: which of its four pages are; cleared: by `clear`
    auto multiply = [&](uint32_t x, uint32_t b, uint32_t there, bool cleared) __attribute__((always_inline)) {
      // Fragments come from LDS four at a time, a group ahead of the products that use them; the scheduling
      // barriers keep it so (left alone the compiler waits for every read right behind it).
      constexpr int NT = BF16_ROWS ? 2 : 4, PERS = BF16_ROWS ? 16 : 4;
      Acc s[NT];
      bf16x8 kf[2][4];
      // operand A's row `col` is position 32 t + kr of the block (f32 rows: kr of 32 (t / 2), 4 (t & 1) further)
      const uint32_t kr = BF16_ROWS ? 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3)
                                    : 8 * (col >> 2) + (col & 3);
      // fragment n of group o: bf16 rows score tile o / 2, dims 16 (4 (o & 1) + n) ..; f32 rows score tile
      // 2 (o / 2) + (n & 1), dims 32 (2 (o & 1) + n / 2) .., so that two sums take turns
      auto tile_of = [](int o, int n) __attribute__((always_inline)) { return BF16_ROWS ? o / 2 : 2 * (o / 2) + (n & 1); };
      auto dims_of = [](int o, int n) __attribute__((always_inline)) { return BF16_ROWS ? 4 * (o & 1) + n : 2 * (o & 1) + n / 2; };
      auto k_part = [&](int o, int n) __attribute__((always_inline)) {
        const int t = tile_of(o, n), j = dims_of(o, n);
        const uint32_t p = BF16_ROWS ? 32 * t + kr : 32 * (t / 2) + 4 * (t & 1) + kr;
        return *reinterpret_cast<const bf16x8*>(buf[b] + p * 256 + (((64 / WR * j + grp) ^ swap(p)) * 16));
      };
#pragma unroll
      for (int n = 0; n < 4; n++) kf[0][n] = k_part(0, n);
#pragma unroll
      for (int o = 0; o < 4; o++) {
        if (o < 3)
#pragma unroll
          for (int n = 0; n < 4; n++) kf[(o + 1) & 1][n] = k_part(o + 1, n);
        __builtin_amdgcn_sched_barrier(0);
        if (!(o & 1))
#pragma unroll
          for (int t = tile_of(o, 0); t <= tile_of(o, 3); t++) s[t] = 0.f;
        if constexpr (BF16_ROWS) {
#pragma unroll
          for (int n = 0; n < 4; n++)
            s[o / 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[o & 1][n], qf[dims_of(o, n)][0], s[o / 2], 0, 0, 0);
        } else {
#pragma unroll
          for (int n = 0; n < 4; n += 2)
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
              for (int e = n; e < n + 2; e++)
                s[tile_of(o, e)] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[o & 1][e], qf[dims_of(o, e)][i], s[tile_of(o, e)], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // score i of tile t: position in the block
      auto position = [&](int t, int i) __attribute__((always_inline)) {
        return BF16_ROWS ? 32 * t + 16 * (i >> 3) + 4 * ((i >> 2) & 1) + (i & 3) + 8 * grp
                         : 32 * (t / 2) + 4 * (t & 1) + i + 8 * grp;
      };
      const bool masked = int32_t(x + kBlock - 1) > free_to || there != 15;
      if (masked) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int i = 0; i < PERS; i++) {
            const uint32_t in = position(t, i);
            if (int32_t(x + in) > row_pos || !(there >> (in / 16) & 1)) s[t][i] = -INFINITY;
          }
      }
      float mx = s[0][0];
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < PERS; i++) mx = fmaxf(mx, s[t][i]);
      mx = fmaxf(m, (BF16_ROWS ? max_halves(mx) : max_groups(mx)) * a.c);
      if (__any(mx > m + kSlack)) {
        const float f = rebase(m, mx);
        l *= f;
#pragma unroll
        for (int t = 0; t < NACC; t++) acc[t] *= f;
        m = mx;
      }
      const float ref = m == -INFINITY ? 0.f : m;
      bf16x8 pf[2][NS];
      bf16x8 vf[2][4];
      // weights of positions 16 u + 8 grp .. (f32 rows: 32 u + 8 grp ..)
      auto weights = [&](int u, bf16x8 (&o)[NS]) __attribute__((always_inline)) {
        float e[8];
        f32x4 vs[2];
        if constexpr (FP8) {
          vs[0] = *reinterpret_cast<const f32x4*>(&vscale[b][(BF16_ROWS ? 16 : 32) * u + 8 * grp]);
          vs[1] = *reinterpret_cast<const f32x4*>(&vscale[b][(BF16_ROWS ? 16 : 32) * u + 8 * grp + 4]);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float z = BF16_ROWS ? s[u / 2][8 * (u & 1) + i] : s[2 * u + i / 4][i & 3];
          const float y = exp2_fast(fmaf(z, a.c, -ref));
          l += y;
          e[i] = y;
          if constexpr (FP8) e[i] *= vs[i / 4][i & 3];
        }
        split_bf16<NS>(e, o);
      };
      // group o: bf16 rows 16 positions and all dims, f32 rows 32 positions and half of them
      auto group = [&](int o, bf16x8 (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 4; t++) v[t] = BF16_ROWS ? v_part(b, t, o) : v_part(b, 4 * (o & 1) + t, o / 2);
      };
      group(0, vf[0]);
      weights(0, pf[0]);
#pragma unroll
      for (int o = 0; o < 4; o++) {
        if (o < 3) group(o + 1, vf[(o + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
        // products of these positions beside the next ones' weights
        if constexpr (BF16_ROWS) {
#pragma unroll
          for (int t = 0; t < 4; t++)
            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[o & 1][t], pf[o & 1][0], acc[t], 0, 0, 0);
          if (o < 3) weights(o + 1, pf[(o + 1) & 1]);
        } else {
#pragma unroll
          for (int i = 0; i < NS; i++)
#pragma unroll
            for (int t = 0; t < 4; t++)
              acc[4 * (o & 1) + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[o & 1][t], pf[o / 2][i], acc[4 * (o & 1) + t], 0, 0, 0);
          if (o == 0) weights(1, pf[1]);
        }
      }
      // (not only where this wave masks: `clear` is for the whole tile, whose first rows attend less)
      if (cleared && foul_from == kNowhere && uniform(foul[b]) != 0) foul_from = x;
    };
    // which of a block's four runs of 16 positions have a page
    auto pages_there = [&](uint32_t x) __attribute__((always_inline)) {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) bits |= uint32_t(is_page(page_at(x + 16 * i))) << i;
      return bits;
    };

    // Loads of q, then the first blocks', so that q is cut into its parts while those are under way (rows
    // behind the sequence's last are read as that one and come to nothing).
    constexpr int NQ = BF16_ROWS ? 1 : 2;
    const int32_t page0 = page_at(first + 16 * run), page1 = page_at(first + kBlock + 16 * run);
    u32x4 raw[NJ][NQ];
    const uint8_t* const q_row = a.q + (row_element(a, cu.q, head, min(r, cu.q.rows - 1), a.q_stride) + 8 * (fresh / WR)) * (BF16_ROWS ? 2 : 4);
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int i = 0; i < NQ; i++) raw[j][i] = *reinterpret_cast<const u32x4*>(q_row + (512 / WR) * (BF16_ROWS ? 2 : 4) * j + 16 * i);
    __syncthreads();  // the buffers' last readers are done
    // e4m3: block x is in LDS and x + 1 in registers when x is multiplied; bf16: STAGES - 1 are on their way
    if (first < last) {
      fetch(first, 0, page0);
      if (!FP8 && STAGES == 3 && first + kBlock < last) fetch(first + kBlock, 1, page1);
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      if constexpr (BF16_ROWS) {
        qf[j][0] = __builtin_bit_cast(bf16x8, raw[j][0]);
      } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __uint_as_float(raw[j][i / 4][i & 3]);
        split_bf16<NS>(x, qf[j]);
      }
    }
    if (first < last) {
      widen(0);
      if (FP8 && first + kBlock < last) fetch(first + kBlock, 1, page1);
      if (tid == 0) foul[0] = 0;
      constexpr uint32_t AHEAD = FP8 || STAGES == 3 ? 2 : 1;
      uint32_t b = 0, there = pages_there(first);
      int32_t page = page_at(first + AHEAD * kBlock + 16 * run);  // of this wave's part of the block fetched next
      for (uint32_t x = first; x < last; x += kBlock) {
        if constexpr (!FP8) {
          if (STAGES == 3 && x + kBlock < last) wait_dma<2 * LOADS>();
          else wait_dma<0>();
        }
        __syncthreads();  // block x is in LDS; the readers of the block before are done
        const bool cleared = int32_t(x + kBlock - 1) > tile_free || there != 15;
        if (cleared) {
          clear(x, b, there >> run & 1);
          __syncthreads();
        }
        const uint32_t b1 = b + 1 == STAGES ? 0 : b + 1, b2 = b1 + 1 == STAGES ? 0 : b1 + 1;
        if (FP8 && x + kBlock < last) widen(b1);
        if (x + AHEAD * kBlock < last) fetch(x + AHEAD * kBlock, STAGES == 3 ? b2 : b1, page);
        const uint32_t there_next = pages_there(x + kBlock);
        page = page_at(x + (AHEAD + 1) * kBlock + 16 * run);
        if (x < end) multiply(x, b, there, cleared);
        if (tid == 0) foul[b1] = 0;  // (its last readers are done; its next writers come after a barrier)
        there = there_next;
        b = b1;
      }
    }

    // what was cleared, to the rows that attend it: infinity and NaN stay what they are under a weight
    for (uint32_t j = foul_from; j < min(last, end); j++) {
      const int32_t page = page_at(j);
      if (!is_page(page)) continue;
      const size_t e = v_element(a.p, page, head, j & ps_mask);
#pragma unroll
      for (int n = 0; n < NSUM; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float v = v_value<FP8>(a.st.v, e + 16 * (dim_of(n, grp) + i));
          if (!(fabsf(v) < INFINITY) && int32_t(j) <= row_pos) acc[n / PER][4 * (n % PER) + i] += v;
        }
    }
    l = BF16_ROWS ? add_halves(l) : add_groups(l);
    const bool whole = cu.block == 0 && take == cu.blocks;
    {
      const uint32_t lane = afresh(tid & 63), col = lane & (WR - 1), grp = lane / WR;
      if (whole) {
        // through LDS (each wave in its own part of the buffers), so that rows are stored in one piece
        const float inv = l == 0.f ? 0.f : 1.f / l;
        constexpr uint32_t ROW = kPageDim * (BF16_ROWS ? 2 : 4), PIECES = ROW / 16;
        uint8_t* const rows_at = buf[0] + wave * WR * ROW;
        __syncthreads();  // the buffers' last readers are done
#pragma unroll
        for (int n = 0; n < NSUM; n++) {
          const f32x4 v = sum_of(n) * inv;
          const uint32_t d = dim_of(n, grp);
          if constexpr (BF16_ROWS) {
            uint2 u;
            u.x = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[0], v[1]}), bf16x2));
            u.y = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{v[2], v[3]}), bf16x2));
            *reinterpret_cast<uint2*>(rows_at + col * ROW + ((d / 8 ^ (col & 15)) * 16) + 8 * grp) = u;
          } else {
            *reinterpret_cast<f32x4*>(rows_at + col * ROW + ((d / 4 ^ col) * 16)) = v;
          }
        }
#pragma unroll
        for (uint32_t i = 0; i < WR * PIECES / 64; i++) {
          const uint32_t in = i * (64 / PIECES) + lane / PIECES, piece = lane % PIECES;
          if (in < wrows) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(rows_at + in * ROW + ((piece ^ (in & (PIECES - 1))) * 16));
            *reinterpret_cast<u32x4*>(a.out + row_element(a, cu.q, head, wr0 + in, a.out_stride) * (BF16_ROWS ? 2 : 4) + piece * 16) = v;
          }
        }
      } else {
        // sums as [32 rows][8 dims][half of them][row][4 dims]
        float* const part = my_parts + (cu.block == 0 ? size_t(R) * kPartRow : 0);
        if (wrows) {
          const uint32_t in = WR * wave + col;
#pragma unroll
          for (int n = 0; n < NSUM; n++) {
            const uint32_t d = dim_of(n, grp);
            *reinterpret_cast<f32x4*>(part + ((in / 32 * 16 + d / 8) * 64 + (d / 4 & 1) * 32 + in % 32) * 4) = sum_of(n);
          }
          if (grp == 0) {
            part[R * kPageDim + in] = m;
            part[R * kPageDim + R + in] = l;
          }
        }
        if (cu.block == 0 && tid == 0)
          begin_joint(a.joints[w], (whole_part - left + cu.blocks - 1) / per + 1, cu, R);
      }
    }
    left -= take;
    if (left == 0 || !next_tile(a, cu, R)) break;
  }
}

// ---------------------------------------------------------------------------------------------
// Joins the parts of the items that more than one workgroup attended: workgroup (w, y) the item whose
// first part is slot 1 of workgroup w, 16 of its rows at a time; the parts that follow it are the
// slots 0 of the workgroups after w. Small tiles' parts are rows of 128 sums; TILES: 32 rows side by side.
// Bound by its launch and two load latencies: 4 to 5 us (15 where 256 items of 256 rows are cut), as long as a
// thread has one or two rounds of parts. Where there would be more the workgroups of the parts share an item: a
// row over 31,180 positions, 16 over 1 heads (16 rows of 244 parts) 54 us with one workgroup, so 17; 20 rows over
// 20,000 (320 rows, 128 parts, f32 and bf16) 52 and 56 us, so 31 and 36; 64 x 8 items of two parts 108 us with
// one, 113 so. A workgroup runs on the XCD that wrote its part: with first parts at multiples of 8 and no such
// order all of it ran on one XCD, 13 us more.
// ---------------------------------------------------------------------------------------------
// The share of workgroup w + who, who in 0 .. n - 1, in joining the item that begins in workgroup w, joint j.
template <bool BF16_ROWS, bool TILES>
__device__ __forceinline__ void join_item(const AttnArgs& a, uint32_t R, const Joint& j, uint32_t w, uint32_t who) {
  const uint32_t tid = threadIdx.x;
  const uint32_t rows = j.rows, r0 = blockIdx.y * 16;
  if (r0 >= rows) return;
  const uint32_t here = min(rows - r0, 16u), most = joiners(j.n, rows, R);
  const uint32_t helpers = TILES ? most : min(most, here);
  if (who >= helpers) return;
  // Small tiles: rows r0 + who, + helpers, ..., `slots` of them side by side, a thread 8 dims after another; the
  // 16 / slots threads of a row's dims share its parts. Large ones: 16 rows after another, a thread each, and
  // `slots` times 8 dims; the threads that have the same share the parts.
  uint32_t slots = TILES ? 16 / helpers : 1;
  if (!TILES)
    while (slots * helpers < here - who) slots *= 2;
  const uint32_t u = tid / 16, share = 16 / slots, me = u / slots;
  const uint32_t d = (TILES ? who * slots + u % slots : tid % 16) * 8;
  const uint32_t r = r0 + (TILES ? tid % 16 : who + helpers * (u % slots));
  const uint32_t e0 = TILES ? ((r / 32 * 16 + d / 8) * 64 + r % 32) * 4 : r * kPageDim + d, e1 = e0 + (TILES ? 128 : 4);
  const size_t slot = size_t(R) * kPartRow;
  const bool real = r < r0 + here;
  float mx = -INFINITY, sum = 0.f, o[8] = {};
  if (real) {
    // a few parts at a time, all their loads together
    constexpr uint32_t AT = TILES ? 8 : 4;
    for (uint32_t i0 = me; i0 < j.n; i0 += AT * share) {
      float pm[AT], pl[AT];
      f32x4 x[AT], y[AT];
#pragma unroll
      for (uint32_t b = 0; b < AT; b++) {
        const uint32_t i = i0 + b * share;
        pm[b] = -INFINITY;
        pl[b] = 0.f;
        x[b] = y[b] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (i < j.n) {
          const float* part = a.parts + (2 * size_t(w + i) + (i == 0)) * slot;
          pm[b] = part[R * kPageDim + r];
          pl[b] = part[R * kPageDim + R + r];
          x[b] = *reinterpret_cast<const f32x4*>(part + e0);
          y[b] = *reinterpret_cast<const f32x4*>(part + e1);
        }
      }
      float top = mx;
#pragma unroll
      for (uint32_t b = 0; b < AT; b++) top = fmaxf(top, pm[b]);
      float f = rebase(mx, top);
      sum *= f;
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] *= f;
#pragma unroll
      for (uint32_t b = 0; b < AT; b++) {
        f = rebase(pm[b], top);
        sum = fmaf(pl[b], f, sum);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          o[e] = fmaf(x[b][e], f, o[e]);
          o[e + 4] = fmaf(y[b][e], f, o[e + 4]);
        }
      }
      mx = top;
    }
  }
  if (share > 1) {  // in order of the shares
    __shared__ __align__(16) float sums[256 * 8];
    __shared__ float top[256], mass[256];
    __syncthreads();  // the item before has been read
#pragma unroll
    for (int e = 0; e < 8; e++) sums[tid * 8 + e] = o[e];
    top[tid] = mx;
    mass[tid] = sum;
    __syncthreads();
    if (me != 0) return;
    float all = mx;
    for (uint32_t i = 1; i < share; i++) all = fmaxf(all, top[tid + i * slots * 16]);
    float f = rebase(mx, all);
    sum *= f;
#pragma unroll
    for (int e = 0; e < 8; e++) o[e] *= f;
    for (uint32_t i = 1; i < share; i++) {
      const uint32_t k = tid + i * slots * 16;
      f = rebase(top[k], all);
      sum = fmaf(mass[k], f, sum);
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = fmaf(sums[k * 8 + e], f, o[e]);
    }
  }
  if (!real) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 8; e++) o[e] *= inv;
  Seq q;
  q.row0 = j.row0;
  store_out8<BF16_ROWS>(a.out, row_element(a, q, j.head, j.first + r, a.out_stride) + d, o);
}

template <bool BF16_ROWS, bool TILES>
__global__ __launch_bounds__(256) void k_page_join(AttnArgs a, uint32_t R) {
  const uint32_t x = part_index();  // on the XCD that wrote the part
  const Joint j = a.joints[x];
  if (j.n) join_item<BF16_ROWS, TILES>(a, R, j, x, 0);
  if (j.from != kNowhere) join_item<BF16_ROWS, TILES>(a, R, a.joints[j.from], j.from, x - j.from);
}

constexpr uint32_t kWorkgroups = 512;  // two for each CU

// How calls are cut, by the most rows (new tokens x q heads of a KV head) a sequence can have: tiles of 16
// or 32 rows with K and V straight from memory, or tiles of 128 or (bf16 rows) 256 with them shared
// through LDS. One workgroup on a CU at 256 rows, and of f32 rows through LDS, else two.
struct Cut {
  uint32_t rows, workgroups;
};
Cut cut_of(uint64_t max_new, uint64_t group, bool bf16, uint64_t seq_heads) {
  const uint64_t most = max_new && max_new < 256 ? max_new * group : 256;
  // few rows: two workgroups for each CU where there are as many items (64 x 8 of 4.6k positions 108 us in a graph,
  // 114 with one), one where items are cut up all the same (16 x 8: 27.8 us with two, so 26.6)
  if (most <= 32) return {most <= 16 ? 16u : 32u, seq_heads >= kWorkgroups ? kWorkgroups : kWorkgroups / 2};
  if (!bf16) return {128, kWorkgroups / 2};
  return most <= 128 ? Cut{128, kWorkgroups} : Cut{256, kWorkgroups / 2};
}
// Up to so many positions in a table's row no item of few rows is cut, and no join follows (one row at 197
// positions 8.8 us in a graph, 10.2 with it; at 500 11.5 whole, so 10.2; f32 tiles of 128 rows at 250 17.9 and 14.5).
constexpr uint64_t kWholeItems = 256;

// n rows of `width` bytes, `stride` (at least width) bytes apart; addresses in more than 64 bits, as the last
// row's may be.
struct RowSpan {
  __int128 base, stride, width, n;
  __int128 end() const { return base + (n - 1) * stride + width; }
  // the first row that ends behind `at`
  __int128 behind(__int128 at) const { return at < base + width ? 0 : (at - base - width) / stride + 1; }
  __int128 row(__int128 i) const { return base + i * stride; }
};
// Whether a row of either shares memory with one of the other; rows may lie between each other's.
bool overlap(const RowSpan& a, const RowSpan& b) {
  if (a.end() <= b.base || b.end() <= a.base) return false;
  if (a.stride == b.stride && a.n == b.n) {  // every row of `hi` lies to the rows of `lo` as its first does
    const RowSpan &lo = a.base <= b.base ? a : b, &hi = a.base <= b.base ? b : a;
    return lo.row(lo.behind(hi.base)) < hi.base + hi.width;
  }
  for (__int128 i = a.behind(b.base), j = 0; i < a.n && j < b.n;) {
    if (b.row(j) + b.width <= a.row(i)) j = b.behind(a.row(i));
    else if (a.row(i) + a.width <= b.row(j)) i = a.behind(b.row(j));
    else return true;
  }
  return false;
}

}  // namespace
}  // namespace qe

extern "C" {

uint64_t qe_op_page_attention_work_bytes(uint64_t n_heads, uint64_t n_kv_heads, uint64_t max_new) {
  if (!n_kv_heads || !n_heads || n_heads % n_kv_heads) return 0;
  uint64_t rows = 0;  // of all workgroups
  for (bool bf16 : {false, true}) {
    const qe::Cut c = qe::cut_of(max_new, n_heads / n_kv_heads, bf16, ~0ull);
    rows = rows > uint64_t(c.rows) * c.workgroups ? rows : uint64_t(c.rows) * c.workgroups;
  }
  return rows * 2 * qe::kPartRow * 4 + qe::kWorkgroups * sizeof(qe::Joint);
}

int qe_op_page_attention(const qe_pages* pages, const void* q, void* out, uint64_t n_rows, uint64_t n_heads,
                         uint64_t q_stride, uint64_t out_stride, uint64_t max_new, int dtype, void* work,
                         uint64_t work_bytes, void* stream) {
  qe::AttnArgs a{};
  if (int rc = qe::check_pages(pages, &a.p, &a.st)) return rc;
  if (dtype != QE_KV_F32 && dtype != QE_KV_BF16) return qe::set_error(QE_ERR_ARG, "rows are QE_KV_F32 or QE_KV_BF16");
  if (n_heads == 0 || n_heads % a.p.n_kv || n_heads > 65536)
    return qe::set_error(QE_ERR_ARG, "n_heads must be a multiple of n_kv_heads, at most 65536");
  if (n_rows == 0) return QE_OK;
  if (!q || !out || !work) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_rows > 0x7FFFFFFFull / n_heads) return qe::set_error(QE_ERR_ARG, "need n_rows * n_heads < 2^31");
  const uint64_t el = dtype == QE_KV_F32 ? 4 : 2;
  for (uint64_t stride : {q_stride, out_stride})
    if (stride < n_heads * qe::kPageDim || stride > 0xFFFFFFFFull || stride * el % 16)
      return qe::set_error(QE_ERR_ARG, "row strides must be at least n_heads * 128 elements and multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(work)) % 16)
    return qe::set_error(QE_ERR_ARG, "q, out and work must be 16-byte aligned");
  if (work_bytes < qe_op_page_attention_work_bytes(n_heads, a.p.n_kv, max_new))
    return qe::set_error(QE_ERR_ARG, "work holds %llu bytes, fewer than qe_op_page_attention_work_bytes gives",
                         (unsigned long long)work_bytes);
  const bool fp8 = pages->kv_dtype == QE_KV_FP8;
  auto span = [](const void* p, uint64_t stride, uint64_t width, uint64_t n) {
    return qe::RowSpan{__int128(reinterpret_cast<uintptr_t>(p)), __int128(stride), __int128(width), __int128(n)};
  };
  const qe::RowSpan rows = span(out, out_stride * el, n_heads * qe::kPageDim * el, n_rows);
  const uint64_t page_rows = pages->n_pages * pages->n_kv_heads, kv_bytes = pages->page_size * qe::kPageDim * (fp8 ? 1 : 2);
  auto over = [&](const void* p, uint64_t bytes) { return qe::overlap(rows, span(p, bytes, bytes, page_rows)); };
  if (qe::overlap(rows, span(q, q_stride * el, n_heads * qe::kPageDim * el, n_rows)) || over(pages->k, kv_bytes) ||
      over(pages->v, kv_bytes) || (fp8 && (over(pages->k_exp, pages->page_size) || over(pages->v_exp, pages->page_size))))
    return qe::set_error(QE_ERR_ARG, "out must not overlap q or the pages");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == QE_KV_BF16;
  a.q = static_cast<const uint8_t*>(q);
  a.out = static_cast<uint8_t*>(out);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.n_rows = uint32_t(n_rows);
  a.group = uint32_t(n_heads / a.p.n_kv);
  // shift = ceil(log2 group), magic = ceil(2^(31 + shift) / group): exact below 2^31
  while ((1ull << a.group_shift) < a.group) a.group_shift++;
  a.group_magic = uint32_t(((1ull << (31 + a.group_shift)) + a.group - 1) / a.group);
  a.c = 1.44269504f / sqrtf(float(qe::kPageDim));
  a.joints = static_cast<qe::Joint*>(work);
  a.parts = reinterpret_cast<float*>(a.joints + qe::kWorkgroups);
  // (fewer rows than max_new says need no more than the work that was asked for)
  const uint64_t bound = max_new && max_new < n_rows ? max_new : n_rows;
  const qe::Cut c = qe::cut_of(bound, a.group, bf16, uint64_t(a.p.n_seqs) * a.p.n_kv);
  const uint32_t R = c.rows, grid = c.workgroups;
  a.whole_items = R <= 32 && pages->table_stride * pages->page_size <= qe::kWholeItems;
  a.join = !a.whole_items;
  auto go = [&](auto* kern) { kern<<<grid, R == 256 || (R == 128 && !bf16) ? 512 : 256, 0, st>>>(a); };
  if (R == 256) {
    go(fp8 ? qe::k_page_attn_tiles<true, true, 8> : qe::k_page_attn_tiles<false, true, 8>);
  } else if (R == 128) {
    if (fp8) go(bf16 ? qe::k_page_attn_tiles<true, true, 4> : qe::k_page_attn_tiles<true, false, 8>);
    else go(bf16 ? qe::k_page_attn_tiles<false, true, 4> : qe::k_page_attn_tiles<false, false, 8>);
  } else if (R == 32) {
    if (fp8) go(bf16 ? qe::k_page_attn_rows<true, true, 2> : qe::k_page_attn_rows<true, false, 2>);
    else go(bf16 ? qe::k_page_attn_rows<false, true, 2> : qe::k_page_attn_rows<false, false, 2>);
  } else {
    if (fp8) go(bf16 ? qe::k_page_attn_rows<true, true, 1> : qe::k_page_attn_rows<true, false, 1>);
    else go(bf16 ? qe::k_page_attn_rows<false, true, 1> : qe::k_page_attn_rows<false, false, 1>);
  }
  if (a.join) {
    const dim3 join(grid, R / 16);
    auto join_by = [&](auto* kern) { kern<<<join, 256, 0, st>>>(a, R); };
    if (R >= 128) join_by(bf16 ? qe::k_page_join<true, true> : qe::k_page_join<false, true>);
    else join_by(bf16 ? qe::k_page_join<true, false> : qe::k_page_join<false, false>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "page attention launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
