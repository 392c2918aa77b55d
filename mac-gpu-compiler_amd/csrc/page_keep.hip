// A paged cache of bounded size: which positions each KV head keeps (qe_op_page_keep), and the move of
// kept rows to the front (qe_op_page_move). No reference counterpart.
#include "pages.h"

#include "device_common.h"
#include "status.h"

#include <type_traits>

namespace qe {
namespace {

// ---- the choice ----
// A float as a whole number that orders as it does: NaN below all, -0 as 0. What is always kept is above them, what
// is not there below.
constexpr uint32_t kAlways = 0xFFFFFFFFu, kNever = 0;
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 1;
  const uint32_t u = x == 0.f ? 0 : __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr uint32_t kKeepThreads = 1024;

struct KeepArgs {
  const float* mass;
  const int32_t* lens;
  int32_t *kept, *count;
  uint64_t mass_stride, kept_stride;
  uint32_t n_kv, keep, sinks, recent;
};

// A wave has a contiguous part of the row, in groups of 256 positions, a lane 4 consecutive ones of each.
constexpr uint32_t kGroup = 256, kWaves = kKeepThreads / 64;
constexpr uint32_t kDigits = 2048, kCopies = 4;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// The sum of the waves' values before `wave`.
__device__ __forceinline__ uint32_t sum_below(const uint32_t* waves, uint32_t wave) {
  const uint32_t lane = threadIdx.x & 63, v = waves[lane < kWaves ? lane : 0];
  return from_lane(wave_scan(lane < wave ? v : 0), 63);
}

// A workgroup for each sequence and KV head. The value that the `need`-th largest of the middle has is found by its
// digits from the top, 11, 11 and 10 bits: the values that agree so far are counted by their next digit in LDS (the
// first time in four copies, since masses share few exponents), and the digit is where the count from above
// reaches `need`. Then everything above that value is kept, and of what equals it the first.
// Bound by latency, not by the 4 bytes a position: a chain of some ten barriers, and a few operations a value on each CU.
// 8 rows of 4500 values to 1024 7.8 us; 256 rows of up to 32,000 to 4096 19.5 (the row 6, the digits 8, the places 5); 8
// of up to 43,632 23. A row that is read again for each pass: 8 of up to 70,000 51.
// GROUPS: of a wave, that are held in registers (0: the row is read again for each pass).
template <int GROUPS>
__global__ __launch_bounds__(kKeepThreads) void k_page_keep(KeepArgs a) {
  constexpr bool REGS = GROUPS > 0;
  __shared__ uint32_t digits[(kCopies + 2) * kDigits];
  __shared__ uint32_t waves[3][kWaves], found[3][2], above[kWaves], equal[kWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t s = blockIdx.x / a.n_kv, h = blockIdx.x - s * a.n_kv;
  const uint32_t len = uint32_t(min(int64_t(max(a.lens[s], 0)), int64_t(a.mass_stride)));
  const uint32_t keep = min(len, a.keep), sinks = min(a.sinks, keep), recent = min(a.recent, keep - sinks);
  const uint32_t from = sinks, to = len - recent, want = keep - sinks - recent;  // `want` of from .. to - 1
  const float* mass = a.mass + uint64_t(blockIdx.x) * a.mass_stride;
  int32_t* kept = a.kept + uint64_t(blockIdx.x) * a.kept_stride;
  for (uint32_t i = keep + tid; i < a.keep; i += kKeepThreads) kept[i] = -1;
  if (h == 0 && tid == 0) a.count[s] = int32_t(keep);
  if (want == to - from) {  // all of them
    for (uint32_t j = tid; j < len; j += kKeepThreads) kept[j] = int32_t(j);
    return;
  }
  const uint32_t groups = (len + kWaves * kGroup - 1) / (kWaves * kGroup), j0 = wave * groups * kGroup + 4 * lane;
  auto load = [&](uint32_t g, uint32_t (&key)[4]) __attribute__((always_inline)) {
    const uint32_t j = j0 + g * kGroup;
    if (j + 3 < len) {
      const f32x4u x = *reinterpret_cast<const f32x4u*>(mass + j);
#pragma unroll
      for (int e = 0; e < 4; e++) key[e] = order_of(x[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) key[e] = j + e < len ? order_of(mass[j + e]) : kNever;
    }
    if (j < from || j + 3 >= to)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (j + e < len && (j + e < from || j + e >= to)) key[e] = kAlways;
  };
  uint32_t keys[REGS ? GROUPS : 1][4];
  if constexpr (REGS) {
#pragma unroll
    for (uint32_t g = 0; g < GROUPS; g++)
      if (g < groups) load(g, keys[g]);
  }
  // f(first position, keys) of each group
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (REGS) {
#pragma unroll
      for (uint32_t g = 0; g < GROUPS; g++)
        if (g < groups) f(j0 + g * kGroup, keys[g]);
    } else {
      for (uint32_t g = 0; g < groups; g++) {
        load(g, keys[0]);
        f(j0 + g * kGroup, keys[0]);
      }
    }
  };
  uint32_t prefix = 0, need = want;  // the digits so far; how many of the values that have them are kept
  if (want) {
    for (uint32_t i = tid; i < (kCopies + 2) * kDigits; i += kKeepThreads) digits[i] = 0;
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, high = pass == 1 ? 21 : 10;  // of the digit; of those before
      const uint32_t n = pass == 2 ? 1024 : 2048;
      uint32_t* const bins = digits + (pass == 0 ? (wave % kCopies) * kDigits : (kCopies + pass - 1) * kDigits);
      each([&](uint32_t j, const uint32_t (&key)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (pass == 0 ? key[e] - 1 < kAlways - 1 : key[e] >> high == prefix >> high)
            atomicAdd(&bins[key[e] >> shift & (n - 1)], 1u);
      });
      __syncthreads();
      // from above: thread t has the digits n - 1 - 2 t and n - 2 - 2 t
      uint32_t c[2] = {};
      if (2 * tid < n)
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (uint32_t k = 0; k < (pass == 0 ? kCopies : 1); k++)
            c[i] += digits[(pass == 0 ? k : kCopies + pass - 1) * kDigits + n - 1 - 2 * tid - i];
      uint32_t upto = wave_scan(c[0] + c[1]);
      if (lane == 63) waves[pass][wave] = upto;
      __syncthreads();
      upto += sum_below(waves[pass], wave);
      const uint32_t before = upto - c[0] - c[1];
      if (before < need && upto >= need) {
        const bool second = before + c[0] < need;
        found[pass][0] = n - 1 - 2 * tid - second;
        found[pass][1] = before + (second ? c[0] : 0);
      }
      __syncthreads();
      prefix |= found[pass][0] << shift;
      need -= found[pass][1];
    }
  }
  else prefix = kAlways - 1;
  // which are kept: what is above the value, and of what equals it the first
  uint32_t n_above = 0, n_equal = 0;
  each([&](uint32_t, const uint32_t (&key)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      n_above += __builtin_popcountll(__ballot(key[e] > prefix));
      n_equal += __builtin_popcountll(__ballot(key[e] == prefix));
    }
  });
  if (lane == 0) {
    above[wave] = n_above;
    equal[wave] = n_equal;
  }
  __syncthreads();
  uint32_t ties = sum_below(equal, wave), at = sum_below(above, wave) + min(ties, need);  // equal, and kept, before this wave's positions
  // positions go through LDS, where the counts were, if they fit: stored in order then
  int32_t* const stage = reinterpret_cast<int32_t*>(digits);
  const bool staged = keep <= (kCopies + 2) * kDigits;
  // (rank of a lane's position among those of a group: the lanes before it, then its own)
  auto below = [&](uint64_t m) { return __builtin_amdgcn_mbcnt_hi(uint32_t(m >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(m), 0)); };
  auto places = [&](int32_t* to) __attribute__((always_inline)) {
    each([&](uint32_t j, const uint32_t (&key)[4]) __attribute__((always_inline)) {
      bool in[4];
      uint64_t m[4];
#pragma unroll
      for (int e = 0; e < 4; e++) m[e] = __ballot(in[e] = key[e] > prefix);
      uint64_t tie[4];
#pragma unroll
      for (int e = 0; e < 4; e++) tie[e] = __ballot(key[e] == prefix);
      if (tie[0] | tie[1] | tie[2] | tie[3]) {
        uint32_t rank = ties;
#pragma unroll
        for (int e = 0; e < 4; e++) rank += below(tie[e]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          ties += __builtin_popcountll(tie[e]);
          if (key[e] == prefix) in[e] = rank++ < need;
          m[e] = __ballot(in[e]);
        }
      }
      uint32_t place = at;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        place += below(m[e]);
        at += __builtin_popcountll(m[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (in[e]) to[place++] = int32_t(j + e);
    });
  };
  if (staged) places(stage);
  else places(kept);
  if (!staged) return;
  __syncthreads();
  for (uint32_t i = tid; i < keep; i += kKeepThreads) kept[i] = stage[i];
}

// ---- the move ----
struct MoveArgs {
  PagePlan p;
  PageStore st;
  const int32_t *src, *count, *first;
  float* mass;
  uint64_t mass_stride;
  uint32_t src_heads, src_stride;
};

constexpr uint32_t kMoveThreads = 256, kNoSlot = 0xFFFFFFFFu;

// The moves of a sequence and KV head. Slots are row indexes in the pages (below 2^32 - 1, as the host checks).
struct Moves {
  const int32_t* src;
  int64_t first;
  uint32_t s, head, count;
};
__device__ __forceinline__ Moves moves_of(const MoveArgs& a, uint32_t item) {
  Moves m;
  m.s = item / a.p.n_kv;
  m.head = item - m.s * a.p.n_kv;
  m.first = a.first ? a.first[m.s] : 0;
  m.count = uint32_t(min(int64_t(max(a.count[m.s], 0)), int64_t(a.src_stride)));
  m.src = a.src + (uint64_t(m.s) * a.src_heads + (a.src_heads == 1 ? 0 : m.head)) * a.src_stride;
  return m;
}
__device__ __forceinline__ uint32_t slot_of(const MoveArgs& a, const Moves& m, int64_t pos) {
  if (pos < 0 || pos >= capacity_of(a.p)) return kNoSlot;
  const int32_t page = page_of(a.p, m.s, pos);
  return page < 0 ? kNoSlot : uint32_t(page_row(a.p, page, m.head, uint32_t(pos) & ((1u << a.p.page_shift) - 1)));
}
// Where row i comes from and goes to; neither, unless both are there and differ.
struct Move {
  uint32_t from, to;
};
__device__ __forceinline__ Move move_of(const MoveArgs& a, const Moves& m, uint32_t i) {
  Move v{kNoSlot, kNoSlot};
  if (i >= m.count) return v;
  const int32_t at = m.src[i];
  if (at < 0 || at == int32_t(i)) return v;
  v.from = slot_of(a, m, m.first + at);
  v.to = slot_of(a, m, m.first + i);
  if (v.from == kNoSlot || v.to == kNoSlot) v.from = v.to = kNoSlot;
  return v;
}
// The wave's loads have arrived: no wave of the workgroup writes before all of them, behind a barrier, are done.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }

template <bool FP8>
struct Element {
  typedef typename std::conditional<FP8, uint8_t, uint16_t>::type type;
};
// V of row `slot`, dim d, in elements
__device__ __forceinline__ size_t v_at(uint32_t slot, uint32_t d) {
  return size_t(slot & ~(kPageRun - 1)) * kPageDim + d * kPageRun + (slot & (kPageRun - 1));
}

// mass of the rows moved, and 0 behind them; the exponents. Row i is thread i % 256's.
template <bool FP8, int N>
__device__ __forceinline__ void move_rest(const MoveArgs& a, const Moves& m, uint32_t item) {
  const uint32_t tid = threadIdx.x;
  float* const mass = a.mass ? a.mass + uint64_t(item) * a.mass_stride : nullptr;
  if (!FP8 && !mass) return;
  for (uint32_t i0 = 0; i0 < m.count; i0 += kMoveThreads * N) {
    uint32_t to[N], ke[N], ve[N];
    int64_t place[N];
    float v[N];
#pragma unroll
    for (int n = 0; n < N; n++) {
      const uint32_t i = i0 + n * kMoveThreads + tid;
      to[n] = kNoSlot;
      place[n] = -1;
      ke[n] = ve[n] = 0;
      v[n] = 0.f;
      if (FP8) {
        const Move w = move_of(a, m, i);
        to[n] = w.to;
        if (w.from != kNoSlot) {
          ke[n] = a.st.k_exp[w.from];
          ve[n] = a.st.v_exp[w.from];
        }
      }
      if (mass && i < m.count) {
        const int32_t at = m.src[i];
        const int64_t x = m.first + at, y = m.first + i;
        if (at >= 0 && x >= 0 && y >= 0 && x < int64_t(a.mass_stride) && y < int64_t(a.mass_stride)) {
          place[n] = y;
          v[n] = mass[x];
        }
      }
    }
    wait_loads();
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) {
      if (FP8 && to[n] != kNoSlot) {
        a.st.k_exp[to[n]] = uint8_t(ke[n]);
        a.st.v_exp[to[n]] = uint8_t(ve[n]);
      }
      if (place[n] >= 0) mass[place[n]] = v[n];
    }
  }
  if (mass) {
    __syncthreads();
    const int64_t end = min(int64_t(a.p.lens[m.s]), int64_t(a.mass_stride));
    for (int64_t j = max(m.first + m.count, int64_t(0)) + tid; j < end; j += kMoveThreads) mass[j] = 0.f;
  }
}

// Up to 64 rows of a sequence and KV head, as a path has them: a workgroup reads all of them and writes them.
// Bound by its chain: count, src, table, rows. 48 sequences of 8 KV heads, paths of a few rows, e4m3: 5.1 us.
constexpr uint32_t kFewMoves = 64;
template <bool FP8>
__global__ __launch_bounds__(kMoveThreads) void k_page_move_few(MoveArgs a) {
  typedef typename Element<FP8>::type T;
  constexpr uint32_t ROW = kPageDim * sizeof(T), PIECES = ROW / 16, ROWS = kMoveThreads / PIECES, NK = kFewMoves / ROWS;
  constexpr uint32_t NV = kFewMoves * kPageDim / kMoveThreads;
  __shared__ Move moves[kFewMoves];
  const uint32_t tid = threadIdx.x, item = blockIdx.x;
  const Moves m = moves_of(a, item);
  if (tid < kFewMoves) moves[tid] = move_of(a, m, tid);
  __syncthreads();
  u32x4_t k[NK];
#pragma unroll
  for (uint32_t n = 0; n < NK; n++) {
    const uint32_t i = n * ROWS + tid / PIECES;
    if (n * ROWS < m.count && moves[i].from != kNoSlot)
      k[n] = *reinterpret_cast<const u32x4_t*>(a.st.k + size_t(moves[i].from) * ROW + (tid % PIECES) * 16);
  }
  T* const pages = reinterpret_cast<T*>(a.st.v);
  T v[NV];
#pragma unroll
  for (uint32_t n = 0; n < NV; n++) {
    const uint32_t i = 2 * n + tid / kPageDim;
    if (2 * n < m.count && moves[i].from != kNoSlot) v[n] = pages[v_at(moves[i].from, tid % kPageDim)];
  }
  wait_loads();
  __syncthreads();
#pragma unroll
  for (uint32_t n = 0; n < NK; n++) {
    const uint32_t i = n * ROWS + tid / PIECES;
    if (n * ROWS < m.count && moves[i].from != kNoSlot)
      *reinterpret_cast<u32x4_t*>(a.st.k + size_t(moves[i].to) * ROW + (tid % PIECES) * 16) = k[n];
  }
#pragma unroll
  for (uint32_t n = 0; n < NV; n++) {
    const uint32_t i = 2 * n + tid / kPageDim;
    if (2 * n < m.count && moves[i].from != kNoSlot) pages[v_at(moves[i].to, tid % kPageDim)] = v[n];
  }
  move_rest<FP8, 1>(a, m, item);
}

// Many rows. Dims do not meet, so a sequence and KV head is shared by workgroups that have 64 bytes of each K row, or
// 8 dims of V; one has what there is one of for a row. Rows ascend and only ever move to the front, so what a chunk
// of rows writes no later chunk reads: within one everything is read before anything is written, and the next one's
// reads are under way while it is written. Where the rows lie is found for 2048 of them at a time (src, then the
// table: two load latencies, which a chunk would otherwise wait for). V is gathered 2 bytes (1 of e4m3) at a time and
// stored in whole runs of 16 positions. Bound by those gathers: 6 sequences of up to 8192 positions, 8 KV heads, bf16, to
// 2048 with their mass, 40 us, e4m3 25 (K alone 18, V alone 36; 16 dims of V a workgroup 54 in all, 4 dims 51). Runs staged whole in LDS took 90. Workgroup (part, item): the parts of an item share
// an XCD where the items are a multiple of 8.
constexpr uint32_t kPlan = 2048, kSliceV = 8;
template <bool FP8>
constexpr uint32_t move_parts() { return kPageDim * (FP8 ? 1 : 2) / 64 + kPageDim / kSliceV + 1; }

template <bool FP8>
__global__ __launch_bounds__(kMoveThreads) void k_page_move(MoveArgs a, uint32_t items) {
  typedef typename Element<FP8>::type T;
  constexpr uint32_t ROW = kPageDim * sizeof(T), K_PARTS = ROW / 64, V_PARTS = kPageDim / kSliceV;
  __shared__ uint32_t from[kPlan], to[kPlan];
  const uint32_t tid = threadIdx.x, part = blockIdx.x / items, item = blockIdx.x - part * items;
  const Moves m = moves_of(a, item);
  // Rows p0 - lead .. of the plan, in chunks that are read one ahead.
  auto run = [&](uint32_t lead, uint32_t chunk, auto&& read, auto&& write, auto& v0, auto& v1) __attribute__((always_inline)) {
    const uint32_t total = m.count + lead;
    for (uint32_t p0 = 0; p0 < total; p0 += kPlan) {
#pragma unroll
      for (uint32_t n = 0; n < kPlan / kMoveThreads; n++) {
        const uint32_t p = n * kMoveThreads + tid;
        const Move w = p0 + p >= lead ? move_of(a, m, p0 + p - lead) : Move{kNoSlot, kNoSlot};
        from[p] = w.from;
        to[p] = w.to;
      }
      __syncthreads();
      const uint32_t n = (min(total - p0, kPlan) + chunk - 1) / chunk;
      read(v0, 0);
      for (uint32_t c = 0; c < n; c += 2) {
        wait_loads();
        __syncthreads();  // chunk c has been read
        if (c + 1 < n) read(v1, (c + 1) * chunk);
        write(v0, c * chunk);
        if (c + 1 == n) break;
        wait_loads();
        __syncthreads();
        if (c + 2 < n) read(v0, (c + 2) * chunk);
        write(v1, (c + 1) * chunk);
      }
      __syncthreads();  // the plan has been read
    }
  };
  if (part < K_PARTS) {
    constexpr uint32_t ROWS = kMoveThreads / 4, N = 4;
    uint8_t* const pages = a.st.k + part * 64 + (tid & 3) * 16;
    struct Rows {
      u32x4_t v[N];
    } v0, v1;
    run(0, ROWS * N, [&](Rows& r, uint32_t at) __attribute__((always_inline)) {
#pragma unroll
          for (uint32_t n = 0; n < N; n++) {
            const uint32_t x = from[at + n * ROWS + tid / 4];
            if (x != kNoSlot) r.v[n] = *reinterpret_cast<const u32x4_t*>(pages + size_t(x) * ROW);
          }
        },
        [&](const Rows& r, uint32_t at) __attribute__((always_inline)) {
#pragma unroll
          for (uint32_t n = 0; n < N; n++) {
            const uint32_t x = to[at + n * ROWS + tid / 4];
            if (x != kNoSlot) *reinterpret_cast<u32x4_t*>(pages + size_t(x) * ROW) = r.v[n];
          }
        }, v0, v1);
  } else if (part < K_PARTS + V_PARTS) {
    // runs of 16 positions as they lie in the pages: a thread has a dim of a run
    const uint32_t at = tid / kSliceV * kPageRun, d = (part - K_PARTS) * kSliceV + tid % kSliceV;
    T* const pages = reinterpret_cast<T*>(a.st.v);
    struct Run {
      T v[kPageRun];
    } v0, v1;
    run(uint32_t(m.first) & (kPageRun - 1),  // positions of the first run before the rows
        kMoveThreads / kSliceV * kPageRun,
        [&](Run& r, uint32_t p) __attribute__((always_inline)) {
#pragma unroll
          for (uint32_t k = 0; k < kPageRun; k++) {
            const uint32_t x = from[p + at + k];
            r.v[k] = pages[v_at(x != kNoSlot ? x : 0, d)];
          }
        },
        [&](const Run& r, uint32_t p) __attribute__((always_inline)) {
          uint32_t have = 0, first = 0;
#pragma unroll
          for (uint32_t k = 0; k < kPageRun; k++) {
            const uint32_t x = to[p + at + k];
            if (x != kNoSlot) {
              have |= 1u << k;
              first = x & ~(kPageRun - 1);
            }
          }
          if (!have) return;
          T* const o = pages + v_at(first, d);
          if (have == (1u << kPageRun) - 1) {
            u32x4_t w[kPageRun * sizeof(T) / 16];
#pragma unroll
            for (uint32_t i = 0; i < kPageRun * sizeof(T) / 4; i++) {
              w[i / 4][i % 4] = 0;
#pragma unroll
              for (uint32_t e = 0; e < 4 / sizeof(T); e++) w[i / 4][i % 4] |= uint32_t(r.v[i * (4 / sizeof(T)) + e]) << (8 * sizeof(T) * e);
            }
#pragma unroll
            for (uint32_t i = 0; i < kPageRun * sizeof(T) / 16; i++) reinterpret_cast<u32x4_t*>(o)[i] = w[i];
          } else {
#pragma unroll
            for (uint32_t k = 0; k < kPageRun; k++)
              if (have >> k & 1) o[k] = r.v[k];
          }
        }, v0, v1);
  } else {
    move_rest<FP8, 8>(a, m, item);
  }
}

}  // namespace
}  // namespace qe

extern "C" {

int qe_op_page_keep(const float* mass, uint64_t mass_stride, const int32_t* lens, uint64_t n_seqs, uint64_t n_kv_heads,
                    uint64_t keep, uint64_t sinks, uint64_t recent, int32_t* kept, uint64_t kept_stride,
                    int32_t* count, void* stream) {
  if (!mass || !lens || !kept || !count) return qe::set_error(QE_ERR_ARG, "null argument");
  if (n_kv_heads == 0 || n_kv_heads > 1024) return qe::set_error(QE_ERR_ARG, "n_kv_heads must be 1..1024");
  if (n_seqs == 0 || n_seqs > 65536 || n_seqs * n_kv_heads >= 1u << 22)
    return qe::set_error(QE_ERR_ARG, "n_seqs must be 1..65536, and n_seqs * n_kv_heads below 2^22");
  if (mass_stride == 0 || mass_stride > 0x7FFFFFFFull || kept_stride > 0x7FFFFFFFull)
    return qe::set_error(QE_ERR_ARG, "need mass_stride > 0, and both strides below 2^31");
  if (keep == 0 || keep > kept_stride) return qe::set_error(QE_ERR_ARG, "keep must be 1..kept_stride");
  if (sinks > keep || recent > keep - sinks) return qe::set_error(QE_ERR_ARG, "sinks + recent must be at most keep");
  if ((reinterpret_cast<uintptr_t>(mass) | reinterpret_cast<uintptr_t>(lens) | reinterpret_cast<uintptr_t>(kept) |
       reinterpret_cast<uintptr_t>(count)) % 4)
    return qe::set_error(QE_ERR_ARG, "mass, lens, kept and count must be 4-byte aligned");
  const uint64_t rows = n_seqs * n_kv_heads;
  const qe::Bytes m{mass, 4 * mass_stride * rows}, l{lens, 4 * n_seqs}, k{kept, 4 * ((rows - 1) * kept_stride + keep)}, c{count, 4 * n_seqs};
  if (k.meets(m) || k.meets(l) || k.meets(c) || c.meets(m) || c.meets(l))
    return qe::set_error(QE_ERR_ARG, "kept and count must not overlap each other, mass or lens");
  qe::KeepArgs a{mass, lens, kept, count, mass_stride, kept_stride, uint32_t(n_kv_heads), uint32_t(keep), uint32_t(sinks), uint32_t(recent)};
  // positions of a row that registers hold: groups x 256 x 16 waves
  auto* const kern = mass_stride <= 8 * 4096 ? qe::k_page_keep<8> : mass_stride <= 16 * 4096 ? qe::k_page_keep<16> : qe::k_page_keep<0>;
  kern<<<uint32_t(rows), qe::kKeepThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "page keep launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

int qe_op_page_move(const qe_pages* pages, const int32_t* src, uint64_t src_heads, uint64_t src_stride,
                    const int32_t* count, const int32_t* first, float* mass, uint64_t mass_stride, void* stream) {
  qe::MoveArgs a{};
  if (int rc = qe::check_pages(pages, &a.p, &a.st)) return rc;
  if (!src || !count) return qe::set_error(QE_ERR_ARG, "null argument");
  if (src_heads != 1 && src_heads != a.p.n_kv) return qe::set_error(QE_ERR_ARG, "src_heads must be 1 or n_kv_heads");
  if (src_stride == 0 || src_stride > 0x7FFFFFFFull || mass_stride > 0x7FFFFFFFull || (mass && mass_stride == 0))
    return qe::set_error(QE_ERR_ARG, "src_stride and mass_stride must be above 0 and below 2^31");
  if (pages->n_pages > 0xFFFFFFFEull / (pages->page_size * pages->n_kv_heads))
    return qe::set_error(QE_ERR_ARG, "need n_pages * n_kv_heads * page_size < 2^32 - 1");
  if (uint64_t(a.p.n_seqs) * a.p.n_kv >= 1u << 19) return qe::set_error(QE_ERR_ARG, "need n_seqs * n_kv_heads < 2^19");
  if ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(count) | reinterpret_cast<uintptr_t>(first) |
       reinterpret_cast<uintptr_t>(mass)) % 4)
    return qe::set_error(QE_ERR_ARG, "src, count, first and mass must be 4-byte aligned");
  const uint64_t page_bytes = qe_page_bytes(pages->n_pages, pages->page_size, pages->n_kv_heads, pages->kv_dtype);
  const uint64_t exps = pages->kv_dtype == QE_KV_FP8 ? page_bytes / qe::kPageDim : 0;
  const uint64_t items = uint64_t(a.p.n_seqs) * a.p.n_kv;
  const qe::Bytes to[] = {{pages->k, page_bytes}, {pages->v, page_bytes}, {pages->k_exp, exps}, {pages->v_exp, exps},
                          {mass, 4 * mass_stride * items}};
  const qe::Bytes in[] = {{src, 4 * src_stride * src_heads * a.p.n_seqs}, {count, 4ull * a.p.n_seqs}, {first, 4ull * a.p.n_seqs}};
  for (const qe::Bytes& t : to)
    for (const qe::Bytes& i : in)
      if (t.meets(i)) return qe::set_error(QE_ERR_ARG, "src, count and first must not overlap what is moved");
  for (int i = 0; i < 4; i++)
    if (to[4].meets(to[i])) return qe::set_error(QE_ERR_ARG, "mass must not overlap the pages");
  a.src = src;
  a.count = count;
  a.first = first;
  a.mass = mass;
  a.mass_stride = mass_stride;
  a.src_heads = uint32_t(src_heads);
  a.src_stride = uint32_t(src_stride);
  const bool fp8 = pages->kv_dtype == QE_KV_FP8;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (src_stride <= qe::kFewMoves) {
    (fp8 ? qe::k_page_move_few<true> : qe::k_page_move_few<false>)<<<uint32_t(items), qe::kMoveThreads, 0, st>>>(a);
  } else {
    const uint32_t grid = uint32_t(items) * (fp8 ? qe::move_parts<true>() : qe::move_parts<false>());
    (fp8 ? qe::k_page_move<true> : qe::k_page_move<false>)<<<grid, qe::kMoveThreads, 0, st>>>(a, uint32_t(items));
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "page move launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
