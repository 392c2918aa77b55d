// A paged cache of bounded size: which positions each KV head keeps (qe_op_page_keep), and the move of
// kept rows to the front (qe_op_page_move). No reference counterpart.
#include "pages.h"

#include "device_common.h"
#include "status.h"

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
constexpr uint32_t kGroup = 256, kGroupsInRegs = 8, kWaves = kKeepThreads / 64;
constexpr uint32_t kInRegs = kWaves * kGroupsInRegs * kGroup;  // positions of a row that fit in registers
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
// Bound by latency, not by the 4 bytes a position: some ten barriers, and LDS counts that meet in one place.
template <bool REGS>
__global__ __launch_bounds__(kKeepThreads) void k_page_keep(KeepArgs a) {
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
  uint32_t keys[REGS ? kGroupsInRegs : 1][4];
  if constexpr (REGS) {
#pragma unroll
    for (uint32_t g = 0; g < kGroupsInRegs; g++)
      if (g < groups) load(g, keys[g]);
  }
  // f(first position, keys) of each group
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (REGS) {
#pragma unroll
      for (uint32_t g = 0; g < kGroupsInRegs; g++)
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

constexpr uint32_t kMoveThreads = 256;
enum Part { kMoveK, kMoveV, kMoveRest };

// A workgroup for a part of every row of a sequence and KV head: slices of 16 dims of K and of V, and what
// there is one of for a row (exponents, mass). Rows ascend and only ever move to the front, so what a chunk
// of rows writes no later chunk reads: within one, everything is read before anything is written.
template <bool FP8>
__global__ __launch_bounds__(kMoveThreads) void k_page_move(MoveArgs a) {
  constexpr uint32_t EL = FP8 ? 1 : 2, SLICES = 8;
  const uint32_t tid = threadIdx.x, item = blockIdx.x / (2 * SLICES + 1), part = blockIdx.x - item * (2 * SLICES + 1);
  const uint32_t s = item / a.p.n_kv, h = item - s * a.p.n_kv;
  const int64_t first = a.first ? a.first[s] : 0, capacity = capacity_of(a.p);
  const uint32_t count = uint32_t(min(int64_t(max(a.count[s], 0)), int64_t(a.src_stride)));
  const int32_t* src = a.src + (uint64_t(s) * a.src_heads + (a.src_heads == 1 ? 0 : h)) * a.src_stride;
  const uint32_t mask = (1u << a.p.page_shift) - 1;
  auto slot_of = [&](int64_t pos) -> int64_t {  // row index in the pages, -1: not there
    if (pos < 0 || pos >= capacity) return -1;
    const int32_t page = page_of(a.p, s, pos);
    return page < 0 ? -1 : int64_t(page_row(a.p, page, h, uint32_t(pos) & mask));
  };
  if (part < 2 * SLICES) {
    const bool k = part < SLICES;
    const uint32_t d = (part % SLICES) * 16 + (tid & 15);
    for (uint32_t i0 = 0; i0 < count; i0 += kMoveThreads / 16) {
      const uint32_t i = i0 + tid / 16;
      uint8_t* to = nullptr;
      uint32_t v = 0;
      if (i < count && src[i] != int32_t(i) && src[i] >= 0) {
        const int64_t x = slot_of(first + src[i]), y = slot_of(first + i);
        if (x >= 0 && y >= 0) {
          auto at = [&](int64_t r) {
            return k ? a.st.k + (size_t(r) * kPageDim + d) * EL
                     : a.st.v + (size_t(r & ~int64_t(kPageRun - 1)) * kPageDim + (r & (kPageRun - 1)) + d * kPageRun) * EL;
          };
          v = FP8 ? *at(x) : *reinterpret_cast<const uint16_t*>(at(x));
          to = at(y);
        }
      }
      __syncthreads();
      if (to) {
        if (FP8) *to = uint8_t(v);
        else *reinterpret_cast<uint16_t*>(to) = uint16_t(v);
      }
    }
    return;
  }
  float* mass = a.mass ? a.mass + uint64_t(item) * a.mass_stride : nullptr;
  for (uint32_t i0 = 0; i0 < count; i0 += kMoveThreads) {
    const uint32_t i = i0 + tid;
    int64_t to = -1, place = -1;
    uint32_t ke = 0, ve = 0;
    float m = 0.f;
    if (i < count && src[i] != int32_t(i) && src[i] >= 0) {
      const int64_t x = first + src[i], y = first + i, from = slot_of(x);
      if (FP8 && from >= 0 && (to = slot_of(y)) >= 0) {
        ke = a.st.k_exp[from];
        ve = a.st.v_exp[from];
      }
      if (mass && x >= 0 && y >= 0 && x < int64_t(a.mass_stride) && y < int64_t(a.mass_stride)) {
        place = y;
        m = mass[x];
      }
    }
    __syncthreads();
    if (to >= 0) {
      a.st.k_exp[to] = uint8_t(ke);
      a.st.v_exp[to] = uint8_t(ve);
    }
    if (place >= 0) mass[place] = m;
  }
  if (mass) {
    __syncthreads();
    const int64_t end = min(int64_t(a.p.lens[s]), int64_t(a.mass_stride));
    for (int64_t j = max(first + count, int64_t(0)) + tid; j < end; j += kMoveThreads) mass[j] = 0.f;
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
  (mass_stride <= qe::kInRegs ? qe::k_page_keep<true> : qe::k_page_keep<false>)<<<uint32_t(rows), qe::kKeepThreads, 0,
                                                                                  static_cast<hipStream_t>(stream)>>>(a);
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
  const uint32_t grid = uint32_t(items) * 17;
  (pages->kv_dtype == QE_KV_FP8 ? qe::k_page_move<true> : qe::k_page_move<false>)<<<grid, qe::kMoveThreads, 0,
                                                                                     static_cast<hipStream_t>(stream)>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return qe::set_error(QE_ERR_HIP, "page move launch failed: %s", hipGetErrorString(e));
  return QE_OK;
}

}  // extern "C"
