// A paged cache of bounded size: which positions each KV head keeps (qe_op_page_keep), and the move of
// kept rows to the front (qe_op_page_move). No reference counterpart.
#include "pages.h"

#include "device_common.h"
#include "status.h"

namespace qe {
namespace {

// ---- the choice ----
// A float as a whole number that orders as it does: NaN (0) below all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0;
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

// Sum over the workgroup's threads up to each, without its own; `all`: of all of them.
__device__ uint32_t scan_below(uint32_t v, uint32_t* waves, uint32_t& all) {
  const uint32_t wave = threadIdx.x >> 6, up = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) waves[wave] = up;
  __syncthreads();
  uint32_t below = up - v;
  all = 0;
  for (uint32_t i = 0; i < kKeepThreads / 64; i++) {
    if (i < wave) below += waves[i];
    all += waves[i];
  }
  return below;
}

// A workgroup for each sequence and KV head: the `need`-th largest of the middle by its digits of 8 bits
// from the top (a count of each digit among the values that agree so far), then everything above it and the
// first of what equals it.
__global__ __launch_bounds__(kKeepThreads) void k_page_keep(KeepArgs a) {
  __shared__ uint32_t digits[256], waves[kKeepThreads / 64], found[2];
  const uint32_t tid = threadIdx.x, s = blockIdx.x / a.n_kv, h = blockIdx.x - s * a.n_kv;
  const uint32_t len = uint32_t(min(int64_t(max(a.lens[s], 0)), int64_t(a.mass_stride)));
  const uint32_t keep = min(len, a.keep), sinks = min(a.sinks, keep), recent = min(a.recent, keep - sinks);
  const uint32_t from = sinks, to = len - recent;
  const float* mass = a.mass + uint64_t(blockIdx.x) * a.mass_stride;
  int32_t* kept = a.kept + uint64_t(blockIdx.x) * a.kept_stride;
  uint32_t need = keep - sinks - recent;  // of from .. to - 1
  uint32_t prefix = 0;
  const bool choose = need < to - from;
  if (choose && need)
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) digits[tid] = 0;
      __syncthreads();
      for (uint32_t j = from + tid; j < to; j += kKeepThreads) {
        const uint32_t key = order_of(mass[j]);
        if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&digits[key >> shift & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t d = 255, above = 0;
        while (above + digits[d] < need) above += digits[d--];
        found[0] = d;
        found[1] = above;
      }
      __syncthreads();
      prefix |= found[0] << shift;
      need -= found[1];
    }
  uint32_t at = 0, ties = 0;
  for (uint32_t x = 0; x < len; x += kKeepThreads) {
    const uint32_t j = x + tid;
    bool in = j < len, tie = false;
    if (in && choose && j >= from && j < to) {
      const uint32_t key = order_of(mass[j]);
      tie = need && key == prefix;
      in = keep - sinks - recent && key > prefix;
    }
    uint32_t all;
    const uint32_t rank = ties + scan_below(tie, waves, all);
    ties += all;
    in = in || (tie && rank < need);
    const uint32_t place = at + scan_below(in, waves, all);
    at += all;
    if (in) kept[place] = int32_t(j);
  }
  for (uint32_t i = keep + tid; i < a.keep; i += kKeepThreads) kept[i] = -1;
  if (h == 0 && tid == 0) a.count[s] = int32_t(keep);
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
  qe::k_page_keep<<<uint32_t(rows), qe::kKeepThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
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
