// Logits processing between the head and the sampler (q3s_process_logits):
// penalties for repeated tokens, per-row biases and grammar masks.  Per entry
// v of a row, with n its occurrences in the history after the prompt:
//
//   x = logits[v];  seen: x < 0 ? x * rho : x / rho;  n > 0: (x - n * f) - p
//   biased: x + b;  not allowed by the mask: -inf
//
// Bytes that cannot be done without: the row once in (where the mask allows) and
// once out, its ids, its biases and its mask.  Two kernels:
//
// logits_kernel, few rows or rows that are long, ragged or in place.  A block owns
// a chunk of one row: it asks for the entries that the mask allows, counts the
// row's history ids that fall into the chunk in shared memory while they are on
// their way (integer atomics, so the order does not matter), and makes one pass
// over them.  The entries of the bias list, which are few as a rule, are written by
// one warp at the end.  In place, entries that nothing changes are neither read nor
// written.  Latency bounds it: a launch, then metadata, ids, counters, entries.
// One row of 3072 f32 (256 ids, 8 biases, a mask): 4.0 us; 1024 rows (up to 4096
// ids, 32 biases, masks): 12.4 us with the rows in L2 (4.5 us at the copy rate), of
// which 6.8 us without the histories; 48 rows of 100003 bf16 (up to 6000 ids): 15.5 us.
//
// stream_kernel, eight rows a multiprocessor or more, of one length up to 4096 and
// on 16 bytes.  Blocks stay and stream rows through shared memory; see there.
#include <cmath>
#include <cstdint>
#include <string>

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/q3s_sampler.h"
#include "q3s_device.cuh"
#include "q3s_internal.h"

namespace q3s {
namespace {

// 128 threads: with 256, and a thread's vectors in registers, 1024 rows of 3072 took
// 25 us against 22 us.
constexpr int THREADS = 128;
constexpr int STEP = 8 * THREADS;   // a block's chunk of a row is a multiple of it
constexpr int CHUNK = 3 * STEP, MAX_CHUNK = 8 * STEP;
constexpr int BLOCKS = 7;           // of a multiprocessor
constexpr int SM_BYTES = 227 << 10;  // shared memory of a multiprocessor's blocks
constexpr int MAX_STREAM = 4096;     // entries of a row of the stream kernel
constexpr int MAX_VOCAB = 1 << 26;

constexpr int BIASES = 64;          // a chunk's bias entries that are kept at hand
constexpr int WINDOW = 2 * BIASES;  // places whose sums take the same memory
constexpr int MAX_BIASES = 1 << 20;  // of a row: 20 ms in one chunk, 81 ms in place

// A counter word: the occurrences after the prompt, whether the prompt has the
// id, and whether the bias list does.
constexpr uint32_t SEEN = 1u << 31;
constexpr uint32_t BIASED = 1u << 30;
constexpr uint32_t COUNT = BIASED - 1;

struct LogitsArgs {
  q3s_logits_batch b;
  long long row0;  // of the launch's first block
  int chunk;      // entries of a block
  int places;     // counters per chunk, a multiple of 8; 0 without histories
  int stage;      // bytes of the chunk's entries in shared memory
  bool in_place;
  int id_shift;   // log2 of the bytes of an id of the history
  uint64_t wait_ns;  // limit of the wait for a row's copy
  bool hold_refill;  // testing hook: no row after the first ones is asked for
};

__device__ __forceinline__ float neg_infinity() { return __int_as_float(0xff800000); }

template <int DT>
constexpr int width = DT == Q3S_DTYPE_F32 ? 4 : 2;  // bytes of an element

template <int DT>
__device__ __forceinline__ float load_logit(const void* p, long long i) {
  if (DT == Q3S_DTYPE_F32) return static_cast<const float*>(p)[i];
  return __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}

template <int DT>
__device__ __forceinline__ void store_logit(void* p, long long i, float x) {
  if (DT == Q3S_DTYPE_F32)
    static_cast<float*>(p)[i] = x;
  else
    static_cast<uint16_t*>(p)[i] = __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// VE entries as they lie in memory.
template <int DT, int VE>
struct Raw {
  static constexpr int WORDS = VE * width<DT> < 4 ? 1 : VE * width<DT> / 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const char* p) {
    if (WORDS == 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      w[0] = x.x, w[1 % WORDS] = x.y, w[2 % WORDS] = x.z, w[3 % WORDS] = x.w;
    } else if (WORDS == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x, w[1 % WORDS] = x.y;
    } else if (VE * width<DT> == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if (DT == Q3S_DTYPE_F32) return __uint_as_float(w[i % WORDS]);
    return __uint_as_float(i & 1 ? w[i / 2 % WORDS] & 0xFFFF0000u : w[i / 2 % WORDS] << 16);
  }
  __device__ __forceinline__ void set(int i, float x) {
    if (DT == Q3S_DTYPE_F32) {
      w[i % WORDS] = __float_as_uint(x);
    } else {
      const uint32_t h = __bfloat16_as_ushort(__float2bfloat16_rn(x));
      w[i / 2 % WORDS] = i & 1 ? w[i / 2 % WORDS] | h << 16 : h;
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if (WORDS == 4)
      __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1 % WORDS], w[2 % WORDS], w[3 % WORDS]));
    else if (WORDS == 2)
      __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1 % WORDS]));
    else if (VE * width<DT> == 4)
      __stcs(reinterpret_cast<uint32_t*>(p), w[0]);
    else
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
  }
};

constexpr uint32_t NOWHERE = 0xFFFFFFFFu;

// Four consecutive ids as they lie in memory.
struct RawIds {
  uint4 a, b;  // b: of 64-bit ids

  __device__ __forceinline__ void load(const char* p, int type, uint32_t i) {
    if (type == Q3S_IDS_U16) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p + i * 2ull));
      a.x = x.x, a.y = x.y;
    } else if (type == Q3S_IDS_U32) {
      a = __ldg(reinterpret_cast<const uint4*>(p + i * 4ull));
    } else {
      const uint4* q = reinterpret_cast<const uint4*>(p + i * 8ull);
      a = __ldg(q), b = __ldg(q + 1);
    }
  }
};

// Ids of a row's history as places of its chunk, NOWHERE for other ids.
struct Ids {
  const char* p;
  int type;
  uint32_t n;            // ids
  uint32_t head;         // of them before the first multiple of four in memory
  uint32_t first, span;  // places [first, first + span)
  uint32_t from;         // the id at place `first`, below 2^26

  __device__ __forceinline__ uint32_t fours() const { return (n - head) / 4; }
  // An id below `from` wraps to more than any span.
  __device__ __forceinline__ uint32_t place(uint32_t id) const {
    return id - from < span ? id - from + first : NOWHERE;
  }
  __device__ __forceinline__ uint32_t place64(uint32_t low, uint32_t high) const {
    return high ? NOWHERE : place(low);
  }
  __device__ __forceinline__ uint32_t one(uint32_t i) const {
    if (type == Q3S_IDS_U16) return place(__ldg(reinterpret_cast<const uint16_t*>(p) + i));
    if (type == Q3S_IDS_U32) return place(__ldg(reinterpret_cast<const uint32_t*>(p) + i));
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p) + i);
    return place64(x.x, x.y);
  }
  __device__ __forceinline__ uint4 places(const RawIds& r) const {
    if (type == Q3S_IDS_U16)
      return make_uint4(place(r.a.x & 0xFFFFu), place(r.a.x >> 16), place(r.a.y & 0xFFFFu),
                        place(r.a.y >> 16));
    if (type == Q3S_IDS_U32) return make_uint4(place(r.a.x), place(r.a.y), place(r.a.z), place(r.a.w));
    return make_uint4(place64(r.a.x, r.a.y), place64(r.a.z, r.a.w), place64(r.b.x, r.b.y),
                      place64(r.b.z, r.b.w));
  }
};

// All that the batch says of a row, asked for at once: what depends on it waits
// for one access, not for one after another.
struct Meta {
  q3s_logits_params p{1.0f, 0.0f, 0.0f};
  long long mask = -1, offset = 0, h0 = 0, h1 = 0, prompt = 0, e0 = 0, e1 = 0;
  int vocab;

  __device__ __forceinline__ Meta(const LogitsArgs& a, long long r) {
    const q3s_logits_batch& b = a.b;
    vocab = b.vocab;
    if (b.params) p = b.params[r * b.params_stride];
    if (b.masks) mask = b.mask_rows ? b.mask_rows[r] : r;
    if (b.row_vocab) vocab = b.row_vocab[r];
    if (b.row_offsets) offset = b.row_offsets[r];
    if (a.places) {
      h0 = b.history_offsets[r];
      h1 = b.history_ends ? b.history_ends[r] : b.history_offsets[r + 1];
      if (b.prompt_lens) prompt = b.prompt_lens[r];
    }
    if (b.bias_offsets) {
      e0 = b.bias_offsets[r];
      e1 = b.bias_offsets[r + 1];
    }
  }
  __device__ __forceinline__ int status(const LogitsArgs& a) const {
    if (vocab < 0 || vocab > a.b.vocab || h1 - h0 > (long long)COUNT || e1 - e0 > MAX_BIASES)
      return Q3S_STATUS_UNSUPPORTED;
    if (!isfinite(p.repetition) || p.repetition <= 0.0f) return Q3S_STATUS_INVALID_REPETITION_PENALTY;
    if (!isfinite(p.presence) || !isfinite(p.frequency)) return Q3S_STATUS_INVALID_PENALTY;
    return mask >= a.b.num_masks ? Q3S_STATUS_INVALID_MASK : Q3S_STATUS_OK;
  }
};

// What a chunk needs of its row.
struct Row {
  const char* in;  // entry 0
  char* out;
  int lo;     // first entry of the chunk; below 0 by the row's skew in chunk 0
  int first;  // places [first, end) of the chunk hold entries lo + place
  int end;
  const uint32_t* words;  // the row's mask, or NULL
  q3s_logits_params p;
  double inverse;  // of the repetition penalty
  uint32_t ids, prompt;  // of the history, and how many of them are the prompt's
  long long e0, e1;      // biases

  // Chunk `part` of row r.  Places start as far before the row as out's row starts
  // behind a vector of VE: whole vectors of places are then aligned there.
  template <int IN, int OUT, int VE>
  static __device__ __forceinline__ Row part_of(const LogitsArgs& a, const Meta& m, long long r, int part) {
    const q3s_logits_batch& b = a.b;
    Row w;
    w.in = static_cast<const char*>(b.logits) + (b.row_offsets ? m.offset : r * b.row_stride) * width<IN>;
    w.out = static_cast<char*>(b.out) + (b.row_offsets ? m.offset : r * b.out_stride) * width<OUT>;
    w.lo = part * a.chunk - (int)(reinterpret_cast<uintptr_t>(w.out) / width<OUT> % VE);
    w.first = w.lo < 0 ? -w.lo : 0;
    w.end = min(m.vocab - w.lo, a.chunk);
    return w;
  }

  // The rest from the metadata of a valid row; returns its history.
  __device__ __forceinline__ Ids take(const LogitsArgs& a, const Meta& m) {
    p = m.p;
    e0 = m.e0, e1 = m.e1;
    words = m.mask >= 0 ? a.b.masks + m.mask * a.b.mask_stride : nullptr;
    ids = m.h1 > m.h0 ? (uint32_t)(m.h1 - m.h0) : 0;
    if (p.repetition == 1.0f && p.presence == 0.0f && p.frequency == 0.0f) ids = 0;
    inverse = ids ? __drcp_rn((double)p.repetition) : 0.0;
    prompt = (uint32_t)max(0ll, min(m.prompt, (long long)COUNT));
    const uintptr_t history = reinterpret_cast<uintptr_t>(a.b.history) + (m.h0 << a.id_shift);
    Ids h;
    h.p = reinterpret_cast<const char*>(history);
    h.type = a.b.history_type;
    h.n = ids;
    h.head = min(ids, (uint32_t)(-(long long)(history >> a.id_shift) & 3));
    h.first = first;
    h.span = end - first;
    h.from = lo + first;
    return h;
  }
};

// x / rho rounded to nearest (with divisions the pass over a chunk of 3072 took 12.5
// thousand cycles, with products 5.9), as one product in 64 bits: inverse is 1 / rho to
// 53 bits, so the product is within 2^-52 of the quotient, relatively.  A
// quotient of two 24-bit significands is no midpoint between two f32 values and
// no nearer to one than 2^-49: X 2^k - M P, with X and P below 2^24, M below 2^25
// and odd and k at least 24, is a whole number and not 0.  So both round alike.
// Quotients below the normal range can be midpoints: they are divided.
__device__ __forceinline__ float quotient(float x, double inverse) {
  return __double2float_rn(__dmul_rn((double)x, inverse));
}

// Whether the quotient q of x has to be divided.
__device__ __forceinline__ bool subnormal(float x, float q) {
  return fabsf(q) < 1.17549435e-38f && x != 0.0f;
}

// x of an entry with counter c, where q is x / repetition.
__device__ __forceinline__ float penalised_by(float x, uint32_t c, const q3s_logits_params& p,
                                              float q) {
  const uint32_t n = c & COUNT;
  const float y = x < 0.0f ? __fmul_rn(x, p.repetition) : q;
  if ((n || (c & SEEN)) && p.repetition != 1.0f) x = y;
  const float z = __fsub_rn(__fsub_rn(x, __fmul_rn((float)n, p.frequency)), p.presence);
  return n ? z : x;
}

__device__ __forceinline__ float penalised(float x, uint32_t c, const q3s_logits_params& p,
                                        double inverse) {
  float q = quotient(x, inverse);
  if (subnormal(x, q)) q = __fdiv_rn(x, p.repetition);
  return penalised_by(x, c, p, q);
}

__device__ __forceinline__ bool masked(const Row& row, int v) {
  return row.words && !(__ldg(row.words + (v >> 5)) >> (v & 31) & 1);
}

__device__ __forceinline__ void count_id(uint32_t* count, uint32_t at, bool prompt) {
  if (at == NOWHERE) return;
  if (prompt)
    atomicOr(count + at, SEEN);
  else
    atomicAdd(count + at, 1u);
}

// Counts the row's history.  Four ids at a time from the first multiple of four
// in memory on (`next`: this thread's first, already asked for); the up to six
// others one by one.
template <int THREADS>
__device__ __forceinline__ void count_ids(const Ids& ids, uint32_t prompt, uint32_t* c,
                                          RawIds next) {
  const uint32_t fours = ids.fours(), rest = ids.n - 4 * fours, rank = threadIdx.x;
  if (rank < rest) {
    const uint32_t i = rank < ids.head ? rank : rank + 4 * fours;
    count_id(c, ids.one(i), i < prompt);
  }
  for (uint32_t i = rank; i < fours; i += THREADS) {
    const uint4 at = ids.places(next);
    if (i + THREADS < fours) next.load(ids.p, ids.type, ids.head + 4 * (i + THREADS));
    const uint32_t first = ids.head + 4 * i;  // ids first .. first + 3
    count_id(c, at.x, first < prompt);
    count_id(c, at.y, first + 1 < prompt);
    count_id(c, at.z, first + 2 < prompt);
    count_id(c, at.w, first + 3 < prompt);
  }
}

// The entries of the row's bias list that fall into the chunk, in list order, or
// the sums of a window of places (add_many_biases).
union Biases {
  struct {
    uint32_t at[BIASES];
    float value[BIASES];
  };
  uint32_t sum[WINDOW];
};

// An entry as it lies in memory.
struct RawBias {
  uint32_t id;
  float value;

  __device__ __forceinline__ void load(const q3s_logits_batch& b, long long i) {
    id = __ldg(b.bias_ids + i);
    value = __ldg(b.bias_values + i);
  }
};

// One warp: collects them, as far as they fit, and marks their counters.  `next`
// is the lane's entry of the first 32, already asked for.  Returns how many
// there are.
__device__ __forceinline__ int collect_biases(const q3s_logits_batch& b, const Row& row,
                                              const Ids& ids, uint32_t* count, Biases& list,
                                              RawBias next) {
  const int lane = threadIdx.x % 32;
  int n = 0;
  for (long long e = row.e0; e < row.e1; e += 32) {
    if (e > row.e0 && e + lane < row.e1) next.load(b, e + lane);
    const uint32_t at = e + lane < row.e1 ? ids.place(next.id) : NOWHERE;
    const unsigned in = __ballot_sync(0xFFFFFFFFu, at != NOWHERE);
    const int to = n + __popc(in & ((1u << lane) - 1));
    if (at != NOWHERE) {
      if (to < BIASES) list.at[to] = at, list.value[to] = next.value;
      if (row.ids) atomicOr(count + at, BIASED);
    }
    n += __popc(in);
  }
  __syncwarp();
  return n;
}

// The same warp, a lane for each of the n entries of the list: the lane of
// an id's first entry adds up its values in list order and writes the entry.
// TAKE: the entry's counter is left at 0.  `held`: the lane's first entry's
// logit and mask, already asked for.
struct Held {
  float x;
  bool off;
};

template <int IN>
__device__ __forceinline__ Held hold(const Row& row, uint32_t at) {
  const int i = row.lo + (int)at;
  return at == NOWHERE ? Held{0.0f, true} : Held{load_logit<IN>(row.in, i), masked(row, i)};
}

// The place of the lane's first entry of the n that collect_biases() found.
__device__ __forceinline__ uint32_t first_place(int n, const Biases& list) {
  const int lane = threadIdx.x % 32;
  return lane < n ? list.at[lane] : NOWHERE;
}

// Writes the entry at a place with the sum of its biases.
template <int OUT, bool TAKE>
__device__ __forceinline__ void write_biased(const Row& row, uint32_t* count, uint32_t at, Held held,
                                             float sum) {
  const uint32_t c = !row.ids ? 0 : TAKE ? atomicExch(count + at, 0u) : count[at];
  if (!held.off)
    store_logit<OUT>(row.out, row.lo + (int)at,
                     __fadd_rn(c ? penalised(held.x, c, row.p, row.inverse) : held.x, sum));
}

template <int IN, int OUT, bool TAKE>
__device__ __forceinline__ void add_biases(const Row& row, uint32_t* count, int n, Held held,
                                           const Biases& list) {
  const int lane = threadIdx.x % 32;
  for (int e = lane; e < n; e += 32) {
    const uint32_t at = list.at[e];
    float sum = list.value[e];
    if (e >= 32) held = hold<IN>(row, at);
    bool first = true;
    for (int o = 0; o < n; ++o) {
      const uint32_t other = list.at[o];
      const float v = list.value[o];  // asked for with the place, whether it counts or not
      if (other != at) continue;
      if (o < e) first = false;
      if (o > e) sum = __fadd_rn(sum, v);
    }
    if (first) write_biased<OUT, TAKE>(row, count, at, held, sum);
  }
}

// The same warp, where the chunk has more entries than `Biases` holds: the sums of a
// window of places at a time, each in one walk over the row's list.  Looking each
// entry's id up among all the others would take time in the square of the list;
// this takes the list times the windows.  Lanes with one place take turns, so the
// list order holds.  The sums lie where the chunk's entries did (`stage`, four bytes
// a place), or where that is too small (in place there is none) in `list`: 300
// biases on a row of 3072 f32 take 12 us in the one and 41 us in the other, 5000
// 103 and 370 us.
//
// For chunk `part` of row r, from the batch alone and after all else in the kernel:
// nothing has to live in registers until then.  (Called with the row in the middle of
// stream_kernel, its loop spilled: 61440 rows of 2048 bf16 164 us instead of 126.)
template <int IN, int OUT, int VE>
__device__ __forceinline__ void add_many_biases(const LogitsArgs& a, long long r, int part,
                                                uint32_t* count, Biases& list, char* stage,
                                                int stage_bytes) {
  constexpr int AHEAD = 4;
  constexpr uint32_t NONE = 0xFFFFFFFFu;  // a NaN that no sum is left as
  const int lane = threadIdx.x % 32;
  const bool wide = stage_bytes >= 2 * (int)sizeof(Biases);
  uint32_t* sum = wide ? reinterpret_cast<uint32_t*>(stage) : list.sum;
  const int window = wide ? stage_bytes / 16 * 4 : WINDOW;
  const q3s_logits_batch& b = a.b;
  const Meta m(a, r);
  Row row = Row::part_of<IN, OUT, VE>(a, m, r, part);
  const Ids ids = row.take(a, m);
  // Calls each(place in the window, value, whether there is one) for the list.
  const auto walk = [&](int w0, const auto& each) {
#pragma unroll 1
    for (long long e = row.e0; e < row.e1; e += 32 * AHEAD) {
      RawBias raw[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (e + j * 32 + lane < row.e1) raw[j].load(b, e + j * 32 + lane);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const uint32_t at = e + j * 32 + lane < row.e1 ? ids.place(raw[j].id) : NOWHERE;
        const uint32_t to = at - (uint32_t)w0;
        each(to, raw[j].value, at != NOWHERE && to < (uint32_t)window);
      }
    }
  };
  const auto write = [&](int w0, uint32_t to, uint32_t s) {
    const uint32_t at = (uint32_t)w0 + to;
    write_biased<OUT, false>(row, count, at, hold<IN>(row, at), __uint_as_float(s));
  };
  __syncwarp();
#pragma unroll 1
  for (int w0 = row.first; w0 < row.end; w0 += window) {
    for (int j = 4 * lane; j < window; j += 128)
      *reinterpret_cast<uint4*>(sum + j) = make_uint4(NONE, NONE, NONE, NONE);
    __syncwarp();
    walk(w0, [&](uint32_t to, float value, bool mine) {
      if (!__any_sync(0xFFFFFFFFu, mine)) return;
      const unsigned same = __match_any_sync(0xFFFFFFFFu, mine ? to : (uint32_t)window + lane);
      const int turn = __popc(same & ((1u << lane) - 1));
      for (int k = 0; __any_sync(0xFFFFFFFFu, mine && turn >= k); ++k) {
        if (mine && turn == k) {
          const uint32_t s = sum[to];
          const float v = s == NONE ? value : __fadd_rn(__uint_as_float(s), value);
          sum[to] = isnan(v) ? 0x7FFFFFFFu : __float_as_uint(v);
        }
        __syncwarp();
      }
    });
    // Then each sum's entry: over the list once more, where who takes a sum writes
    // its entry, or over the places, whichever are fewer.
    if (row.e1 - row.e0 <= window) {
      walk(w0, [&](uint32_t to, float, bool mine) {
        const uint32_t s = mine ? atomicExch(sum + to, NONE) : NONE;
        if (s != NONE) write(w0, to, s);
      });
    } else {
#pragma unroll 4
      for (int j = lane; j < window; j += 32)
        if (sum[j] != NONE) write(w0, j, sum[j]);
    }
    __syncwarp();
  }
}

template <int BYTES>
__device__ __forceinline__ void copy_async(char* dst, const char* src) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES)
                 : "memory");
}

// The mask bits of entries v .. v + VE - 1, all of which are the row's.
template <int VE>
__device__ __forceinline__ uint32_t mask_bits(const Row& row, int v) {
  if (!row.words) return (1u << VE) - 1;
  const uint32_t word = __ldg(row.words + (v >> 5));
  uint32_t bits = word >> (v & 31);
  if ((v & 31) > 32 - VE)  // rows that do not start on a vector
    bits = __funnelshift_r(word, __ldg(row.words + (v >> 5) + 1), v & 31);
  return bits & ((1u << VE) - 1);
}

// Copies the chunk's entries to `stage` as they lie relative to 16 bytes: whole
// vectors without waiting, the ends one by one.  Returns where entry row.first is.
template <int IN>
__device__ __forceinline__ const char* copy_unlike(const Row& row, char* stage) {
  const char* src = row.in + (long long)(row.lo + row.first) * width<IN>;
  const int skew = (int)(reinterpret_cast<uintptr_t>(src) % 16);
  const int bytes = (row.end - row.first) * width<IN>;
  const int head = min(bytes, (16 - skew) % 16), body = (bytes - head) / 16 * 16;
  for (int i = head + 16 * threadIdx.x; i < head + body; i += 16 * THREADS)
    copy_async<16>(stage + skew + i, src + i);
  for (int i = threadIdx.x * width<IN>; i < bytes - body; i += THREADS * width<IN>) {
    const int at = i < head ? i : i + body;
    if (IN == Q3S_DTYPE_F32)
      *reinterpret_cast<uint32_t*>(stage + skew + at) = *reinterpret_cast<const uint32_t*>(src + at);
    else
      *reinterpret_cast<uint16_t*>(stage + skew + at) = *reinterpret_cast<const uint16_t*>(src + at);
  }
  return stage + skew;
}

// The chunk in vectors of VE places, thread by thread side by side.  `stage`
// holds the chunk's entries.  ALIKE: the rows of logits and out lie alike relative
// to vectors of VE, and every thread reads back the vectors that it copied there;
// else the places follow out's rows, and the entries are read one by one.  Returns,
// in the warp of the biases, whether they are still to be added (add_many_biases).
template <int IN, int OUT, int VE, bool ALIKE>
__device__ __forceinline__ bool process(const LogitsArgs& a, const Row& row, const Ids& ids,
                                        uint32_t* count, char* stage, Biases& biases) {
  constexpr uint32_t ALL = (1u << VE) - 1;
  const q3s_logits_batch& b = a.b;
  const bool last = threadIdx.x >= THREADS - 32;  // the warp of the biases
  RawIds next;
  RawBias bias;
  if (threadIdx.x < ids.fours()) next.load(ids.p, ids.type, ids.head + 4 * threadIdx.x);
  if (last && row.e0 + threadIdx.x % 32 < row.e1) bias.load(b, row.e0 + threadIdx.x % 32);
  uint64_t allowed = 0;  // bit e of the j-th VE bits: the mask allows entry e of vector j
  const char* entries = stage;  // ALIKE: by place, else from row.first on
  if (ALIKE) {
    constexpr int VECTORS = CHUNK / (THREADS * VE);
#pragma unroll 1
    for (int j0 = 0; j0 * THREADS * VE < row.end; j0 += VECTORS) {
#pragma unroll
      for (int j = 0; j < VECTORS; ++j) {
        const int at = ((j0 + j) * THREADS + threadIdx.x) * VE, v = row.lo + at;
        if (at < row.first || at + VE > row.end) continue;
        const uint32_t bits = mask_bits<VE>(row, v);
        allowed |= (uint64_t)bits << ((j0 + j) * VE);
        if (bits && !a.in_place)
          copy_async<VE * width<IN>>(stage + at * width<IN>, row.in + (long long)v * width<IN>);
      }
    }
  } else {
    entries = copy_unlike<IN>(row, stage);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (row.ids) {
    // Whole vectors, so that the places behind the row hold 0 too.
    for (int i = 4 * threadIdx.x; i < (row.end + 7) / 8 * 8; i += 4 * THREADS)
      *reinterpret_cast<uint4*>(count + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    count_ids<THREADS>(ids, row.prompt, count, next);
  }
  int given = 0;
  Held held{0.0f, true};
  if (row.e0 < row.e1 && last) {
    given = collect_biases(b, row, ids, count, biases, bias);
    if (given <= BIASES) held = hold<IN>(row, first_place(given, biases));
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (row.ids || !ALIKE) __syncthreads();
#pragma unroll 1
  for (int j = 0; j * THREADS * VE < row.end; ++j) {
    const int at = (j * THREADS + threadIdx.x) * VE, v = row.lo + at;
    if (at >= row.end || at + VE <= row.first) continue;
    uint32_t n[VE], any = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) n[e] = 0;
    if (row.ids) {
#pragma unroll
      for (int e = 0; e < VE; e += 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(count + at + e);
        n[e] = q.x, n[e + 1] = q.y, n[e + 2] = q.z, n[e + 3] = q.w;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) any |= n[e];
    }
    if (at >= row.first && at + VE <= row.end) {
      const uint32_t bits = ALIKE ? (uint32_t)(allowed >> (j * VE)) & ALL : mask_bits<VE>(row, v);
      float f[VE];
      if (ALIKE) {
        Raw<IN, VE> x;
        if (!a.in_place) {
          x.load(entries + at * width<IN>);
        } else {
          if (bits == ALL && !any) continue;
          if (bits) x.load(row.in + (long long)v * width<IN>);
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = bits >> e & 1 ? x.at(e) : 0.0f;  // others were not copied
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = load_logit<IN>(entries, at - row.first + e);
      }
      if (any) {  // all of a vector side by side, so that their latencies overlap
        float q[VE];
        bool divide = false;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          q[e] = quotient(f[e], row.inverse);
          divide = divide || subnormal(f[e], q[e]);
        }
        if (divide) {
#pragma unroll
          for (int e = 0; e < VE; ++e) q[e] = __fdiv_rn(f[e], row.p.repetition);
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          // The biases' own entries are left as they are.
          const float y = penalised_by(f[e], n[e], row.p, q[e]);
          if (!(n[e] & BIASED)) f[e] = y;
        }
      }
      Raw<OUT, VE> y;
#pragma unroll
      for (int e = 0; e < VE; ++e) y.set(e, bits >> e & 1 ? f[e] : neg_infinity());
      y.store(row.out + (long long)v * width<OUT>);
    } else {  // the row's ends
#pragma unroll 1
      for (int e = 0; e < VE; ++e) {
        if (at + e < row.first || at + e >= row.end) continue;
        const uint32_t c = row.ids ? count[at + e] : 0;
        float f = neg_infinity();
        if (!masked(row, v + e)) {
          f = load_logit<IN>(row.in, v + e);
          if (c && !(c & BIASED)) f = penalised(f, c, row.p, row.inverse);
        }
        store_logit<OUT>(row.out, v + e, f);
      }
    }
  }
  if (row.e0 >= row.e1) return false;
  __syncthreads();
  if (given > BIASES) return true;
  if (given) add_biases<IN, OUT, false>(row, count, given, held, biases);
  return false;
}

template <int IN, int OUT, int VE, bool ALIKE>
__global__ void __launch_bounds__(THREADS, BLOCKS) logits_kernel(
    const __grid_constant__ LogitsArgs a) {
  static_assert(MAX_CHUNK / THREADS <= 64, "the mask bits of a thread fit two words");
  extern __shared__ uint4 smem[];
  __shared__ Biases biases;
  char* stage = reinterpret_cast<char*>(smem);
  uint32_t* count = reinterpret_cast<uint32_t*>(stage + a.stage);
  const q3s_logits_batch& b = a.b;
  const long long r = a.row0 + blockIdx.x;
  const Meta m(a, r);
  const int status = m.status(a);
  if (blockIdx.y == 0 && threadIdx.x == 0) b.status[r] = (uint8_t)status;
  if (status == Q3S_STATUS_UNSUPPORTED) return;
  Row row = Row::part_of<IN, OUT, VE>(a, m, r, blockIdx.y);
  if (row.end <= row.first) return;
  if (status != Q3S_STATUS_OK) {
    for (int i = row.first + threadIdx.x; i < row.end; i += THREADS)
      store_logit<OUT>(row.out, row.lo + i, neg_infinity());
    return;
  }
  const Ids ids = row.take(a, m);
  if (process<IN, OUT, VE, ALIKE>(a, row, ids, count, stage, biases))
    add_many_biases<IN, OUT, VE>(a, r, blockIdx.y, count, biases, stage, a.stage);
}

// The rows of a block of stream_kernel whose bias lists hold more than `Biases`
// does, after all its rows have been written without them: their entries once more,
// from logits, with their counters counted again.  Apart from the loop, which has no
// registers to spare; until then the row's status is that it has not run.
template <int IN, int OUT, int VE, int T>
__device__ __forceinline__ void add_long_lists(const LogitsArgs& a, uint32_t* count, Biases& biases,
                                               char* ring, int ring_bytes) {
  const int rank = threadIdx.x;
#pragma unroll 1
  for (long long r = blockIdx.x; r < a.b.num_rows; r += gridDim.x) {
    const Meta m(a, r);
    if (m.status(a) != Q3S_STATUS_OK || m.e1 - m.e0 <= BIASES) continue;  // else done
    Row row = Row::part_of<IN, OUT, VE>(a, m, r, 0);
    const Ids ids = row.take(a, m);
    RawIds raw;
    if (rank < ids.fours()) raw.load(ids.p, ids.type, ids.head + 4 * rank);
    if (row.ids) count_ids<T>(ids, row.prompt, count, raw);
    __syncthreads();
    if (rank >= T - 32) add_many_biases<IN, OUT, VE>(a, r, 0, count, biases, ring, ring_bytes);
    if (rank == 0) a.b.status[r] = Q3S_STATUS_OK;
    __syncthreads();
    if (row.ids)
      for (int i = 4 * rank; i < a.places; i += 4 * T)
        *reinterpret_cast<uint4*>(count + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
}

// Many rows of one length: blocks of T threads that stay, each with ROWS rows
// under way or in hand in shared memory.  A row is written out as it
// came, masked, and the entries that its biases and its history touch are then
// computed and written once more: with rows this many they are few, and a lane
// for each of them costs less than a look at every counter.
//
// HBM bounds it.  61440 rows of 2048, bf16 to f32, with masks and 4 biases (756 MB):
// 124 us, 93 % of the rate of a copy; 65536 rows of 3072 f32 with 256 ids each
// (1.6 GB): 272 us, 91 %, the scattered second stores on top.  logits_kernel on the
// same rows: 238 and 352 us.  Earlier steps: one bulk copy a row by one thread 137 / 327
// us where cp.async by all lanes took 157 / 434; with the ids and biases asked for at
// the top and counted after the row is out, 129 / 308; T = 64 then, 32 threads 137 / 371,
// 128 threads 160 / 319.
template <int IN, int OUT, int VE, int ROWS, int T>
__global__ void __launch_bounds__(T, ROWS == 2 ? 6 : 12) stream_kernel(
    const __grid_constant__ LogitsArgs a) {
  constexpr uint32_t ALL = (1u << VE) - 1;
  constexpr int AHEAD = 4;
  extern __shared__ uint4 smem[];
  __shared__ Biases biases;
  const q3s_logits_batch& b = a.b;
  const int rank = threadIdx.x, vocab = b.vocab;
  const auto sync = [] {
    if (T == 32)
      __syncwarp();
    else
      __syncthreads();
  };
  char* ring = reinterpret_cast<char*>(smem);
  uint32_t* count = reinterpret_cast<uint32_t*>(ring + ROWS * a.stage);
  for (int i = 4 * rank; i < a.places; i += 4 * T)
    *reinterpret_cast<uint4*>(count + i) = make_uint4(0, 0, 0, 0);
  __shared__ uint64_t arrived[ROWS];
  __shared__ int here[ROWS];  // one a row under way: a refused row ends without a barrier
  __shared__ int late;  // rows whose bias lists are left to add_long_lists()
  if (rank == 0) {
    late = 0;
    for (int s = 0; s < ROWS; ++s) mbar_init(&arrived[s], 1);
    fence_mbarrier_init();
  }
  sync();
  const auto copy = [&](long long r, int slot) {
    if (rank != 0 || r >= b.num_rows) return;
    fence_proxy_async_smem();  // the slot's last row has been read
    mbar_arrive_expect_tx(&arrived[slot], a.stage);
    bulk_copy_g2s(ring + slot * a.stage,
                  static_cast<const char*>(b.logits) + r * b.row_stride * width<IN>, a.stage,
                  &arrived[slot]);
  };
  long long r = blockIdx.x;
#pragma unroll 1
  for (int s = 0; s < ROWS - 1; ++s) copy(r + (long long)s * gridDim.x, s);
  Meta next(a, r);
  int slot = 0;
  uint32_t parity = 0;
#pragma unroll 1
  for (; r < b.num_rows; r += gridDim.x) {
    const Meta m = next;
    const int status = m.status(a);
    const bool ok = status == Q3S_STATUS_OK;
    Row row;
    row.out = static_cast<char*>(b.out) + r * b.out_stride * width<OUT>;
    row.lo = row.first = 0;
    row.end = vocab;
    const Ids ids = row.take(a, m);
    // On their way while the row is waited for and written out.  Of a refused row
    // nothing is read: its ranges may lie anywhere.
    const bool last = rank >= T - 32;  // the warp of the biases
    RawIds raw;
    RawBias bias;
    if (ok && rank < ids.fours()) raw.load(ids.p, ids.type, ids.head + 4 * rank);
    if (ok && last && row.e0 + rank % 32 < row.e1) bias.load(b, row.e0 + rank % 32);
    if (!a.hold_refill) copy(r + (ROWS - 1ll) * gridDim.x, slot ? slot - 1 : ROWS - 1);
    const char* stage = ring + slot * a.stage;
    uint64_t* bar = &arrived[slot];
    const uint32_t phase = parity;
    if (++slot == ROWS) slot = 0, parity ^= 1;
    if (r + gridDim.x < b.num_rows) next = Meta(a, r + gridDim.x);
    if (rank == 0) b.status[r] = (uint8_t)status;
    if (rank == 0) here[slot] = mbar_wait_bounded(bar, phase, a.wait_ns);
    sync();
    if (!here[slot]) break;
    mbar_try_wait(bar, phase);  // this thread, too, sees the copy complete
    if (!ok) {
      if (status != Q3S_STATUS_UNSUPPORTED)
        for (int i = rank; i < vocab; i += T) store_logit<OUT>(row.out, i, neg_infinity());
      continue;
    }
#pragma unroll 1
    for (int i0 = rank * VE; i0 < vocab; i0 += AHEAD * T * VE) {
      Raw<IN, VE> x[AHEAD];
      uint32_t word[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = i0 + j * T * VE;
        if (i >= vocab) break;
        word[j] = row.words ? __ldg(row.words + (i >> 5)) : 0xFFFFFFFFu;
        x[j].load(stage + i * width<IN>);
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = i0 + j * T * VE;
        if (i >= vocab) break;
        const uint32_t bits = word[j] >> (i & 31) & ALL;
        Raw<OUT, VE> y;
#pragma unroll
        for (int e = 0; e < VE; ++e) y.set(e, bits >> e & 1 ? x[j].at(e) : neg_infinity());
        y.store(row.out + i * width<OUT>);
      }
    }
    int given = 0;  // known to the last warp
    if (row.e0 < row.e1 && last)
      given = row.e1 - row.e0 > BIASES ? BIASES + 1 : collect_biases(b, row, ids, count, biases, bias);
    if (row.ids) count_ids<T>(ids, row.prompt, count, raw);
    if (row.ids || row.e0 < row.e1) sync();
    row.in = stage;
    if (given > BIASES) {
      if (rank % 32 == 0) b.status[r] = Q3S_STATUS_NOT_RUN, late = 1;
    } else if (given) {
      const Held held = hold<IN>(row, first_place(given, biases));
      add_biases<IN, OUT, true>(row, count, given, held, biases);
    }
    if (row.ids) {
      // Who takes an entry's counter writes the entry; the biases took theirs.
      const auto write = [&](uint4 places) {
        const uint32_t at[4] = {places.x, places.y, places.z, places.w};
        uint32_t c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = at[e] == NOWHERE ? 0 : count[at[e]];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          c[e] = c[e] && !(c[e] & BIASED) ? atomicExch(count + at[e], 0u) : 0;
        if (ROWS == 2) {
          // Side by side, so that their latencies overlap (65536 rows of 3072 f32 274 us, one
          // after the other 289 us); with four rows in the ring there are no registers for
          // that (61440 rows of 2048 bf16 141 us, 127 us this way).
          float x[4], q[4];
          bool divide = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = c[e] ? load_logit<IN>(stage, at[e]) : 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            q[e] = quotient(x[e], row.inverse);
            divide = divide || subnormal(x[e], q[e]);
          }
          if (divide) {
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = __fdiv_rn(x[e], row.p.repetition);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c[e] && !masked(row, (int)at[e]))
              store_logit<OUT>(row.out, at[e], penalised_by(x[e], c[e], row.p, q[e]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c[e] && !masked(row, (int)at[e]))
              store_logit<OUT>(row.out, at[e],
                               penalised(load_logit<IN>(stage, at[e]), c[e], row.p, row.inverse));
        }
      };
      const uint32_t fours = ids.fours(), rest = ids.n - 4 * fours;
      if (rank < rest)
        write(make_uint4(ids.one(rank < ids.head ? rank : rank + 4 * fours), NOWHERE, NOWHERE,
                         NOWHERE));
#pragma unroll 1
      for (uint32_t i = rank; i < fours; i += T) {
        if (i >= T) raw.load(ids.p, ids.type, ids.head + 4 * i);
        write(ids.places(raw));
      }
    }
    sync();  // the row and the counters are no longer read
  }
  if (r >= b.num_rows) {
    if (late) add_long_lists<IN, OUT, VE, T>(a, count, biases, ring, ROWS * a.stage);
    return;
  }
  // A copy did not come in time: its row and those after it have not run.  The
  // block stays, for a limited time, until no copy is under way to its ring.
  if (rank == 0) {
    const int first = slot ? slot - 1 : ROWS - 1;  // row r's
    const uint32_t phase = slot ? parity : parity ^ 1;
    for (int s = 0; s < ROWS; ++s)
      if (r + (long long)s * gridDim.x < b.num_rows)
        mbar_wait_bounded(&arrived[(first + s) % ROWS], first + s < ROWS ? phase : phase ^ 1,
                          a.wait_ns);
    for (; r < b.num_rows; r += gridDim.x) b.status[r] = Q3S_STATUS_NOT_RUN;
  }
}

template <int IN, int OUT, int VE, bool ALIKE>
cudaError_t launch(LogitsArgs& a, bool aligned, const ContextInfo& ci, cudaStream_t st) {
  // A row may start up to VE - 1 entries behind a vector's start.
  const long long places = a.b.vocab + (aligned ? 0 : VE - 1);
  const bool history = a.b.params && a.b.history_offsets;
  const int bytes = (a.in_place ? 0 : width<IN>) + (history ? 4 : 0);  // of an entry
  const auto chunks = [&](int chunk) { return places > chunk ? (places + chunk - 1) / chunk : 1; };
  const auto held = [&](int chunk) {  // blocks that the device holds
    const int fit = SM_BYTES / (chunk * bytes + 2048);
    return (long long)ci.sm_count * (fit < BLOCKS ? fit : BLOCKS);
  };
  // The smallest chunk with which all blocks are on the device at once: few rows
  // are spread over more blocks (one row of 3072: 4.0 us in three chunks, 6.0 us in
  // one), and long rows, whose every chunk looks at all of the row's history, over
  // no more than are at work together (48 rows of 100003: 15.5 us with chunks of
  // 5120, 20.4 us with 3072 at an earlier step).  Where none does that, 3072 (600 rows of 30001 f32:
  // 44 us, 63 us with 8192).
  a.chunk = STEP;
  while (a.chunk <= MAX_CHUNK && a.b.num_rows > held(a.chunk) / chunks(a.chunk)) a.chunk += STEP;
  if (a.chunk > MAX_CHUNK) a.chunk = CHUNK;
  const int most = places < a.chunk ? (int)((places + 7) / 8 * 8) : a.chunk;
  if (history) a.places = most;
  a.stage = a.in_place ? 0 : most * width<IN> + (ALIKE ? 0 : 16);
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem((const void*)logits_kernel<IN, OUT, VE, ALIKE>,
                                   MAX_CHUNK * (width<IN> + 4) + 16, ci.device, allowed);
  if (e != cudaSuccess) return e;
  for (a.row0 = 0; a.row0 < a.b.num_rows; a.row0 += 0x7FFFFFFF) {  // as many as a grid can have
    const long long rows = a.b.num_rows - a.row0;
    const dim3 grid((unsigned)(rows < 0x7FFFFFFF ? rows : 0x7FFFFFFF), (unsigned)chunks(a.chunk));
    logits_kernel<IN, OUT, VE, ALIKE><<<grid, THREADS, a.stage + a.places * 4, st>>>(a);
    const cudaError_t l = cudaGetLastError();
    if (l != cudaSuccess) return l;
  }
  return cudaSuccess;
}

template <int IN, int OUT, int VE, int ROWS, int T>
cudaError_t launch_stream(LogitsArgs& a, const ContextInfo& ci, cudaStream_t st) {
  a.stage = a.b.vocab * width<IN>;
  a.chunk = a.b.vocab;
  if (a.b.params && a.b.history_offsets) a.places = a.b.vocab;
  const int smem = ROWS * a.stage + a.places * 4;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem((const void*)stream_kernel<IN, OUT, VE, ROWS, T>,
                                   ROWS * MAX_STREAM * width<IN> + MAX_STREAM * 4, ci.device, allowed);
  if (e != cudaSuccess) return e;
  // As many blocks as the device holds at once.
  int held = 0;
  e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, stream_kernel<IN, OUT, VE, ROWS, T>, T, smem);
  if (e != cudaSuccess) return e;
  const long long blocks = (long long)ci.sm_count * (held > 0 ? held : 1);
  const int grid = (int)(a.b.num_rows < blocks ? a.b.num_rows : blocks);
  stream_kernel<IN, OUT, VE, ROWS, T><<<grid, T, smem, st>>>(a);
  return cudaGetLastError();
}

template <int IN, int OUT>
cudaError_t launch_typed(LogitsArgs& a, const ContextInfo& ci, cudaStream_t st) {
  constexpr int VE = IN == Q3S_DTYPE_F32 || OUT == Q3S_DTYPE_F32 ? 4 : 8;
  const q3s_logits_batch& b = a.b;
  const uintptr_t in = reinterpret_cast<uintptr_t>(b.logits) / width<IN>;
  const uintptr_t out = reinterpret_cast<uintptr_t>(b.out) / width<OUT>;
  const bool one = b.num_rows == 1 && !b.row_offsets;
  const bool alike = (in - out) % VE == 0 &&
                     (one || b.row_offsets || (b.row_stride - b.out_stride) % VE == 0);
  const bool aligned = in % VE == 0 && (one || (!b.row_offsets && b.row_stride % VE == 0));
  // Eight rows a multiprocessor, of one length, that start on 16 bytes.  Two rows of
  // 8192 bytes or more in the ring (registers for six blocks a multiprocessor at
  // least; twelve spill, 442 us against 308 for 65536 rows of 3072 f32 at that step),
  // four of shorter ones (twelve blocks: 124 us for 61440 rows of 2048 bf16, 128 us
  // with ten).
  const int stage = b.vocab * width<IN>;
  if (b.num_rows >= 8LL * ci.sm_count && !b.row_offsets && !b.row_vocab && !a.in_place && alike &&
      b.vocab > 0 && b.vocab <= MAX_STREAM && b.vocab % 8 == 0 &&
      reinterpret_cast<uintptr_t>(b.logits) % 16 == 0 && b.row_stride * width<IN> % 16 == 0)
    return stage >= 8192 ? launch_stream<IN, OUT, VE, 2, 64>(a, ci, st)
                         : launch_stream<IN, OUT, VE, 4, 64>(a, ci, st);
  return alike ? launch<IN, OUT, VE, true>(a, aligned, ci, st)
               : launch<IN, OUT, VE, false>(a, false, ci, st);
}

int bad(const char* msg) {
  return record_error(Q3S_E_INVALID_ARGUMENT, std::string("q3s_process_logits: ") + msg);
}

int process_logits(q3s_context* ctx, const q3s_logits_batch* b, void* stream) {
  if (!ctx || !b) return bad("NULL context or batch");
  if (b->num_rows < 0 || b->vocab < 0) return bad("num_rows and vocab must be >= 0");
  if (b->vocab > MAX_VOCAB) return bad("vocab must be at most 2^26");
  if ((b->dtype != Q3S_DTYPE_F32 && b->dtype != Q3S_DTYPE_BF16) ||
      (b->out_dtype != Q3S_DTYPE_F32 && b->out_dtype != Q3S_DTYPE_BF16))
    return bad("dtype and out_dtype must be Q3S_DTYPE_F32 or Q3S_DTYPE_BF16");
  if (b->num_rows == 0) return Q3S_OK;
  if ((b->vocab > 0 && (!b->logits || !b->out)) || !b->status)
    return bad("logits, out and status are required");
  if (!b->row_offsets && (b->row_stride < 0 || b->out_stride < b->vocab))
    return bad("row_stride must be >= 0 and out_stride >= vocab");
  if (b->vocab > 0 && b->logits == b->out &&
      (b->dtype != b->out_dtype ||
       (!b->row_offsets && b->num_rows > 1 && b->row_stride != b->out_stride)))
    return bad("in place, out needs the type and the strides of logits");
  if (b->params_stride != 0 && b->params_stride != 1) return bad("params_stride must be 0 or 1");
  if (b->history_type != Q3S_IDS_U16 && b->history_type != Q3S_IDS_U32 &&
      b->history_type != Q3S_IDS_I64)
    return bad("unknown history_type");
  if (b->history_offsets && !b->history) return bad("history_offsets without history");
  if (b->bias_offsets && (!b->bias_ids || !b->bias_values))
    return bad("bias_offsets need bias_ids and bias_values");
  if (b->masks && (b->mask_stride < (b->vocab + 31LL) / 32 || b->num_masks < 0))
    return bad("mask_stride must be >= (vocab + 31) / 32 and num_masks >= 0");
  if (b->masks && !b->mask_rows && b->num_masks < b->num_rows)
    return bad("without mask_rows there must be a mask for each row");
  const ContextInfo ci = context_info(ctx);
  DeviceScope scope(ci.device);
  if (scope.err != cudaSuccess) return record_cuda_error(scope.err, "cudaSetDevice");
  LogitsArgs a;
  a.b = *b;
  const bool in32 = b->dtype == Q3S_DTYPE_F32, out32 = b->out_dtype == Q3S_DTYPE_F32;
  if (reinterpret_cast<uintptr_t>(b->logits) % (in32 ? 4 : 2) ||
      reinterpret_cast<uintptr_t>(b->out) % (out32 ? 4 : 2))
    return bad("logits and out must be aligned to their elements");
  a.in_place = b->logits == b->out;
  a.id_shift = b->history_type == Q3S_IDS_U16 ? 1 : b->history_type == Q3S_IDS_U32 ? 2 : 3;
  if (reinterpret_cast<uintptr_t>(b->history) & ((1 << a.id_shift) - 1))
    return bad("history must be aligned to its ids");
  a.places = 0;
  a.wait_ns = ci.test_wait_ns ? ci.test_wait_ns : 1000000000;
  a.hold_refill = ci.test_hold_refill;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e =
      in32 ? (out32 ? launch_typed<Q3S_DTYPE_F32, Q3S_DTYPE_F32>(a, ci, st)
                    : launch_typed<Q3S_DTYPE_F32, Q3S_DTYPE_BF16>(a, ci, st))
           : (out32 ? launch_typed<Q3S_DTYPE_BF16, Q3S_DTYPE_F32>(a, ci, st)
                    : launch_typed<Q3S_DTYPE_BF16, Q3S_DTYPE_BF16>(a, ci, st));
  if (e != cudaSuccess) return record_cuda_error(e, "logits kernel launch");
  return Q3S_OK;
}

}  // namespace
}  // namespace q3s

extern "C" int q3s_process_logits(q3s_context* ctx, const q3s_logits_batch* batch, void* stream) {
  return q3s::no_throw([&] { return q3s::process_logits(ctx, batch, stream); });
}
