// Gradient of the embedding tables (q3s_embed_grad), by sorted tokens:
// grads[g][v] = scale * sum of grad_out[r] over the valid rows r with
// codes[r, g] = v.
//
// 1. split_kernel (several groups): the sort keys group by group, with the
//    rows that have a code outside its codebook dropped.
// 2. sort_kernel: sorts the kept rows of a group by code, rows of one code in
//    ascending order.  A cluster of blocks owns a bucket of consecutive codes
//    and reads all of the group's keys, each block a part: it counts those below
//    its bucket, which is where its rows go, and places its own.  Blocks of a
//    cluster tell each other their counts; no cluster waits for another.
// 3. reduce_kernel: warps add up the rows of each code in that order, and
//    those of long runs in pieces that are then joined in order.
//
// The order of the additions is fixed by the rows, so the gradient is the same bit
// for bit from call to call; atomics on the table would change it.  Bytes that
// cannot be done without: each row of grad_out once and the tables once.  A row
// is read once for each group; the groups' reads of rows that are still in L2
// count against L2.  Each kernel starts while the one before it ends.
#include <algorithm>
#include <cstdint>
#include <mutex>
#include <string>
#include <type_traits>

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/q3s_sampler.h"
#include "q3s_internal.h"

namespace cg = cooperative_groups;

namespace q3s {
namespace {

constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_BUCKET_BITS = 10;
constexpr int MAX_BUCKET = 1 << MAX_BUCKET_BITS;
constexpr int LIST = 512;  // keys of its bucket that a warp keeps in shared memory
constexpr int LIST_ROWS = 1 << (32 - MAX_BUCKET_BITS);  // rows that an entry can tell apart
constexpr int BATCH = 8;  // keys per lane in flight
constexpr int SPLIT_THREADS = 256;
constexpr int TEXT_THREADS = 256;
constexpr int REDUCE_THREADS = 128;
constexpr int REDUCE_WARPS = REDUCE_THREADS / 32;
constexpr uint32_t DROPPED = 0xFFFFFFFFu;
constexpr int MAX_HIDDEN = 1 << 30;  // 32-bit columns of a row's tiles go somewhat beyond its end
constexpr int JOIN = 16;           // pieces of a long run that one warp joins
constexpr uint32_t GROUPS = 1u << 16;  // `arrived` counts pieces below it, groups of them from it on

// Per-group workspace.
struct GroupWork {
  uint32_t* keys;   // [rows], several groups: the code of each row, or DROPPED
  uint32_t* rows;   // the kept rows, sorted by code
  uint2* range;     // [vocab]: first and one past last position in rows
  uint32_t* count;  // kept rows
  float4* partial;  // [blocks][2][tiles][32 lanes' columns]: sums of the pieces of long runs
  uint32_t* arrived;  // [blocks][2][tiles]: at the first of JOIN pieces, how many are done, and
                      // at the run's first one how many groups of them
};

struct GradArgs {
  q3s_embed_grad_batch b;  // grads and vocab (host arrays) are not read on the device
  void* grads[Q3S_MAX_CODE_GROUPS + 1];  // one more: the broadcast text
  int vocab[Q3S_MAX_CODE_GROUPS + 1];
  GroupWork work[Q3S_MAX_CODE_GROUPS + 1];
  int bucket_bits;  // log2 of the codes per block of the sort
  int block;   // positions of the sorted list per piece of a long run
  int blocks;  // pieces of the whole list; 0: no run can be long
  int slots;   // entries of `arrived`
  int tiles;  // column tiles of a row
  int chunk;  // consecutive codes per warp, at most 32
};

// What a kernel writes that the next one reads is read by ordinary loads or __ldcg: the
// next one starts before it is written, and __ldg is for memory that nothing writes
// while the kernel lives.
__device__ __forceinline__ void await_inputs() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void admit_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ uint64_t load_code(const void* p, int type, long long i) {
  if (type == Q3S_IDS_U16) return static_cast<const uint16_t*>(p)[i];
  if (type == Q3S_IDS_U32) return static_cast<const uint32_t*>(p)[i];
  return static_cast<const uint64_t*>(p)[i];
}

// Row r's code in a group, or DROPPED: a row with a code outside its
// codebook, or the padding id.
__device__ __forceinline__ uint32_t kept(const GradArgs& a, uint64_t code) {
  return a.b.padding_id >= 0 && code == (uint64_t)a.b.padding_id ? DROPPED : (uint32_t)code;
}

// The sort keys of several groups, group by group: a block reads the codes of
// SPLIT_ROWS rows as they lie in memory and turns them in shared memory (read
// column by column instead, every code of a warp lies in another line).  A
// broadcast text is one more group, with code 0 for every valid row.
constexpr int SPLIT_ROWS = 32;

// Bound by latency: 6 us for 4096 rows of 16 codes, 8 us for 32768, most of it the launch and two
// accesses one after the other.
__global__ void __launch_bounds__(SPLIT_THREADS) split_kernel(const GradArgs a, int groups) {
  const q3s_embed_grad_batch& b = a.b;
  __shared__ uint32_t code[SPLIT_ROWS * (Q3S_MAX_CODE_GROUPS + 1)];
  admit_next();
  const int pitch = b.groups | 1;  // odd: a column's rows lie in 32 banks
  const long long r0 = (long long)blockIdx.x * SPLIT_ROWS;
  const int rows = (int)min((long long)SPLIT_ROWS, b.num_rows - r0);
  for (int i = threadIdx.x; i < rows * b.groups; i += SPLIT_THREADS) {
    const int r = i / b.groups, k = i - r * b.groups;
    const uint64_t c = load_code(b.codes, b.ids_type, (r0 + r) * b.codes_stride + k);
    code[r * pitch + k] = c < (uint64_t)a.vocab[k] ? (uint32_t)c : DROPPED;
  }
  __syncthreads();
  const int lane = threadIdx.x % 32;
  if (lane >= rows) return;
  const uint32_t* mine = code + lane * pitch;
  bool ok = true;
  for (int k = 0; k < b.groups; ++k) ok = ok && mine[k] != DROPPED;
  for (int k = threadIdx.x / 32; k < groups; k += SPLIT_THREADS / 32)
    a.work[k].keys[r0 + lane] = !ok ? DROPPED : k == b.groups ? 0 : kept(a, mine[k]);
}

// The BATCH keys k, k + 32, ... below k1 of group g: the codes of those rows, or
// DROPPED.  DIRECT: one group, whose keys are the codes themselves.  The type is
// looked at once, so that the loads do not wait for one another.
template <class Code>
__device__ __forceinline__ void load_codes(const GradArgs& a, long long k, long long k1,
                                           uint64_t (&c)[BATCH]) {
#pragma unroll
  for (int j = 0; j < BATCH; ++j)
    c[j] = k + j * 32 < k1
               ? __ldg(static_cast<const Code*>(a.b.codes) + (k + j * 32) * a.b.codes_stride)
               : ~0ull;
}

template <bool DIRECT>
__device__ __forceinline__ void load_keys(const GradArgs& a, int g, long long k, long long k1,
                                          uint32_t (&key)[BATCH]) {
  if (!DIRECT) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      key[j] = k + j * 32 < k1 ? __ldcg(a.work[g].keys + k + j * 32) : DROPPED;
    return;
  }
  uint64_t c[BATCH];
  if (a.b.ids_type == Q3S_IDS_I64)
    load_codes<unsigned long long>(a, k, k1, c);
  else if (a.b.ids_type == Q3S_IDS_U32)
    load_codes<uint32_t>(a, k, k1, c);
  else
    load_codes<uint16_t>(a, k, k1, c);
#pragma unroll
  for (int j = 0; j < BATCH; ++j) key[j] = c[j] < (uint64_t)a.vocab[g] ? kept(a, c[j]) : DROPPED;
}

// Bound by the issue of the warps that look at every key of the group: 12.7 us for
// 16384 keys and 98 buckets, 8.6 us for 16 groups of 4096, 18 us for 16 groups of 32768 in
// clusters of four.  One block takes a multiprocessor, so beyond 148 buckets of 1024
// codes there is a second wave over all keys.  A radix sort of clusters that exchange
// their digits' totals lost 24 us of 26 to the exchange and to a second wave; this one
// tells only 1024 counts once.  Lanes with one code find each other by a ballot
// for each bit: the instruction that matches lanes by value answers 0.9 lanes a
// clock and multiprocessor, eleven ballots take 2.9 clocks.
//
// MANY: more than one block a cluster.
template <bool DIRECT, bool MANY>
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(const GradArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = MANY ? (int)cluster.num_blocks() : 1;
  const int block = MANY ? (int)cluster.block_rank() : 0;
  const int g = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int bucket = 1 << a.bucket_bits, vocab = a.vocab[g];
  const int buckets = (int)(((long long)vocab + bucket - 1) >> a.bucket_bits);
  admit_next();
  if ((int)blockIdx.x / blocks >= buckets) return;  // the whole cluster
  const GroupWork& w = a.work[g];
  extern __shared__ uint32_t smem[];
  uint32_t* list = smem + (threadIdx.x / 32) * LIST;  // this warp's
  uint32_t* hist = smem + SORT_WARPS * LIST;          // [SORT_WARPS][bucket]
  __shared__ uint32_t sums[2][SORT_WARPS];
  __shared__ uint32_t total[MAX_BUCKET + 1];  // this block's keys per code, and below the bucket
  const uint32_t v0 = blockIdx.x / blocks << a.bucket_bits;
  uint32_t* mine = hist + (warp << a.bucket_bits);
  for (int i = threadIdx.x; i < SORT_WARPS << a.bucket_bits; i += SORT_THREADS) hist[i] = 0;
  if (!DIRECT) await_inputs();
  for (long long i = blockIdx.x * (long long)SORT_THREADS + threadIdx.x; i < a.slots;
       i += (long long)buckets * blocks * SORT_THREADS)
    w.arrived[i] = 0;
  __syncthreads();
  // Every warp counts consecutive rows: its bucket's codes, and all below.
  const long long n = a.b.num_rows;
  const long long per_warp = ((n + blocks * SORT_WARPS - 1) / (blocks * SORT_WARPS) + 31) / 32 * 32;
  const long long k0 = min(n, (block * SORT_WARPS + warp) * per_warp), k1 = min(n, k0 + per_warp);
  // The keys of the bucket go to a list, code in the bucket and row from k0 on,
  // so that they need not be looked for twice; a warp that finds more than the
  // list holds reads its rows again.
  uint32_t below = 0;
  int found = 0;
  for (long long k = k0; k < k1; k += 32 * BATCH) {
    uint32_t key[BATCH];
    load_keys<DIRECT>(a, g, k + lane, k1, key);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      below += key[j] < v0;
      const uint32_t digit = key[j] - v0;
      const bool keep = digit < (uint32_t)bucket;
      const unsigned hits = __ballot_sync(0xFFFFFFFFu, keep);
      const int at = found + __popc(hits & ((1u << lane) - 1));
      if (keep) {
        atomicAdd(&mine[digit], 1u);
        if (at < LIST) list[at] = digit | (uint32_t)(k + j * 32 + lane - k0) << MAX_BUCKET_BITS;
      }
      found += __popc(hits);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xFFFFFFFFu, below, o);
  if (lane == 0) sums[0][warp] = below;
  __syncthreads();
  // Thread t takes code t of the bucket.
  const int d = threadIdx.x;
  if (d < bucket) {
    uint32_t here = 0;
    for (int j = 0; j < SORT_WARPS; ++j) here += hist[(j << a.bucket_bits) + d];
    total[d] = here;
  }
  if (d == 0) {
    uint32_t sum = 0;
    for (int j = 0; j < SORT_WARPS; ++j) sum += sums[0][j];
    total[MAX_BUCKET] = sum;
  }
  uint32_t start = 0, all = 0, before = 0;  // `before`: of the code, by lower blocks
  if (MANY) {
    cluster.sync();
    for (int c = 0; c < blocks; ++c) {
      const uint32_t* other = cluster.map_shared_rank(total, c);
      start += other[MAX_BUCKET];
      const uint32_t x = d < bucket ? other[d] : 0;
      all += x;
      if (c < block) before += x;
    }
  } else {
    __syncthreads();
    start = total[MAX_BUCKET];
    if (d < bucket) all = total[d];
  }
  uint32_t incl = all;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, incl, o);
    if (lane >= o) incl += x;
  }
  if (lane == 31) sums[1][warp] = incl;
  __syncthreads();
  start += incl - all;
  for (int j = 0; j < warp; ++j) start += sums[1][j];
  if (d < bucket) {
    uint32_t at = start + before;
    for (int j = 0; j < SORT_WARPS; ++j) {
      const uint32_t x = hist[(j << a.bucket_bits) + d];
      hist[(j << a.bucket_bits) + d] = at;
      at += x;
    }
    if (block == 0 && v0 + d < (uint32_t)vocab) w.range[v0 + d] = make_uint2(start, start + all);
    if (block == 0 && v0 + d == (uint32_t)vocab - 1) *w.count = start + all;
  }
  if (MANY)
    cluster.sync();  // and no block reads another's counts any more
  else
    __syncthreads();
  // The keys in order, 32 at a time: each goes behind those of its code.
  const auto place = [&](uint32_t digit, uint32_t row) {
    const bool keep = digit < (uint32_t)bucket;
    unsigned peers = __ballot_sync(0xFFFFFFFFu, keep);  // the lanes with this lane's code
    if (peers == 0) return;
    for (int i = 0; i < a.bucket_bits; ++i) {
      const unsigned set = __ballot_sync(0xFFFFFFFFu, digit >> i & 1);
      peers &= digit >> i & 1 ? set : ~set;
    }
    const unsigned lower = peers & ((1u << lane) - 1);
    uint32_t at = 0;
    if (keep) {
      at = mine[digit];
      w.rows[at + __popc(lower)] = row;
    }
    __syncwarp();
    if (keep && lower == 0) mine[digit] = at + __popc(peers);
    __syncwarp();
  };
  if (found <= LIST && per_warp <= LIST_ROWS) {
    for (int i = 0; i < found; i += 32) {
      const uint32_t x = i + lane < found ? list[i + lane] : 0;
      place(i + lane < found ? x & (MAX_BUCKET - 1) : DROPPED,
            (uint32_t)k0 + (x >> MAX_BUCKET_BITS));
    }
    return;
  }
  for (long long k = k0; k < k1; k += 32 * BATCH) {
    uint32_t key[BATCH];
    load_keys<DIRECT>(a, g, k + lane, k1, key);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) place(key[j] - v0, (uint32_t)(k + j * 32 + lane));
  }
}

template <int DT>
constexpr int width = DT == Q3S_DTYPE_F32 ? 4 : 2;  // bytes of an element

template <int DT>
__device__ __forceinline__ float load_value(const void* p, long long i) {
  if (DT == Q3S_DTYPE_F32) return static_cast<const float*>(p)[i];
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

template <int DT>
__device__ __forceinline__ void store_value(void* p, long long i, float x) {
  if (DT == Q3S_DTYPE_F32)
    static_cast<float*>(p)[i] = x;
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Loads VE columns (at most 16 bytes).
template <int DT, int VE>
__device__ __forceinline__ void load_vec(const void* base, long long i, float* x) {
  constexpr int BYTES = VE * width<DT>;
  const char* p = static_cast<const char*>(base) + i * width<DT>;
  uint32_t w[4] = {};
  if (BYTES == 16) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  } else if (BYTES == 8) {
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = q.x, w[1] = q.y;
  } else if (BYTES == 4) {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else {
    w[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
  }
#pragma unroll
  for (int e = 0; e < VE; ++e)
    x[e] = DT == Q3S_DTYPE_F32 ? __uint_as_float(w[e % 4])
                               : __uint_as_float(e & 1 ? w[e / 2 % 4] & 0xFFFF0000u : w[e / 2 % 4] << 16);
}

// Stores VE columns (at most 16 bytes), written once and not read again here.
template <int DT, int VE>
__device__ __forceinline__ void store_vec(void* base, long long i, const float* x) {
  if (DT == Q3S_DTYPE_F32) {
    float* p = static_cast<float*>(base) + i;
    if (VE == 4)
      __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
    else if (VE == 2)
      __stcs(reinterpret_cast<float2*>(p), make_float2(x[0], x[1]));
    else
      __stcs(p, x[0]);
  } else {
    uint16_t* p = static_cast<uint16_t*>(base) + i;
    if (VE == 8)
      __stcs(reinterpret_cast<uint4*>(p),
             make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]),
                        pack_bf16(x[6], x[7])));
    else if (VE == 4)
      __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])));
    else if (VE == 2)
      __stcs(reinterpret_cast<uint32_t*>(p), pack_bf16(x[0], x[1]));
    else
      p[0] = __bfloat16_as_ushort(__float2bfloat16_rn(x[0]));
  }
}

// The COLS sums of a lane.
template <int COLS>
struct Sums {
  float x[COLS];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < COLS; ++i) x[i] = 0.0f;
  }
  // Adds a row's columns: words as they lie in memory, of type DT.  A bf16 is
  // added to an f32 in one instruction, rounded once.
  template <int DT, int WORDS>
  __device__ __forceinline__ void add(const uint32_t (&w)[WORDS]) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if (DT == Q3S_DTYPE_BF16)
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
            "add.rn.f32.bf16 %0, lo, %0;\n\tadd.rn.f32.bf16 %1, hi, %1;\n\t}"
            : "+f"(x[2 * i % COLS]), "+f"(x[(2 * i + 1) % COLS])
            : "r"(w[i]));
      else
        x[i % COLS] = __fadd_rn(x[i % COLS], __uint_as_float(w[i]));
    }
  }
};

// WORDS words of shared memory at address p.
template <int WORDS>
__device__ __forceinline__ void read_words(uint32_t* w, uint32_t p) {
  if (WORDS == 4)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1 % WORDS]), "=r"(w[2 % WORDS]), "=r"(w[3 % WORDS])
                 : "r"(p)
                 : "memory");
  else if (WORDS == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1 % WORDS]) : "r"(p) : "memory");
  else
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(p) : "memory");
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const char* src) {
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES)
                 : "memory");
}

// A warp's tile of a row: lane l holds NV vectors of VE columns, the j-th at
// column (j * 32 + l) * VE of the tile, so that every copy is contiguous.
template <int IN_, int VE_, int NV_>
struct Tile {
  static constexpr int IN = IN_, VE = VE_, NV = NV_;
  static constexpr int COLS = NV * VE;  // per lane
  static constexpr int BYTES = VE * width<IN>;
  static constexpr int SLOT = 32 * NV * BYTES;
  static constexpr int RING = NV * BYTES > 32 ? 4 : 8;  // rows in flight
  static constexpr bool ASYNC = BYTES >= 4;  // else loads through registers
  static constexpr int SMEM = ASYNC ? REDUCE_WARPS * RING * SLOT : 0;
};

// The rows at positions [k0, k1) of the sorted list, one after another, RING of
// them in flight.  Every lane copies its own columns into its own part of the
// warp's ring and reads them back, so nothing but the copies themselves is
// waited for.
template <class T>
struct Rows {
  const uint32_t* rows;
  const char* base;   // of this lane's columns
  long long stride;   // bytes
  uint32_t ring;      // this lane's part, an address in shared memory
  uint32_t issued, k1;
  uint32_t window, next;  // row numbers of 32 positions, one a lane, and of the 32 after
  uint32_t taken;         // rows: of the window, and into the ring
  bool there[T::NV];      // columns of this lane's vectors
  // Without copies: the next rows' columns, and the rows taken from them.
  static constexpr int HELD = T::ASYNC ? 1 : 4;
  uint16_t held[HELD][T::NV];
  uint32_t used;

  __device__ __forceinline__ Rows(const q3s_embed_grad_batch& b, const uint32_t* rows_,
                                  uint32_t k0, uint32_t k1_, int col, char* ring_)
      : rows(rows_), issued(k0), k1(k1_), window(0), taken(0), used(0) {
    const int lane = threadIdx.x % 32;
    base = static_cast<const char*>(b.grad_out) + (long long)col * width<T::IN>;
    stride = b.grad_stride * width<T::IN>;
    ring = (uint32_t)__cvta_generic_to_shared(ring_) + lane * T::BYTES;
    next = k0 + lane < k1 ? __ldcg(rows + k0 + lane) : 0;
#pragma unroll
    for (int j = 0; j < T::NV; ++j) there[j] = col + j * 32 * T::VE < b.hidden;
    if (T::ASYNC)
#pragma unroll 1
      for (int i = 0; i < T::RING - 1; ++i) issue();
  }
  __device__ __forceinline__ const char* source() {
    if (taken % 32 == 0) {
      window = next;
      const uint32_t q = issued + 32 + threadIdx.x % 32;
      next = q < k1 ? __ldcg(rows + q) : 0;
    }
    const uint32_t row = __shfl_sync(0xFFFFFFFFu, window, taken % 32);
    ++issued;
    return base + row * stride;
  }
  __device__ __forceinline__ void issue() {
    if (issued < k1) {
      const char* src = source();
      const uint32_t dst = ring + taken % T::RING * T::SLOT;
#pragma unroll
      for (int j = 0; j < T::NV; ++j)
        if (there[j]) copy_async<T::BYTES>(dst + j * 32 * T::BYTES, src + j * 32 * T::BYTES);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ++taken;
  }
  // acc += the next row.
  __device__ __forceinline__ void add(Sums<T::COLS>& acc) {
    if constexpr (T::ASYNC) {
      issue();
      asm volatile("cp.async.wait_group %0;" ::"n"(T::RING - 1) : "memory");
      constexpr int WORDS = T::BYTES / 4;
      uint32_t w[T::NV * WORDS];
#pragma unroll
      for (int j = 0; j < T::NV; ++j)
        read_words<WORDS>(w + j * WORDS, ring + taken % T::RING * T::SLOT + j * 32 * T::BYTES);
      acc.template add<T::IN>(w);
    } else {  // single bf16 columns: HELD rows are asked for at a time
      const int at = (int)(used++ % HELD);
      if (at == 0) fetch();
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        if (h != at) continue;
        uint32_t w[T::NV];
#pragma unroll
        for (int j = 0; j < T::NV; ++j) w[j] = (uint32_t)held[h][j] << 16;
        acc.template add<Q3S_DTYPE_F32>(w);
      }
    }
  }
  __device__ __forceinline__ void fetch() {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      if (issued >= k1) break;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(source());
#pragma unroll
      for (int j = 0; j < T::NV; ++j) held[h][j] = there[j] ? __ldg(src + j * 32) : 0;
      ++taken;
    }
  }
};

// Writes the sum of code v and clears it; `empty`: the code has no rows.  All
// lanes of the warp take part.
template <class T, int OUT>
__device__ __forceinline__ void finish(const GradArgs& a, int g, long long v, int col, bool empty,
                                       Sums<T::COLS>& sums) {
  const q3s_embed_grad_batch& b = a.b;
  const bool text = g == b.groups;
  const bool keep = b.accumulate && !text;
  if (empty && keep) return;
  float(&acc)[T::COLS] = sums.x;
  const float scale = text ? 1.0f : b.scale;
  const int lane = threadIdx.x % 32;
  // Eight bf16 columns a lane become f32 as two vectors of four: lanes trade
  // them so that each store of the warp is contiguous.
  constexpr bool TRADE = OUT == Q3S_DTYPE_F32 && T::VE == 8;
  constexpr int SE = TRADE ? 4 : T::VE;
  if constexpr (TRADE) {
    if (!empty) {
#pragma unroll
      for (int j = 0; j < T::NV; ++j) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int from = (i / 4 * 32 + lane) / 2;
          const float even = __shfl_sync(0xFFFFFFFFu, acc[j * 8 + i % 4], from);
          const float odd = __shfl_sync(0xFFFFFFFFu, acc[j * 8 + 4 + i % 4], from);
          y[i] = lane & 1 ? odd : even;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j * 8 + i] = y[i];
      }
    }
  }
  const int c0 = col - lane * (T::VE - SE);
  char* out = static_cast<char*>(a.grads[g]) + (v * b.hidden + c0) * width<OUT>;
#pragma unroll
  for (int j = 0; j < T::COLS / SE; ++j) {
    if (c0 + j * 32 * SE < b.hidden) {
      float x[SE];
#pragma unroll
      for (int e = 0; e < SE; ++e) {
        x[e] = __fmul_rn(acc[j * SE + e], scale);
        if (keep) x[e] = __fadd_rn(load_value<OUT>(out, j * 32 * SE + e), x[e]);
      }
      store_vec<OUT, SE>(out, j * 32 * SE, x);
    }
  }
  if (!empty) sums.clear();
}

// The pieces of long runs (longer than two blocks of the sorted list) in one
// block: slot 0 belongs to the run that holds the block's first position, slot
// 1 to a run that starts inside the block and leaves it.  The warp that
// finishes the last of JOIN pieces adds them up in order, and the one that finishes
// the last of these groups the groups' sums.  (Groups of 8 or 32 instead of 16 change no
// case by more than 0.5 us.  When pieces were 128 rows, 256 of them one after another
// took 110 us, in groups of 16 40 us.)
template <class T, int OUT>
__device__ __forceinline__ void add_pieces(const GradArgs& a, int g, long long block, int tile,
                                           char* ring) {
  const q3s_embed_grad_batch& b = a.b;
  const int lane = threadIdx.x % 32, col = tile * 32 * T::COLS + lane * T::VE;
  const GroupWork& w = a.work[g];
  const uint32_t n = *w.count;
  const long long first = block * a.block;
  if (first >= n) return;
  const uint32_t k0 = (uint32_t)first, k1 = (uint32_t)min((long long)n, first + a.block);
  uint2 done = make_uint2(0, 0);
  for (int slot = 0; slot < 2; ++slot) {
    const uint32_t row = w.rows[slot ? k1 - 1 : k0];
    const uint32_t code = g == b.groups ? 0 : (uint32_t)load_code(b.codes, b.ids_type,
                                                                  row * b.codes_stride + g);
    const uint2 run = w.range[code];
    if (slot && run.x == done.x) return;
    done = run;
    if (run.y - run.x <= 2u * a.block) continue;
    Sums<T::COLS> sums;
    sums.clear();
    const uint32_t from_row = max(k0, run.x), to_row = min(k1, run.y);
    Rows<T> list(b, w.rows, from_row, to_row, col, ring);
    for (uint32_t k = from_row; k < to_row; ++k) list.add(sums);
    const long long from = run.x / a.block, to = (run.y - 1) / a.block;
    const bool inside = run.x > from * a.block;  // the first piece is in slot 1
    const auto place = [&](long long k) { return (k * 2 + (k == from && inside)) * a.tiles + tile; };
    // A lane's sums as vectors of four side by side: the warp that joins the
    // pieces holds the same columns.
    constexpr int PIECE = 8 * T::COLS;  // vectors of a warp
    // Hands the sums over at piece k; whether `want` warps had handed theirs over,
    // counted in units of `one` at piece `at`, before.
    const auto hand_over = [&](long long k, long long at, uint32_t one, uint32_t want) {
      float4* out = w.partial + place(k) * PIECE + lane;
#pragma unroll
      for (int i = 0; i < T::COLS / 4; ++i)
        out[i * 32] = make_float4(sums.x[4 * i], sums.x[4 * i + 1], sums.x[4 * i + 2], sums.x[4 * i + 3]);
      __threadfence();
      __syncwarp();
      uint32_t before = 0;
      if (lane == 0) before = atomicAdd(w.arrived + place(at), one);
      before = __shfl_sync(0xFFFFFFFFu, before, 0);
      const bool last = (one == 1 ? before % GROUPS : before / GROUPS) == want;
      if (last) __threadfence();
      return last;
    };
    const auto join = [&](long long k0, long long k1, int step) {
      sums.clear();
#pragma unroll 1
      for (long long k = k0; k <= k1; k += step) {
        const float4* p = w.partial + place(k) * PIECE + lane;
        uint32_t x[T::COLS];
#pragma unroll
        for (int i = 0; i < T::COLS / 4; ++i) {
          const float4 q = __ldcg(p + i * 32);
          x[4 * i] = __float_as_uint(q.x), x[4 * i + 1] = __float_as_uint(q.y);
          x[4 * i + 2] = __float_as_uint(q.z), x[4 * i + 3] = __float_as_uint(q.w);
        }
        sums.template add<Q3S_DTYPE_F32>(x);
      }
    };
    const long long start = block - (block - from) % JOIN, end = min(to, start + JOIN - 1);
    if (!hand_over(block, start, 1, (uint32_t)(end - start))) continue;
    join(start, end, 1);
    if (to - from >= JOIN) {
      if (!hand_over(start, from, GROUPS, (uint32_t)((to - from) / JOIN))) continue;
      join(from, to, JOIN);
    }
    finish<T, OUT>(a, g, code, col, false, sums);
  }
}

// Counters of single cold launches.  A large table is bound by HBM (16384 rows of 1024
// bf16 into 100003 rows of f32, most of them zeros: 77 us, 5.0 TB/s with the launch and
// the tail in it).  Codes with two rows each, in L2, are bound by issue (16 groups of
// 4096 rows of 2048 bf16: 47 us, 57 % of the slots, 220 instructions of a warp for a
// row's 1024 columns).  With more rows than L2 keeps nothing is full (16 groups of 32768
// rows of 1024 bf16, 1.07 GB gathered: 136 us, HBM at 3.0 TB/s, 52 % hits in L2 and 37 %
// of its throughput, issue 44 %, 15 of 20 warps at work): the gathers' latency and the
// tail are what is left.
//
// Whole calls, that last case and the one before: rings of 8 rows of 64 bytes a lane
// 187 and 61 us instead of 151 and 50 with 4; four blocks a multiprocessor 172 and 52,
// six 151 and 49; 16 columns a lane 175 and 56.  A bf16 added to an f32 in one
// instruction took 228 to 211 and 71 to 64 us at that step.  Sums by matrix
// instructions with a selection matrix are not open: 0 times an infinity of another row
// would be NaN.
//
// A warp takes the pieces in one block of the sorted list, or the runs of a
// chunk of consecutive codes, for one tile of columns.  The codes' runs lie one
// after another in the sorted list, so the warp streams their rows with many
// of them in flight across the ends of runs: with one code per warp, each
// paid the latency of its range, its row numbers and its rows in turn.
template <class T, int OUT>
__global__ void __launch_bounds__(REDUCE_THREADS, 5) reduce_kernel(const GradArgs a) {
  extern __shared__ __align__(16) char rings[];
  const q3s_embed_grad_batch& b = a.b;
  await_inputs();
  const int g = blockIdx.y, lane = threadIdx.x % 32;
  char* ring = rings + (T::ASYNC ? threadIdx.x / 32 * (T::RING * T::SLOT) : 0);
  const long long warp = (long long)blockIdx.x * REDUCE_WARPS + threadIdx.x / 32;
  const long long unit = warp / a.tiles;  // a row's tiles lie side by side
  const int tile = (int)(warp - unit * a.tiles);
  if (unit < a.blocks) {
    add_pieces<T, OUT>(a, g, unit, tile, ring);
    return;
  }
  const long long v0 = (unit - a.blocks) * a.chunk;
  if (v0 >= a.vocab[g]) return;
  const int col = tile * 32 * T::COLS + lane * T::VE;
  const int codes = (int)min((long long)a.chunk, a.vocab[g] - v0);
  const GroupWork& w = a.work[g];
  const uint2 run = lane < codes ? w.range[v0 + lane] : make_uint2(0, 0);
  const unsigned used = __ballot_sync(0xFFFFFFFFu, run.y > run.x);
  const unsigned pieces = __ballot_sync(0xFFFFFFFFu, run.y - run.x > 2u * a.block);
  Sums<T::COLS> sums;
  sums.clear();
  int t = 0;
  while (t < codes) {
    // The codes up to the next one whose run comes in pieces.
    const unsigned later = pieces >> t << t;
    const int stop = later ? __ffs(later) - 1 : codes;
    const unsigned mine = used & (stop == 32 ? 0xFFFFFFFFu : (1u << stop) - 1) & ~((1u << t) - 1);
    const uint32_t k0 = mine ? __shfl_sync(0xFFFFFFFFu, run.x, __ffs(mine) - 1) : 0;
    const uint32_t k1 = mine ? __shfl_sync(0xFFFFFFFFu, run.y, 31 - __clz(mine)) : 0;
    Rows<T> list(b, w.rows, k0, k1, col, ring);
#pragma unroll 1
    for (; t < stop; ++t) {
      const uint32_t n = __shfl_sync(0xFFFFFFFFu, run.y - run.x, t);
#pragma unroll 1
      for (uint32_t k = 0; k < n; ++k) list.add(sums);
      finish<T, OUT>(a, g, v0 + t, col, n == 0, sums);
    }
    ++t;  // the run in pieces is written by add_pieces
  }
}

// The gradient of a text operand per row: grad_out, or zeros where the row is
// not valid.  A warp a row: a lane looks at each of its codes, and four vectors a
// lane are in flight.  Bound by HBM: 4096 rows of 2048 bf16 5.4 us (5.1 us at the copy
// rate; 13.5 us with a block a row and single columns), 32768 of 1024 to f32 40 us (31).
template <int IN, int OUT, int VE>
__global__ void __launch_bounds__(TEXT_THREADS) text_kernel(const GradArgs a) {
  constexpr int AHEAD = 4, SE = OUT == Q3S_DTYPE_F32 && VE == 8 ? 4 : VE;
  const q3s_embed_grad_batch& b = a.b;
  const int lane = threadIdx.x % 32, vectors = b.hidden / VE;
  const long long warps = (long long)gridDim.x * (TEXT_THREADS / 32);
  for (long long r = blockIdx.x * (TEXT_THREADS / 32ll) + threadIdx.x / 32; r < b.num_rows; r += warps) {
    const bool valid = __all_sync(
        0xFFFFFFFFu, lane >= b.groups || load_code(b.codes, b.ids_type, r * b.codes_stride + lane) <
                                             (uint64_t)a.vocab[lane]);
    const char* src = static_cast<const char*>(b.grad_out) + r * b.grad_stride * width<IN>;
    char* dst = static_cast<char*>(b.text_grad) + r * b.text_stride * width<OUT>;
    for (int v0 = lane; v0 < vectors; v0 += 32 * AHEAD) {
      float x[AHEAD][VE];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[j][e] = 0.0f;
        if (v0 + j * 32 < vectors && valid) load_vec<IN, VE>(src, (v0 + j * 32) * VE, x[j]);
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (v0 + j * 32 >= vectors) break;
#pragma unroll
        for (int e = 0; e < VE; e += SE) store_vec<OUT, SE>(dst, (v0 + j * 32) * VE + e, x[j] + e);
      }
    }
  }
}

// A launch in clusters (cluster > 1), and with `early` one that may start while
// the kernel before it in the stream still runs: it waits at await_inputs().  The
// one before lets it with admit_next(), when all its blocks are resident.
template <class Kernel>
cudaError_t launch_after(Kernel kernel, dim3 grid, int threads, int smem, cudaStream_t st,
                         bool early, int cluster, const GradArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (early) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

int bad(const char* msg) {
  return record_error(Q3S_E_INVALID_ARGUMENT, std::string("q3s_embed_grad: ") + msg);
}

// Whether two of the call's outputs share memory: two groups would write, or with
// accumulate read and write, the same table at the same time.
bool overlapping(const q3s_embed_grad_batch* b, int width) {
  struct Span {
    uintptr_t start;
    uint64_t bytes;
  } spans[Q3S_MAX_CODE_GROUPS + 1];
  int n = 0;
  for (; n < b->groups; ++n)
    spans[n] = {reinterpret_cast<uintptr_t>(b->grads[n]), (uint64_t)b->vocab[n] * b->hidden * width};
  if (b->text_grad && (b->text_stride == 0 || b->num_rows > 0)) {
    const uint64_t before = b->text_stride ? (uint64_t)(b->num_rows - 1) * b->text_stride : 0;
    spans[n++] = {reinterpret_cast<uintptr_t>(b->text_grad), (before + b->hidden) * width};
  }
  const auto before = [](const Span& x, const Span& y) { return x.start < y.start; };
  if (!std::is_sorted(spans, spans + n, before)) std::sort(spans, spans + n, before);
  for (int k = 1; k < n; ++k)
    if (spans[k].start - spans[k - 1].start < spans[k - 1].bytes) return true;
  return false;
}

int check(const q3s_embed_grad_batch* b) {
  if (b->num_rows < 0 || b->num_rows > 0x7FFFFFFF) return bad("num_rows must be in 0..2^31 - 1");
  if ((b->dtype != Q3S_DTYPE_F32 && b->dtype != Q3S_DTYPE_BF16) ||
      (b->grads_dtype != Q3S_DTYPE_F32 && b->grads_dtype != Q3S_DTYPE_BF16))
    return bad("dtype and grads_dtype must be Q3S_DTYPE_F32 or Q3S_DTYPE_BF16");
  if (b->ids_type != Q3S_IDS_U16 && b->ids_type != Q3S_IDS_U32 && b->ids_type != Q3S_IDS_I64)
    return bad("unknown ids_type");
  if (b->groups < 1 || b->groups > Q3S_MAX_CODE_GROUPS) return bad("groups must be in 1..32");
  if (b->hidden < 1 || b->hidden > MAX_HIDDEN) return bad("hidden must be in 1..2^30");
  if (!b->grads || !b->vocab) return bad("grads and vocab are required");
  if (b->num_rows > 0) {
    if (!b->codes || !b->grad_out) return bad("codes and grad_out are required");
    if (b->codes_stride < b->groups) return bad("codes_stride must be >= groups");
    if (b->grad_stride != 0 && b->grad_stride < b->hidden)
      return bad("grad_stride must be 0 or >= hidden");
  }
  if (b->text_grad && b->text_stride != 0 && b->text_stride < b->hidden)
    return bad("text_stride must be 0 or >= hidden");
  const int in = b->dtype == Q3S_DTYPE_F32 ? 4 : 2, out = b->grads_dtype == Q3S_DTYPE_F32 ? 4 : 2;
  const int id = b->ids_type == Q3S_IDS_U16 ? 2 : b->ids_type == Q3S_IDS_U32 ? 4 : 8;
  const auto off = [](const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
  if (off(b->codes, id) || off(b->grad_out, in) || off(b->text_grad, out))
    return bad("codes, grad_out and text_grad must be aligned to their elements");
  for (int g = 0; g < b->groups; ++g) {
    if (!b->grads[g]) return bad("a gradient table is NULL");
    if (off(b->grads[g], out)) return bad("a gradient table is not aligned to its elements");
    if (b->vocab[g] < 1) return bad("a codebook vocabulary is < 1");
  }
  // The sort looks at every key once for each 1024 ids: 0.43 s at this bound (2^24 rows,
  // as many ids), and in proportion beyond it, without end for what the types hold.
  uint64_t ids = 0;
  for (int g = 0; g < b->groups; ++g) ids += (uint64_t)b->vocab[g];
  if (b->num_rows && ids > (1ull << 48) / (uint64_t)b->num_rows)
    return bad("num_rows times the sum of vocab must be at most 2^48");
  if (overlapping(b, out)) return bad("the gradients must not overlap one another");
  return Q3S_OK;
}

// Whole vectors of `bytes` start on their own size in every row of p.
bool aligned(const void* p, long long stride_bytes, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride_bytes % bytes == 0;
}

template <class T, int OUT>
cudaError_t launch_sums(const GradArgs& a, int groups, int max_vocab, int device,
                        cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem((const void*)reduce_kernel<T, OUT>, T::SMEM, device, allowed);
  if (e != cudaSuccess) return e;
  const long long warps = (a.blocks + ((long long)max_vocab + a.chunk - 1) / a.chunk) * a.tiles;
  const dim3 grid((unsigned)((warps + REDUCE_WARPS - 1) / REDUCE_WARPS), groups);
  const cudaError_t l = launch_after(reduce_kernel<T, OUT>, grid, REDUCE_THREADS, T::SMEM, st, true, 0, a);
  if (l != cudaSuccess) return l;
  if (a.b.text_grad && a.b.text_stride && a.b.num_rows) {
    const long long blocks = (a.b.num_rows + TEXT_THREADS / 32 - 1) / (TEXT_THREADS / 32);
    const int grid = (int)(blocks < 65536 ? blocks : 65536);
    constexpr int BYTES = T::VE * width<OUT>;
    if (aligned(a.b.text_grad, a.b.text_stride * width<OUT>, BYTES < 16 ? BYTES : 16))
      text_kernel<T::IN, OUT, T::VE><<<grid, TEXT_THREADS, 0, st>>>(a);
    else
      text_kernel<T::IN, OUT, 1><<<grid, TEXT_THREADS, 0, st>>>(a);
  }
  return cudaGetLastError();
}

// Columns per vector: 16 bytes where rows, their stride, the tables and H allow
// them and fill a warp, else pairs, else single elements.
int vector_columns(const GradArgs& a, int groups) {
  const q3s_embed_grad_batch& b = a.b;
  const int in = b.dtype == Q3S_DTYPE_F32 ? 4 : 2, out = b.grads_dtype == Q3S_DTYPE_F32 ? 4 : 2;
  const auto fits = [&](int ve) {
    bool ok = b.hidden % ve == 0 && aligned(b.grad_out, b.grad_stride * in, ve * in);
    for (int g = 0; g < groups; ++g)
      ok = ok && aligned(a.grads[g], (long long)b.hidden * out, ve * out < 16 ? ve * out : 16);
    return ok;
  };
  const int wide = 16 / in;
  return b.hidden >= 32 * wide && fits(wide) ? wide : fits(2) ? 2 : 1;
}

template <bool DIRECT, bool MANY>
cudaError_t launch_sort(const GradArgs& a, int groups, int max_vocab, int cluster, int device,
                        cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem((const void*)sort_kernel<DIRECT, MANY>,
                                   SORT_WARPS * 4 * (LIST + MAX_BUCKET), device, allowed);
  if (e != cudaSuccess) return e;
  const int buckets = (int)(((long long)max_vocab + (1 << a.bucket_bits) - 1) >> a.bucket_bits);
  return launch_after(sort_kernel<DIRECT, MANY>, dim3(buckets * cluster, groups), SORT_THREADS,
                      SORT_WARPS * 4 * (LIST + (1 << a.bucket_bits)), st, !DIRECT, cluster, a);
}

int embed_grad(q3s_context* ctx, const q3s_embed_grad_batch* b, void* stream) {
  if (!ctx || !b) return bad("NULL context or batch");
  int rc = check(b);
  if (rc != Q3S_OK) return rc;
  GradArgs a;
  a.b = *b;
  const bool text_sum = b->text_grad && b->text_stride == 0;
  const int groups = b->groups + (text_sum ? 1 : 0);
  int max_vocab = 1;
  for (int g = 0; g < groups; ++g) {
    a.grads[g] = g < b->groups ? b->grads[g] : b->text_grad;
    a.vocab[g] = g < b->groups ? b->vocab[g] : 1;
    if (a.vocab[g] > max_vocab) max_vocab = a.vocab[g];
  }
  const ContextInfo ci = context_info(ctx);
  DeviceScope scope(ci.device);
  if (scope.err != cudaSuccess) return record_cuda_error(scope.err, "cudaSetDevice");
  // Pieces of about sqrt(rows) / 8 positions, 32 at least: a warp then adds at
  // most two pieces' rows in turn, or JOIN pieces, or the groups of the longest
  // possible run (32 positions, 64, 128: 16 groups of 32768 rows, a few codes frequent,
  // 151, 158 and 164 us; 20000 rows of 1024 f32, one group, 29, 39 and 58 us; every code
  // as frequent, 16 groups of 32768 rows, 120, 116 and 113 us; 16 of 4096, 50, 49, 48).
  // Their sums are most of the workspace: 4 bytes a column, two for every piece that
  // rows can have, 134 MB for the 16 groups of 32768 rows of 1024.
  a.block = 32;
  while (64LL * a.block * a.block < b->num_rows) a.block *= 2;
  const int ve = vector_columns(a, groups);
  // As many 16-byte vectors a lane, up to four, as leave no lane idle (what a row
  // costs besides its columns is then shared by more of them: at most two instead of
  // four, 50 -> 56 us for 16 groups of 4096 rows of 2048 bf16, 151 -> 175 us for 32768 of
  // 1024, 29 -> 27 us for 20000 rows of 1024 f32, no difference for text).
  const int nv = ve * (b->dtype == Q3S_DTYPE_F32 ? 4 : 2) < 16 ? 8 / ve
                 : b->hidden > 64 * ve                         ? 4
                 : b->hidden > 32 * ve                         ? 2
                                                               : 1;
  const int tile = 32 * ve * nv;
  a.tiles = (b->hidden + tile - 1) / tile;
  // The sort's clusters: as many blocks as leave each 4096 rows, as long as there
  // is a bucket size with which all blocks find a multiprocessor (16 groups of 32768
  // rows: 151 us, 155 us in single blocks; 16 groups of 4096: 50 us, 55 us with clusters
  // from 1024 rows a block on).
  long long all = 0;
  for (int g = 0; g < groups; ++g) all += a.vocab[g];
  const auto sort_blocks = [&](int bits, int cluster) {
    long long n = 0;
    for (int g = 0; g < groups; ++g) n += ((long long)a.vocab[g] + (1 << bits) - 1) >> bits;
    return n * cluster;
  };
  int cluster = MAX_CLUSTER;
  while (cluster > 1 && (b->num_rows < 4096LL * cluster ||
                         sort_blocks(MAX_BUCKET_BITS, cluster) > ci.sm_count))
    cluster /= 2;
  a.bucket_bits = 5;
  while (a.bucket_bits < MAX_BUCKET_BITS && sort_blocks(a.bucket_bits, cluster) > ci.sm_count)
    ++a.bucket_bits;
  // Codes per warp: as many as leave two warps for every place on the device
  // (32 a multiprocessor).  One code a warp: 16384 rows into 100003 codes 84 -> 90 us, 16
  // groups of 4096 50 -> 71 us; an eighth of the warps: 102 and 59 us.
  const long long units = all * a.tiles;
  const long long chunk = units / (2LL * 32 * ci.sm_count);
  a.chunk = chunk < 1 ? 1 : chunk > 32 ? 32 : (int)chunk;
  // ... but not so many that the rows of a warp, on average, exceed 64: a bound on what
  // one warp still has to do when the others are done (16 groups of 32768 rows 151 us
  // with and without it).
  while (a.chunk > 1 && a.chunk * b->num_rows > 64LL * max_vocab) a.chunk /= 2;
  a.blocks = b->num_rows > 2 * a.block ? (int)((b->num_rows + a.block - 1) / a.block) : 0;
  a.slots = a.blocks * 2 * a.tiles;
  const size_t partial = align256((size_t)a.blocks * 2 * a.tiles * tile * 4) +
                         align256((size_t)a.slots * 4);
  const size_t list = align256((size_t)b->num_rows * 4);
  size_t need = 0;
  for (int g = 0; g < groups; ++g)
    need += list * (groups > 1 ? 2 : 1) + align256((size_t)a.vocab[g] * sizeof(uint2)) + partial;
  need += align256((size_t)groups * 4);
  unsigned char* p = nullptr;
  std::unique_lock<std::mutex> busy;
  rc = stream_scratch(ctx, stream, need, &p, &busy);
  if (rc != Q3S_OK) return rc;
  for (int g = 0; g < groups; ++g) {
    a.work[g].rows = reinterpret_cast<uint32_t*>(p);
    p += list;
    a.work[g].keys = nullptr;
    if (groups > 1) {
      a.work[g].keys = reinterpret_cast<uint32_t*>(p);
      p += list;
    }
    a.work[g].range = reinterpret_cast<uint2*>(p);
    p += align256((size_t)a.vocab[g] * sizeof(uint2));
    a.work[g].partial = reinterpret_cast<float4*>(p);
    a.work[g].arrived = reinterpret_cast<uint32_t*>(
        p + align256((size_t)a.blocks * 2 * a.tiles * tile * 4));
    p += partial;
  }
  for (int g = 0; g < groups; ++g) a.work[g].count = reinterpret_cast<uint32_t*>(p) + g;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (groups > 1 && b->num_rows) {
    const int blocks = (int)((b->num_rows + SPLIT_ROWS - 1) / SPLIT_ROWS);
    split_kernel<<<blocks, SPLIT_THREADS, 0, st>>>(a, groups);
    if ((e = cudaGetLastError()) != cudaSuccess) return record_cuda_error(e, "split kernel launch");
  }
  const auto sort = [&](auto direct, auto many) {
    return launch_sort<decltype(direct)::value, decltype(many)::value>(a, groups, max_vocab, cluster,
                                                                       ci.device, st);
  };
  const std::true_type yes;
  const std::false_type no;
  e = groups > 1 ? (cluster > 1 ? sort(no, yes) : sort(no, no))
                 : (cluster > 1 ? sort(yes, yes) : sort(yes, no));
  if (e != cudaSuccess) return record_cuda_error(e, "sort kernel launch");
  const bool in32 = b->dtype == Q3S_DTYPE_F32, out32 = b->grads_dtype == Q3S_DTYPE_F32;
  const auto sums = [&](auto type, auto out) {
    constexpr int IN = decltype(type)::value, OUT = decltype(out)::value;
    constexpr int WIDE = IN == Q3S_DTYPE_F32 ? 4 : 8;
    if (ve == WIDE)
      return nv == 4   ? launch_sums<Tile<IN, WIDE, 4>, OUT>(a, groups, max_vocab, ci.device, st)
             : nv == 2 ? launch_sums<Tile<IN, WIDE, 2>, OUT>(a, groups, max_vocab, ci.device, st)
                       : launch_sums<Tile<IN, WIDE, 1>, OUT>(a, groups, max_vocab, ci.device, st);
    if (ve == 2) return launch_sums<Tile<IN, 2, 4>, OUT>(a, groups, max_vocab, ci.device, st);
    return launch_sums<Tile<IN, 1, 8>, OUT>(a, groups, max_vocab, ci.device, st);
  };
  const std::integral_constant<int, Q3S_DTYPE_F32> f32;
  const std::integral_constant<int, Q3S_DTYPE_BF16> bf16;
  e = in32 ? (out32 ? sums(f32, f32) : sums(f32, bf16)) : (out32 ? sums(bf16, f32) : sums(bf16, bf16));
  if (e != cudaSuccess) return record_cuda_error(e, "embedding gradient launch");
  return Q3S_OK;
}

}  // namespace
}  // namespace q3s

extern "C" int q3s_embed_grad(q3s_context* ctx, const q3s_embed_grad_batch* batch, void* stream) {
  return q3s::no_throw([&] { return q3s::embed_grad(ctx, batch, stream); });
}
