// Embedding lookup with scaling (q3s_embed_lookup):
// out[i] = scale * table[ids[i]], the f32 product rounded once.
//
// HBM-bound gather: a row is read (from L2 where ids repeat) and written once.
// 65536 ids into 100003 rows of 1024 bf16, a few ids frequent: 38.4 us, 83 % of the
// copy rate for each table row read once and the output (32 us); 20011 ids into rows
// of 1003 f32, which lie on no vector: 27.7 us (20 us).  16 ids of a decode step: 2.9 us,
// the launch and two accesses one after the other.
#include <cstdint>
#include <string>

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../../include/q3s_sampler.h"
#include "q3s_internal.h"

namespace q3s {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_HIDDEN = 1 << 30;  // 32-bit counters of a row's vectors go somewhat beyond its end

template <int DT>
constexpr int width = DT == Q3S_DTYPE_F32 ? 4 : 2;  // bytes of an element

__device__ __forceinline__ uint64_t load_id(const void* p, int type, long long i) {
  if (type == Q3S_IDS_U16) return __ldg(static_cast<const uint16_t*>(p) + i);
  if (type == Q3S_IDS_U32) return __ldg(static_cast<const uint32_t*>(p) + i);
  return __ldg(static_cast<const unsigned long long*>(p) + i);
}

// VE elements as they lie in memory.
template <int DT, int VE>
struct Raw {
  static constexpr int WORDS = VE * width<DT> < 4 ? 1 : VE * width<DT> / 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const char* p) {
    if (WORDS == 4) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = x.x, w[1 % WORDS] = x.y, w[2 % WORDS] = x.z, w[3 % WORDS] = x.w;
    } else if (WORDS == 2) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = x.x, w[1 % WORDS] = x.y;
    } else if (VE * width<DT> == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      w[0] = __ldg(reinterpret_cast<const uint16_t*>(p));
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

struct LookupArgs {
  q3s_lookup_batch b;
  int vectors;  // of a row
  int lanes;    // lanes per id: the least power of two that covers a row, at most 32
};

// `lanes` lanes take an id and its row, AHEAD vectors of it in flight each (a block
// for each id took 118 us for the 65536 ids, one vector at a time).
// Rows whose starts allow no vector of VE (VE == 1) take single elements.
template <int IN, int OUT, int VE>
__global__ void __launch_bounds__(THREADS) lookup_kernel(const LookupArgs a) {
  constexpr int AHEAD = VE == 1 ? 8 : 4;
  const q3s_lookup_batch& b = a.b;
  const int rank = threadIdx.x & (a.lanes - 1);
  const int per_block = THREADS / a.lanes;
  for (long long i = (long long)blockIdx.x * per_block + threadIdx.x / a.lanes; i < b.num_ids;
       i += (long long)gridDim.x * per_block) {
    const uint64_t id = load_id(b.ids, b.ids_type, i);
    const bool inside = id < (uint64_t)b.vocab;
    const bool zero = !inside || (b.padding_id >= 0 && id == (uint64_t)b.padding_id);
    if (rank == 0) b.status[i] = inside ? Q3S_STATUS_OK : Q3S_STATUS_INVALID_CODE;
    const char* src = static_cast<const char*>(b.table) +
                      (zero ? 0 : (long long)id * b.table_stride) * width<IN>;
    char* dst = static_cast<char*>(b.out) + i * b.out_stride * width<OUT>;
    for (int v0 = rank; v0 < a.vectors; v0 += AHEAD * a.lanes) {
      Raw<IN, VE> x[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int v = v0 + j * a.lanes;
        if (v < a.vectors && !zero) x[j].load(src + (long long)v * (VE * width<IN>));
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int v = v0 + j * a.lanes;
        if (v >= a.vectors) break;
        Raw<OUT, VE> y;
#pragma unroll
        for (int e = 0; e < VE; ++e) y.set(e, zero ? 0.0f : __fmul_rn(x[j].at(e), b.scale));
        y.store(dst + (long long)v * (VE * width<OUT>));
      }
    }
  }
}

template <int IN, int OUT, int VE>
cudaError_t launch(LookupArgs& a, cudaStream_t st) {
  a.vectors = a.b.hidden / VE;
  a.lanes = 1;
  while (a.lanes < 32 && a.lanes < a.vectors) a.lanes *= 2;
  const long long per_block = THREADS / a.lanes;
  const long long blocks = (a.b.num_ids + per_block - 1) / per_block;
  lookup_kernel<IN, OUT, VE><<<(int)(blocks < 0x7FFFFFFF ? blocks : 0x7FFFFFFF), THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

// Elements per vector: what 16 bytes of the wider type hold, where rows start
// on it in both places, else two, else one.
template <int IN, int OUT>
cudaError_t launch_typed(LookupArgs& a, cudaStream_t st) {
  constexpr int WIDE = 16 / (width<IN> > width<OUT> ? width<IN> : width<OUT>);
  const q3s_lookup_batch& b = a.b;
  const auto fits = [&](int ve) {
    return b.hidden % ve == 0 && b.table_stride % ve == 0 && b.out_stride % ve == 0 &&
           reinterpret_cast<uintptr_t>(b.table) % (ve * width<IN>) == 0 &&
           reinterpret_cast<uintptr_t>(b.out) % (ve * width<OUT>) == 0;
  };
  if (fits(WIDE)) return launch<IN, OUT, WIDE>(a, st);
  return fits(2) ? launch<IN, OUT, 2>(a, st) : launch<IN, OUT, 1>(a, st);
}

int bad(const char* msg) {
  return record_error(Q3S_E_INVALID_ARGUMENT, std::string("q3s_embed_lookup: ") + msg);
}

int embed_lookup(q3s_context* ctx, const q3s_lookup_batch* b, void* stream) {
  if (!ctx || !b) return bad("NULL context or batch");
  if (b->num_ids < 0) return bad("num_ids must be >= 0");
  if ((b->dtype != Q3S_DTYPE_F32 && b->dtype != Q3S_DTYPE_BF16) ||
      (b->out_dtype != Q3S_DTYPE_F32 && b->out_dtype != Q3S_DTYPE_BF16))
    return bad("dtype and out_dtype must be Q3S_DTYPE_F32 or Q3S_DTYPE_BF16");
  if (b->ids_type != Q3S_IDS_U16 && b->ids_type != Q3S_IDS_U32 && b->ids_type != Q3S_IDS_I64)
    return bad("unknown ids_type");
  if (b->hidden < 1 || b->hidden > MAX_HIDDEN) return bad("hidden must be in 1..2^30");
  if (b->vocab < 1) return bad("vocab must be >= 1");
  if (b->table_stride < b->hidden || b->out_stride < b->hidden)
    return bad("table_stride and out_stride must be >= hidden");
  if (b->num_ids == 0) return Q3S_OK;
  if (!b->ids || !b->table || !b->out || !b->status)
    return bad("ids, table, out and status are required");
  const ContextInfo ci = context_info(ctx);
  DeviceScope scope(ci.device);
  if (scope.err != cudaSuccess) return record_cuda_error(scope.err, "cudaSetDevice");
  const bool in32 = b->dtype == Q3S_DTYPE_F32, out32 = b->out_dtype == Q3S_DTYPE_F32;
  const int in = in32 ? 4 : 2, out = out32 ? 4 : 2;
  const int id = b->ids_type == Q3S_IDS_U16 ? 2 : b->ids_type == Q3S_IDS_U32 ? 4 : 8;
  if (reinterpret_cast<uintptr_t>(b->ids) % id || reinterpret_cast<uintptr_t>(b->table) % in ||
      reinterpret_cast<uintptr_t>(b->out) % out)
    return bad("ids, table and out must be aligned to their elements");
  const cudaStream_t st = (cudaStream_t)stream;
  LookupArgs a;
  a.b = *b;
  const cudaError_t e = in32 ? (out32 ? launch_typed<Q3S_DTYPE_F32, Q3S_DTYPE_F32>(a, st)
                                      : launch_typed<Q3S_DTYPE_F32, Q3S_DTYPE_BF16>(a, st))
                             : (out32 ? launch_typed<Q3S_DTYPE_BF16, Q3S_DTYPE_F32>(a, st)
                                      : launch_typed<Q3S_DTYPE_BF16, Q3S_DTYPE_BF16>(a, st));
  if (e != cudaSuccess) return record_cuda_error(e, "lookup kernel launch");
  return Q3S_OK;
}

}  // namespace
}  // namespace q3s

extern "C" int q3s_embed_lookup(q3s_context* ctx, const q3s_lookup_batch* batch, void* stream) {
  return q3s::no_throw([&] { return q3s::embed_lookup(ctx, batch, stream); });
}
