// The cached MoE layer's arithmetic for B200 (sm_100a): the experts of a few tokens read
// from the cache's slots (expert_cache_experts), the same with low-rank adapters of many
// requests (expert_cache_experts_lora), and the router that feeds them
// (expert_cache_route).
//
//   out[t] = sum_j w[t,j] * W2[s] h,   h = silu(G) * U,   [G; U] = W13[s] x[t],
//   s = the slot of the token's j-th expert.
//
// Each routed expert's weights are read once, 3*H*I elements for a handful of tokens: the
// layer is bound by those bytes, so everything else is arranged around streaming them.
//
//   prep_kernel   where up cannot make it itself: x quantised for 8-bit weights (more than
//                 8192 values), A13 x of the adapters.
//   up_kernel     [G; U] and h.  A tile is 8 (gate, up) row pairs of one slot: as the 16 rows
//                 of an m16n8k16 product they leave gate and up of a token in one thread.
//                 The tokens are the 8 columns, so one read of a weight serves them all.
//   mid_kernel    h quantised for 8-bit weights, which needs a row's maximum (small rows are
//                 left to down); A2 h of the adapters.
//   down_kernel   a CTA owns a few columns of `out` and runs over all routed slots, so the
//                 sum over a token's experts stays in its registers: no atomics, no second
//                 pass over out, the same order of sums in every run.
//
// Each kernel lets the next one start early (programmatic dependent launch): its tables are
// built and its first weights on their way while the one before it finishes; it waits only
// for what that one computes.
//
// Measured on a B200 (CUDA graph of calls on fresh weights; floor = bytes at the 6457.7 GB/s
// of a copy):
//   one token of 8 of 64 slots, H 2048, I 768   int8 13.5 us (floor 5.9), bf16 18.7 (11.7);
//     what is above the floor is latency: reading ids and map, the first and last bytes of
//     two streams, h between the kernels
//   8 tokens, 44 experts, H 4096, I 768, fp8    76.6 us (64.5)
//   16 tokens, 96 experts, H 2048, I 768, int8  83.7 us (70.4)
//   2 tokens, 4 experts of 352 MB, bf16         228 us (218): 0.96 of the copy rate
//
// tcgen05 is not used: at n tokens an expert the layer does 2n flops a weight.  For the n of
// a cached step (a few) that is far below what mma.sync feeds (520 Tflop/s measured here in
// bf16, 80 flops for every byte the memory delivers), and mma.sync takes the weights from
// registers in the order in which they arrive, without a detour over a swizzled tile.
//
// Precision: sums in fp32 (int32 for int8, exact).  bf16 layers hold weights[t,j] * h, and all
// layers the adapters' A13 x and A2 h, as the sum of two bf16 values (hi + lo, off by 2^-17 at
// most where fp32 would be by 2^-24), two products with the same weights, so that the layer
// rounds to 8 bits once, at its output; 8-bit layers round x and h (from fp32) as their scheme
// defines.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cstdint>

#include "expert_cache.h"

namespace {

constexpr int kMaxDevices = 64;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxPairs = EXPERT_CACHE_MAX_SLOTS;   // (token, expert) pairs of one launch
constexpr int kMaxTokens = 32;                      // tokens of one launch (4 column tiles)
constexpr int kMaxCols = 16384;                     // pairs x padded tokens of one launch
constexpr size_t kSmem = 227 * 1024;                // shared memory of a CTA

enum WType { kBf16 = 0, kInt8 = 1, kFp8 = 2 };

__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void release_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

struct Adapters {
  const int* index;                // [T] adapter of each token, outside [0, L) = none
  const __nv_bfloat16 *a13, *b13, *a2, *b2;
  const float* scaling;            // [L]
  int L, E, r;                     // r = 0: no adapters
};

struct ExpertsArgs {
  const __nv_bfloat16* x;
  const int* ids;
  const float* weights;
  const int* map;                  // nullptr: ids are slots
  const uint8_t *w13, *w2;
  const float *s13, *s2;
  __nv_bfloat16* out;
  long long ldx, ldo;
  int T, k, H, I, S, n_map;
  float per_k;                     // 1 / k
  // workspace
  __nv_bfloat16 *h_hi, *h_lo;      // bf16 weights: weights[t,j] * h in two parts [P][I]
  float* h;                        // 8-bit weights: h [P][I]
  uint8_t* hq;                     // 8-bit weights: quantised h [P][I]
  float* h_scale;                  // 8-bit weights: its scale x weights[t,j] [P]
  uint8_t* xq;                     // 8-bit weights: quantised x [T][H] where prep_kernel runs
  float* x_scale;                  // and its scales [T]
  int prepared;                    // prep_kernel quantises x
  int self_h;                      // down_kernel quantises h
  __nv_bfloat16 *u_hi, *u_lo;      // adapters: c A13 x in two parts [P][2r]
  __nv_bfloat16 *v_hi, *v_lo;      // adapters: c weights[t,j] A2 h in two parts [P][r]
  Adapters lora;
};

// ---------------------------------------------------------------------------------------
// Which pairs go to which slot.  An entry is one routed slot; its columns are the tokens,
// each with the pair that brought it there or none.  A token that names a slot twice gets
// an entry of its own for every repetition, so that a column never holds two pairs.

struct Routing {
  int* entries;          // [0] entries, [1] does a token repeat a slot, [2] adapted pairs
  unsigned* bits;        // [kMaxPairs / 32] routed slots
  short* slot;           // [P] slot of an entry
  short* pair_slot;      // [P] slot of a pair, -1 = none
  unsigned char* mask;   // [P] column tiles of an entry with a pair in them
  short* col;            // [P][8 NT] pair of an entry's column, -1 = none
  // with adapters
  int* matrix;           // [P] a pair's index among the [L][E] adapter matrices, -1 = none
  unsigned* adapted;     // [P] columns of an entry whose pair has an adapter
  short* list;           // [P] the pairs with adapters
};

constexpr int kRoutingFixed = 16 + (kMaxPairs / 32) * 4;

__host__ __device__ inline size_t routing_bytes(int P, int NT, bool lora) {
  return kRoutingFixed + ((size_t)P * (2 + 2 + 1 + 16 * NT + (lora ? 10 : 0)) + 15) / 16 * 16 + 16;
}

__device__ __forceinline__ Routing routing_at(unsigned char* base, int P, int NT) {
  Routing r;
  r.entries = reinterpret_cast<int*>(base);
  r.bits = reinterpret_cast<unsigned*>(base + 16);
  r.col = reinterpret_cast<short*>(base + kRoutingFixed);
  r.slot = r.col + (size_t)P * 8 * NT;
  r.pair_slot = r.slot + P;
  r.mask = reinterpret_cast<unsigned char*>(r.pair_slot + P);
  r.matrix = reinterpret_cast<int*>(r.mask + (P + 15) / 16 * 16);
  r.adapted = reinterpret_cast<unsigned*>(r.matrix + P);
  r.list = reinterpret_cast<short*>(r.adapted + P);
  return r;
}

__device__ __forceinline__ int token_of(const ExpertsArgs& a, int p) {
  return (int)((p + 0.5f) * a.per_k);          // p / k: exact for p < 2^16, k <= 32
}

__device__ __forceinline__ int slot_of(const ExpertsArgs& a, int p) {
  int s = a.ids[p];
  if (a.map) s = (s >= 0 && s < a.n_map) ? a.map[s] : -1;
  return (s >= 0 && s < a.S) ? s : -1;
}

// The index of a pair's adapter among the [L][E] matrices, or -1.
__device__ __forceinline__ int matrix_of(const ExpertsArgs& a, int p) {
  const int l = a.lora.index[token_of(a, p)], e = a.ids[p];
  return (l < 0 || l >= a.lora.L || e < 0 || e >= a.lora.E) ? -1 : l * a.lora.E + e;
}

// The first reads of a kernel, started before anything else is done.  A map of up to
// kMapCopy entries is copied to shared memory while the ids arrive, so that the two reads do
// not wait for each other (each may be a miss to DRAM, 0.9 us).
constexpr int kMapCopy = 1024;
struct FirstReads {
  int id, map[kMapCopy / kThreads];
  bool copied;
  __device__ __forceinline__ explicit FirstReads(const ExpertsArgs& a) {
    const int tid = threadIdx.x;
    id = tid < a.T * a.k ? a.ids[tid] : -1;
    copied = a.map && a.n_map <= kMapCopy;
#pragma unroll
    for (int j = 0; j < kMapCopy / kThreads; ++j) {
      const int i = tid + j * kThreads;
      map[j] = copied && tid < kThreads && i < a.n_map ? a.map[i] : -1;
    }
  }
};

// Whole CTA (kThreads threads or more); ends with a barrier.  Entries are in ascending slot
// order (repetitions after them in pair order), so sums over entries have one order.
// `scratch`: kMapCopy ints that nothing else uses yet.
template <int NT, bool LORA>
__device__ void build_routing(const ExpertsArgs& a, const Routing& r, const FirstReads& first,
                              int* scratch) {
  const int P = a.T * a.k, tid = threadIdx.x, lane = tid & 31;
  constexpr int kWords = kMaxPairs / 32;
  static_assert(kWords == 32, "a lane holds a word of the slots' bits");
  if (tid < kWords) r.bits[tid] = 0;
  if (tid == 0) r.entries[1] = r.entries[2] = 0;
  for (int i = tid; i < P * 8 * NT / 2; i += blockDim.x)
    reinterpret_cast<int*>(r.col)[i] = -1;
  for (int p = tid; p < P; p += blockDim.x) r.mask[p] = 0;
  const bool copied = first.copied;
  if (copied && tid < kThreads) {
#pragma unroll
    for (int j = 0; j < kMapCopy / kThreads; ++j) scratch[tid + j * kThreads] = first.map[j];
  }
  __syncthreads();
  const auto slot = [&](int id) {
    int s = id;
    if (a.map) s = (id >= 0 && id < a.n_map) ? (copied ? scratch : a.map)[id] : -1;
    return s >= 0 && s < a.S ? s : -1;
  };

  if (P <= 32) {               // one warp, no barriers in between
    if (tid < 32) {
      const unsigned below = (1u << lane) - 1u;
      const int p = lane, s = p < P ? slot(first.id) : -1, t = token_of(a, p);
      const int m = LORA && s >= 0 ? matrix_of(a, p) : -1;
      // pairs of the same slot; one of the same token before this pair makes it a repetition
      const unsigned same = __match_any_sync(0xffffffffu, s);
      const unsigned mine = below & ~((1u << (t * a.k)) - 1u);     // the token's pairs before
      const bool again = s >= 0 && (same & mine) != 0;
      const unsigned lead = __ballot_sync(0xffffffffu, s >= 0 && (same & below) == 0);
      const unsigned rest = __ballot_sync(0xffffffffu, again);
      int e = 0;                                   // leading pairs with a smaller slot
      for (unsigned b = lead; b; b &= b - 1) e += __shfl_sync(0xffffffffu, s, __ffs(b) - 1) < s;
      if (again) e = __popc(lead) + __popc(rest & below);
      if (p < P) r.pair_slot[p] = (short)s;
      if (LORA && p < P) {
        r.matrix[p] = m;
        r.adapted[p] = 0;
      }
      __syncwarp();
      if (s >= 0) {
        r.slot[e] = (short)s;
        r.col[e * 8 * NT + t] = (short)p;
        if (NT == 1) r.mask[e] = 1;
        else atomicOr(reinterpret_cast<unsigned*>(r.mask) + (e >> 2), 1u << (8 * (e & 3) + (t >> 3)));
        if (LORA && m >= 0) atomicOr(&r.adapted[e], 1u << t);
      }
      if (LORA) {
        const unsigned has = __ballot_sync(0xffffffffu, m >= 0);
        if (m >= 0) r.list[__popc(has & below)] = (short)p;
        if (lane == 0) r.entries[2] = __popc(has);
      }
      if (lane == 0) r.entries[0] = __popc(lead) + __popc(rest);
    }
    __syncthreads();
    return;
  }

  for (int p = tid; p < P; p += blockDim.x) {
    r.pair_slot[p] = (short)slot(p == tid ? first.id : a.ids[p]);
    if (LORA) {
      r.matrix[p] = matrix_of(a, p);
      r.adapted[p] = 0;
    }
  }
  __syncthreads();
  for (int p = tid; p < P; p += blockDim.x) {
    const int s = r.pair_slot[p];
    if (s < 0) continue;
    bool again = false;
    for (int q = token_of(a, p) * a.k; q < p; ++q) again |= r.pair_slot[q] == s;
    if (again) r.entries[1] = 1;
    atomicOr(&r.bits[s >> 5], 1u << (s & 31));
  }
  __syncthreads();
  const bool repeats = r.entries[1] != 0;
  const unsigned bits = r.bits[lane];           // every warp counts the entries before a word
  int before = __popc(bits);
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, before, off);
    if (lane >= off) before += o;
  }
  if (tid == 31) r.entries[0] = before;
  before -= __popc(bits);
  for (int p0 = tid - lane; p0 < P; p0 += blockDim.x) {
    const int p = p0 + lane, s = p < P ? r.pair_slot[p] : -1;
    const int word = s >= 0 ? s >> 5 : 0;
    const int base = __shfl_sync(0xffffffffu, before, word);
    const unsigned b = __shfl_sync(0xffffffffu, bits, word);
    const int t = token_of(a, p);
    bool leads = s >= 0;
    if (repeats && s >= 0)
      for (int q = t * a.k; q < p; ++q) leads &= r.pair_slot[q] != s;
    if (!leads) continue;
    const int e = base + __popc(b & ((1u << (s & 31)) - 1u));
    r.slot[e] = (short)s;
    r.col[(size_t)e * 8 * NT + t] = (short)p;
    if (NT == 1) r.mask[e] = 1;
    else atomicOr(reinterpret_cast<unsigned*>(r.mask) + (e >> 2), 1u << (8 * (e & 3) + (t >> 3)));
    if (LORA && r.matrix[p] >= 0) atomicOr(&r.adapted[e], 1u << t);
  }
  if (LORA && tid >= kThreads - 32 && tid < kThreads) {   // the adapted pairs in ascending order
    int n = 0;
    for (int at = 0; at < P; at += 32) {
      const int p = at + lane;
      const bool has = p < P && r.pair_slot[p] >= 0 && r.matrix[p] >= 0;
      const unsigned b = __ballot_sync(0xffffffffu, has);
      if (has) r.list[n + __popc(b & ((1u << lane) - 1u))] = (short)p;
      n += __popc(b);
    }
    if (lane == 0) r.entries[2] = n;
  }
  __syncthreads();
  if (!repeats) return;
  if (tid == 0) {
    int n = r.entries[0];
    for (int p = 0; p < P; ++p) {
      const int s = r.pair_slot[p], t = token_of(a, p);
      bool leads = true;
      for (int q = t * a.k; q < p; ++q) leads &= r.pair_slot[q] != s;
      if (s < 0 || leads) continue;
      r.slot[n] = (short)s;
      r.col[(size_t)n * 8 * NT + t] = (short)p;
      r.mask[n] = (unsigned char)(1u << (t >> 3));
      if (LORA && r.matrix[p] >= 0) r.adapted[n] = 1u << t;
      ++n;
    }
    r.entries[0] = n;
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------------------
// One chunk: 64 bytes of each of 16 weight rows.  Lane (g = lane / 4, q = lane % 4) holds 16
// bytes of rows g and g + 8 and, of column g, the same 16 bytes: which of the chunk's
// columns an index of the product stands for is free as long as both operands agree, so
// every lane loads whole 16-byte vectors.

template <int WT>
struct Kind {
  static constexpr int kItem = WT == kBf16 ? 2 : 1;      // bytes per weight
  using Acc = float;
};
template <>
struct Kind<kInt8> {
  static constexpr int kItem = 1;
  using Acc = int;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2,
                                         unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2,
                                        unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2,
                                       unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two e4m3 values (the low 16 bits) as two fp16 values, exactly.
__device__ __forceinline__ unsigned e4m3x2_to_f16x2(unsigned v) {
  unsigned r;
  asm("{.reg .b16 t, u; mov.b32 {t, u}, %1; cvt.rn.f16x2.e4m3x2 %0, t;}" : "=r"(r) : "r"(v));
  return r;
}

// Sums are kept in four parts, each product's after the one before it in another part: a
// product waits some 20 cycles for its accumulator, and two warps a scheduler do not hide a
// chain of them (12 tokens of 6 of 9 experts 79 -> 76 us).  In two parts for 8-bit weights and
// one column tile: the registers of more keep the next CTA off the SM (one token int8
// 14.2 -> 15.2 us).
template <int WT, int NT>
constexpr int kSumParts = WT != kBf16 && NT == 1 ? 2 : 4;

// (16 rows: a, b) x (8 columns: v) over one chunk, added to parts c0 and c1.
__device__ __forceinline__ void chunk_mma_bf16(float (&c0)[4], float (&c1)[4], const uint4& a,
                                               const uint4& b, const uint4& v) {
  mma_bf16(c0, a.x, b.x, a.y, b.y, v.x, v.y);
  mma_bf16(c1, a.z, b.z, a.w, b.w, v.z, v.w);
}
__device__ __forceinline__ void chunk_mma_s8(int (&c0)[4], int (&c1)[4], const uint4& a,
                                             const uint4& b, const uint4& v) {
  mma_s8(c0, a.x, b.x, a.y, b.y, v.x, v.y);
  mma_s8(c1, a.z, b.z, a.w, b.w, v.z, v.w);
}

// 16 e4m3 values as fp16: lane's words for four m16n8k16 products.
struct Wide {
  unsigned lo[4], hi[4];
};
__device__ __forceinline__ Wide widen(const uint4& v) {
  Wide w;
  const unsigned u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w.lo[i] = e4m3x2_to_f16x2(u[i]);
    w.hi[i] = e4m3x2_to_f16x2(u[i] >> 16);
  }
  return w;
}
template <int N, int NT>
__device__ __forceinline__ void chunk_mma_fp8(float (&c)[N][NT][4], int nt, const Wide& a,
                                              const Wide& b, const uint4& v) {
  const Wide w = widen(v);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    mma_f16(c[i % N][nt], a.lo[i], b.lo[i], a.hi[i], b.hi[i], w.lo[i], w.hi[i]);
}

// The sum of the parts.
template <typename Acc, int N, int NT>
__device__ __forceinline__ Acc whole(const Acc (&c)[N][NT][4], int nt, int i) {
  Acc s = c[0][nt][i];
#pragma unroll
  for (int part = 1; part < N; ++part) s += c[part][nt][i];
  return s;
}

// ---------------------------------------------------------------------------------------
// The stream of weights.  Every thread copies the very bytes that it will multiply into a
// FIFO of its own in shared memory (cp.async), so the stream needs no barrier and no thread
// waits for another's data.  A stage is a block of KB chunks, that is KB * 64 contiguous
// bytes of each of the 16 rows: addresses, waits and branches are paid once a block.  (With
// a stage a chunk the kernels executed 100 to 230 instructions a chunk and were bound by
// issuing them, at 0.37 of the memory's rate.)  The FIFOs leave room for a CTA of up and one
// of down on an SM, so that down has its tables and its first stages before up is done.

constexpr int kUpBlock = 4, kUpStages = 3;
constexpr int kUpFifo = kUpStages * kUpBlock * kThreads * 32;
// Chunks of a thread's FIFO in down: without h in shared memory, with it.
constexpr int kDownChunks[2] = {16, 12};
constexpr int down_fifo(bool hs) { return kDownChunks[hs] * kThreads * 32; }

// size 0: the vector is zero-filled and nothing is read.
__device__ __forceinline__ void copy16_sized(unsigned dst, const uint8_t* src, int size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size)
               : "memory");
}
__device__ __forceinline__ void copy16(unsigned dst, const uint8_t* src, bool in) {
  copy16_sized(dst, src, in ? 16 : 0);
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// All but the newest N groups of copies have landed.
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 16 bytes from L2, or zeros and no read.
__device__ __forceinline__ uint4 load_or_zero(const void* p, bool in) {
  uint4 r;
  asm volatile(
      "{.reg .pred p; setp.ne.b32 p, %5, 0; mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; "
      "mov.b32 %3, 0; @p ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];}"
      : "=&r"(r.x), "=&r"(r.y), "=&r"(r.z), "=&r"(r.w)
      : "l"(p), "r"((int)in)
      : "memory");
  return r;
}

__device__ __forceinline__ uint4 load_shared(unsigned at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(at)
               : "memory");
  return r;
}

template <int KB, int ST, int THREADS = kThreads>
struct Fifo {
  static constexpr int kStage = THREADS * KB * 32, kStages = ST;
  unsigned base, put, get;       // this thread's vectors of stage 0, of the next to fill / read
  __device__ __forceinline__ explicit Fifo(const void* smem) {
    base = (unsigned)__cvta_generic_to_shared(smem) + (threadIdx.x >> 5) * (KB * 1024) +
           (threadIdx.x & 31) * 16;
    put = get = base;
  }
  // The next block of row `a` (row g) and row `b` (row g + 8), `left_*` bytes of them left to
  // read (nothing is read past them).
  __device__ __forceinline__ void push(const uint8_t* a, int left_a, const uint8_t* b, int left_b) {
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      copy16(put + j * 1024, a + j * 64, left_a > j * 64);
      copy16(put + j * 1024 + 512, b + j * 64, left_b > j * 64);
    }
    put = put == base + (kStages - 1) * kStage ? base : put + kStage;
  }
  // The same where the whole block lies in the row; `size_*` 16, or 0 for zeros.
  __device__ __forceinline__ void push_whole(const uint8_t* a, int size_a, const uint8_t* b,
                                             int size_b) {
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      copy16_sized(put + j * 1024, a + j * 64, size_a);
      copy16_sized(put + j * 1024 + 512, b + j * 64, size_b);
    }
    put = put == base + (kStages - 1) * kStage ? base : put + kStage;
  }
  // Waits until the oldest stage has landed; its vectors are at the returned address.
  __device__ __forceinline__ unsigned front() {
    copy_wait<kStages - 1>();
    const unsigned at = get;
    get = get == base + (kStages - 1) * kStage ? base : get + kStage;
    return at;
  }
};

// ---------------------------------------------------------------------------------------
// Quantised rows: q = round(v * Q / top), scale = top / Q, top = max|v|.  The quotient comes
// from a product with Q / top, which is off by 2^-23 of it at most; only where that could
// put it on the other side of a border between two values is it divided (the product v * Q
// of a bf16 v is exact in fp32 and the division correctly rounded, so a quotient that lies
// on a border is seen as such).  Dividing every element took 13 us for 16 tokens of 2048.

struct RowQuant {
  float top, inv;
};
template <int WT>
__device__ __forceinline__ RowQuant row_quant(float top) {
  return RowQuant{top, (WT == kInt8 ? 127.f : 448.f) / top};
}
template <int WT>
__device__ __forceinline__ float quant_scale(float top) {
  return top / (WT == kInt8 ? 127.f : 448.f);
}

template <int WT>
__device__ __noinline__ unsigned quantise_exactly(float v, float top) {
  if (top > 0x1p119f) {          // v * Q must not overflow: 2^119 * 448 < 2^128
    v *= 0x1p-20f;
    top *= 0x1p-20f;
  }
  if (WT == kInt8) return (unsigned)(unsigned char)(signed char)__float2int_rn(v * 127.f / top);
  return __nv_cvt_float_to_fp8(v * 448.f / top, __NV_SATFINITE, __NV_E4M3);
}

// Four values, packed.
template <int WT>
__device__ __forceinline__ unsigned quantise4(float v0, float v1, float v2, float v3,
                                              const RowQuant& s) {
  const float r[4] = {v0 * s.inv, v1 * s.inv, v2 * s.inv, v3 * s.inv};
  unsigned out;
  bool sure;
  if (WT == kInt8) {
    constexpr float kRound = 12582912.f;         // 1.5 * 2^23: adding it rounds to an integer
    float m[4];
    sure = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = __fadd_rn(r[i], kRound);
      sure &= fabsf(r[i] - __fsub_rn(m[i], kRound)) < 0.4999f;    // false for a NaN
    }
    out = __byte_perm(__byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x0040),
                      __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x0040), 0x5410);
  } else {
    constexpr float kLow = 1.f - 0x1p-20f, kHigh = 1.f + 0x1p-20f;
    unsigned short lo[2], hi[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lo[i] = __nv_cvt_float2_to_fp8x2(make_float2(r[2 * i] * kLow, r[2 * i + 1] * kLow),
                                       __NV_SATFINITE, __NV_E4M3);
      hi[i] = __nv_cvt_float2_to_fp8x2(make_float2(r[2 * i] * kHigh, r[2 * i + 1] * kHigh),
                                       __NV_SATFINITE, __NV_E4M3);
    }
    sure = lo[0] == hi[0] && lo[1] == hi[1];
    out = lo[0] | (unsigned)lo[1] << 16;
  }
  if (!sure)
    out = quantise_exactly<WT>(v0, s.top) | quantise_exactly<WT>(v1, s.top) << 8 |
          quantise_exactly<WT>(v2, s.top) << 16 | quantise_exactly<WT>(v3, s.top) << 24;
  return out;
}

// The bits of |v| order as |v| does, a NaN above all, so that a maximum of them keeps it.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float clamp_top(unsigned bits) {
  const float m = __uint_as_float(bits);
  return m < 1e-10f ? 1e-10f : m;
}

// Where chunk j of block `blk` of token t lies in the staged x: [block][T][4 chunks], a
// token's odd and even chunks swapped for odd t, so that eight lanes of two tokens read all
// banks.
__device__ __forceinline__ int staged_at(int T, int blk, int t, int j) {
  return (blk * T + t) * 256 + ((j ^ (t & 1)) * 64);
}

// Byte `pos` of token t's row there.
__device__ __forceinline__ int staged_byte(int T, int t, int pos) {
  return staged_at(T, pos >> 8, t, pos >> 6 & 3) + (pos & 63);
}

// Copies of rows of `row_bytes` (x, or the quantised x) into the staged form, zeros past
// their ends.  Whole CTA; the caller commits, waits and synchronises.
__device__ __forceinline__ void stage_rows(const uint8_t* rows, long long stride, int row_bytes,
                                           int T, unsigned char* st) {
  const unsigned to = (unsigned)__cvta_generic_to_shared(st);
  const int per = (row_bytes + 255) / 256 * 16;
  for (int i = threadIdx.x; i < per * T; i += kThreads) {
    const int t = i / per, pos = (i - t * per) * 16;
    copy16(to + staged_byte(T, t, pos), rows + t * stride + pos, pos < row_bytes);
  }
}

// 8-bit weights: x that up quantises itself, in registers: T * H values at most.  Beyond
// that prep_kernel does it once for all CTAs (13 us of 105 were spent here for 16 tokens of
// 2048, most of it waiting for x behind the first weights).
constexpr int kSelfX = 8192;
constexpr int kSelfXVectors = kSelfX / 8 / kThreads;

struct HeldX {
  uint4 v[kSelfXVectors];
  __device__ __forceinline__ void load(const ExpertsArgs& a) {
    const int per = a.H / 8;
#pragma unroll
    for (int j = 0; j < kSelfXVectors; ++j) {
      v[j] = make_uint4(0, 0, 0, 0);
      if (j * kThreads >= per * a.T) continue;
      const int i = threadIdx.x + j * kThreads, t = i / per;
      if (t < a.T) v[j] = *reinterpret_cast<const uint4*>(a.x + t * a.ldx + (i - t * per) * 8);
    }
  }
};

__device__ __forceinline__ float low_bf16(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_bf16(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

__device__ __forceinline__ unsigned top_bits(const uint4& v) {
  const unsigned u[4] = {v.x, v.y, v.z, v.w};
  unsigned top = 0;
#pragma unroll
  for (int m = 0; m < 4; ++m) top = max(top, max(u[m] << 16 & 0x7fffffffu, u[m] & 0x7fff0000u));
  return top;
}

template <int WT>
__device__ __forceinline__ uint2 quantise8(const uint4& v, const RowQuant& s) {
  return make_uint2(
      quantise4<WT>(low_bf16(v.x), high_bf16(v.x), low_bf16(v.y), high_bf16(v.y), s),
      quantise4<WT>(low_bf16(v.z), high_bf16(v.z), low_bf16(v.w), high_bf16(v.w), s));
}

// The held x, quantised, into the staged form.  Whole CTA; ends with a barrier.
template <int WT>
__device__ void stage_held(const ExpertsArgs& a, const HeldX& x, unsigned char* st, float* xs) {
  __shared__ unsigned tops[kMaxTokens];
  __shared__ float inv[kMaxTokens];
  const int tid = threadIdx.x, lane = tid & 31, per = a.H / 8;
  if (tid < kMaxTokens) tops[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSelfXVectors; ++j) {
    // (code that is not run is not fetched: skipping the empty vectors saves 1 us)
    if (j * kThreads >= per * a.T) break;
    const int t = (tid + j * kThreads) / per;
    const unsigned top = top_bits(x.v[j]);
    if (__all_sync(0xffffffffu, t == __shfl_sync(0xffffffffu, t, 0))) {
      const unsigned m = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0 && t < a.T) atomicMax(&tops[t], m);
    } else if (t < a.T) {
      atomicMax(&tops[t], top);
    }
  }
  __syncthreads();
  if (tid < a.T) {
    const float top = clamp_top(tops[tid]);
    tops[tid] = __float_as_uint(top);
    inv[tid] = row_quant<WT>(top).inv;
    xs[tid] = quant_scale<WT>(top);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSelfXVectors; ++j) {
    if (j * kThreads >= per * a.T) break;
    const int i = tid + j * kThreads, t = i / per;
    if (t < a.T)
      *reinterpret_cast<uint2*>(st + staged_byte(a.T, t, (i - t * per) * 8)) =
          quantise8<WT>(x.v[j], RowQuant{__uint_as_float(tops[t]), inv[t]});
  }
  const int tail = (a.H + 255) / 256 * 256 - a.H;            // zeros, 16 bytes at a time
  for (int i = tid; i < tail / 16 * a.T; i += kThreads) {
    const int t = i / (tail / 16), pos = a.H + (i - t * (tail / 16)) * 16;
    *reinterpret_cast<uint4*>(st + staged_byte(a.T, t, pos)) = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
}

// A sum as two bf16 values (an infinite high part has no remainder).
__device__ __forceinline__ void split(float v, __nv_bfloat16* hi, __nv_bfloat16* lo) {
  *hi = __float2bfloat16(v);
  const float back = __bfloat162float(*hi);
  *lo = __float2bfloat16(isfinite(back) ? v - back : 0.f);
}

__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float s) {
  const unsigned x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s = fmaf(__uint_as_float(x[j] << 16), __uint_as_float(y[j] << 16), s);
    s = fmaf(__uint_as_float(x[j] & 0xffff0000u), __uint_as_float(y[j] & 0xffff0000u), s);
  }
  return s;
}

// ---------------------------------------------------------------------------------------
// prep: what up needs of x for many rows.  The first `prepared ? T : 0` CTAs quantise a token
// each; the others, with adapters, compute u[p] = c A13[adapter, expert] x[t], a warp a row.

template <int WT, bool LORA>
__global__ void __launch_bounds__(kThreads) prep_kernel(const __grid_constant__ ExpertsArgs a) {
  grid_dependency_wait();
  release_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int block = blockIdx.x;
  if (WT != kBf16 && a.prepared) {
    if (block < a.T) {
      __shared__ unsigned tops[kWarps];
      const __nv_bfloat16* x = a.x + block * a.ldx;
      uint4 held[4];                             // rows of up to 8192 are read once
      unsigned top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (tid + j * kThreads) * 8;
        held[j] = make_uint4(0, 0, 0, 0);
        if (i < a.H) held[j] = *reinterpret_cast<const uint4*>(x + i);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, top_bits(held[j]));
      for (int i = (tid + 4 * kThreads) * 8; i < a.H; i += kThreads * 8)
        top = max(top, top_bits(*reinterpret_cast<const uint4*>(x + i)));
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) tops[warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max(top, tops[w]);
      const float m = clamp_top(top);
      const RowQuant s = row_quant<WT>(m);
      uint8_t* to = a.xq + (size_t)block * a.H;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (tid + j * kThreads) * 8;
        if (i < a.H) *reinterpret_cast<uint2*>(to + i) = quantise8<WT>(held[j], s);
      }
      for (int i = (tid + 4 * kThreads) * 8; i < a.H; i += kThreads * 8)
        *reinterpret_cast<uint2*>(to + i) =
            quantise8<WT>(*reinterpret_cast<const uint4*>(x + i), s);
      if (tid == 0) a.x_scale[block] = quant_scale<WT>(m);
      return;
    }
    block -= a.T;
  }
  if (!LORA) return;
  const int rows = 2 * a.lora.r, per = (rows + kWarps - 1) / kWarps;
  const int p = block / per, row = (block - p * per) * kWarps + warp;
  if (row >= rows || slot_of(a, p) < 0) return;
  const int m = matrix_of(a, p);
  if (m < 0) return;
  const __nv_bfloat16* w = a.lora.a13 + ((long long)m * rows + row) * a.H;
  const __nv_bfloat16* x = a.x + token_of(a, p) * a.ldx;
  const float factor = a.lora.scaling[m / a.lora.E];
  float s = 0.f;
#pragma unroll 8
  for (int i = lane * 8; i < a.H; i += 256)
    s = dot8(*reinterpret_cast<const uint4*>(w + i), *reinterpret_cast<const uint4*>(x + i), s);
#pragma unroll
  for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (lane == 0) {
    const size_t at = (size_t)p * rows + row;
    split(s * factor, a.u_hi + at, a.u_lo + at);
  }
}

// ---------------------------------------------------------------------------------------
// up

// Every entry's row pairs are cut into the same number of tiles of up to 8, and the warps take
// the tiles in turn.  The number is the largest that needs no more turns than tiles of 8 do,
// so that all warps have as many and, within a row, equally large ones; a tile is a row pair
// of 8 at most and never crosses into another entry (a warp whose share did had two tiles to
// stream where the others had one, and held up the layer by 5 us of 25).  No warp waits for
// another: the rows stay in one warp over their whole length, so that h comes straight from
// the accumulators.
struct UpTiles {
  int I, per_entry, all;
  __device__ __forceinline__ UpTiles(int D, int I_, int W) : I(I_) {
    const int least = (I + 7) / 8;
    const int turns = (D * least + W - 1) / W;
    per_entry = D ? min(I, turns * W / D) : 0;
    all = D * per_entry;
  }
};
struct UpTile {
  int e, i0, n;
  __device__ __forceinline__ void at(const UpTiles& t, int i) {
    e = (unsigned)i / (unsigned)t.per_entry;
    const int j = i - e * t.per_entry;
    i0 = (unsigned)(j * t.I) / (unsigned)t.per_entry;              // (at most I * I <= 2^30)
    n = (unsigned)((j + 1) * t.I) / (unsigned)t.per_entry - i0;
  }
};

template <int WT, int NT, bool LORA, bool STAGED>
__global__ void __launch_bounds__(kThreads, 1) up_kernel(const __grid_constant__ ExpertsArgs a) {
  using K = Kind<WT>;
  using Acc = typename K::Acc;
  constexpr int KB = kUpBlock;
  static_assert(KB == 4, "a block of the staged x is four chunks");
  using Stream = Fifo<KB, kUpStages>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int P = a.T * a.k;
  Stream fifo(smem);
  const Routing rt = routing_at(smem + kUpFifo, P, NT);
  float* xs = reinterpret_cast<float*>(smem + kUpFifo + routing_bytes(P, NT, LORA));
  unsigned char* st = reinterpret_cast<unsigned char*>(xs + kMaxTokens);

  // Where prep_kernel runs before this one, it starts this grid once its own wait is over, so
  // the call's inputs are complete and only its results are waited for, below.
  const bool after_prep = LORA || (WT != kBf16 && a.prepared);
  if (!after_prep) grid_dependency_wait();
  release_dependents();
  const FirstReads first(a);
  HeldX held;
  if (WT == kBf16 && STAGED) {
    stage_rows(reinterpret_cast<const uint8_t*>(a.x), a.ldx * 2, a.H * 2, a.T, st);
    copy_commit();
  }
  if (WT != kBf16 && !a.prepared) held.load(a);
  build_routing<NT, LORA>(a, rt, first, reinterpret_cast<int*>(smem));
  const int D = rt.entries[0];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int W = gridDim.x * kWarps, w = warp * gridDim.x + blockIdx.x;
  const UpTiles tiles(D, a.I, W);
  const int row_bytes = a.H * K::kItem, lora_bytes = LORA ? a.lora.r * 2 : 0;
  const long long up_off = (long long)a.I * row_bytes;

  // The blocks of the warp's tiles in order, those of each tile's adapted columns after them;
  // `src` and the counters follow the head of the stream.
  UpTile head;
  int hi = w;                   // its tile
  const uint8_t* src = nullptr;
  int pos = 0;                  // bytes of the row (of B13's, past the row's end) gone by
  unsigned adapted = 0;
  const auto head_at = [&]() {
    head.at(tiles, hi);
    src = a.w13 + ((long long)rt.slot[head.e] * 2 * a.I + head.i0 + g) * row_bytes + q * 16;
    pos = 0;
    if (LORA) adapted = rt.adapted[head.e];
  };
  const auto push = [&]() {
    if (hi < tiles.all) {
      const bool mine = g < head.n;
      if (!LORA || pos < row_bytes) {
        if (pos + KB * 64 <= row_bytes) {
          const int size = mine ? 16 : 0;
          fifo.push_whole(src, size, src + up_off, size);
        } else {
          const int left = mine ? row_bytes - pos - q * 16 : 0;
          fifo.push(src, left, src + up_off, left);
        }
        src += KB * 64;
        pos += KB * 64;
      } else {
        const int at = pos - (row_bytes + KB * 64 - 1) / (KB * 64) * (KB * 64);
        const int p = rt.col[(size_t)head.e * 8 * NT + __ffs(adapted) - 1];
        const uint8_t* b = reinterpret_cast<const uint8_t*>(a.lora.b13) +
                           ((long long)rt.matrix[p] * 2 * a.I + head.i0 + g) * lora_bytes + at +
                           q * 16;
        const int left = mine ? lora_bytes - at - q * 16 : 0;
        fifo.push(b, left, b + (long long)a.I * lora_bytes, left);
        pos += KB * 64;
        if (at + KB * 64 >= lora_bytes) {
          pos -= at + KB * 64;
          adapted &= adapted - 1;
        }
      }
      if (pos >= row_bytes && (!LORA || adapted == 0)) {
        hi += W;
        if (hi < tiles.all) head_at();
      }
    }
    copy_commit();
  };
  if (hi < tiles.all) head_at();
  for (int i = 0; i < Stream::kStages; ++i) push();

  if (WT != kBf16 && !a.prepared) stage_held<WT>(a, held, st, xs);
  // The adapters' u is needed at a tile's end only: unless x comes from prep too, each warp
  // waits for it there.
  bool waited = true;
  if (WT != kBf16 && a.prepared) grid_dependency_wait();
  else waited = !LORA;
  if (WT != kBf16 && a.prepared) {
    stage_rows(a.xq, a.H, a.H, a.T, st);
    copy_commit();
    if (tid < a.T) xs[tid] = __ldcg(a.x_scale + tid);
    copy_wait<0>();
    __syncthreads();
  }
  if (WT == kBf16 && STAGED) {       // x was copied before the stages
    copy_wait<Stream::kStages>();
    __syncthreads();
  }

  // Column g's token of each column tile.  Past the last token: any (the column is not kept).
  const unsigned char *xa[NT], *xb[NT];         // staged: even and odd chunks
  const __nv_bfloat16* xg[NT];                  // not staged: the row in global memory
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int t = min(nt * 8 + g, a.T - 1);
    xa[nt] = st + q * 16 + staged_at(a.T, 0, t, 0);
    xb[nt] = st + q * 16 + staged_at(a.T, 0, t, 1);
    xg[nt] = a.x + t * a.ldx + q * 8;
  }

  UpTile tile;
  for (int i = w; i < tiles.all; i += W) {
    tile.at(tiles, i);
    const int slot = rt.slot[tile.e], r = tile.i0 + g;
    const unsigned mask = rt.mask[tile.e];
    const bool mine = g < tile.n;
    const short* col = rt.col + (size_t)tile.e * 8 * NT;
    float sg = 1.f, su = 1.f;
    if (WT != kBf16 && mine) {
      sg = a.s13[(long long)slot * 2 * a.I + r];
      su = a.s13[(long long)slot * 2 * a.I + a.I + r];
    }
    // u of an adapted column's first chunk (gate's high and low parts, up's), read ahead
    unsigned cols = LORA ? rt.adapted[tile.e] : 0;
    uint4 u[LORA ? 4 : 1];
    const auto read_u = [&](int t, int at, uint4(&to)[LORA ? 4 : 1]) {
      if constexpr (LORA) {
        const bool has = g == (t & 7) && at + q * 16 < lora_bytes;
        const size_t m = (size_t)col[t] * 2 * a.lora.r + q * 8 + at / 2;
        to[0] = load_or_zero(a.u_hi + m, has);
        to[1] = load_or_zero(a.u_lo + m, has);
        to[2] = load_or_zero(a.u_hi + m + a.lora.r, has);
        to[3] = load_or_zero(a.u_lo + m + a.lora.r, has);
      }
    };
    const bool ahead = waited;
    if (LORA && ahead && cols) read_u(__ffs(cols) - 1, 0, u);
    constexpr int kN = kSumParts<WT, NT>;
    Acc acc[kN][NT][4] = {};
    for (int at = 0, blk = 0; at < row_bytes; at += KB * 64) {
      const unsigned f = fifo.front();
      uint4 wa[KB], wb[KB];
#pragma unroll
      for (int j = 0; j < KB; ++j) {
        wa[j] = load_shared(f + j * 1024);
        wb[j] = load_shared(f + j * 1024 + 512);
      }
#pragma unroll
      for (int j = 0; j < KB; ++j) {
        Wide fa, fb;
        if (WT == kFp8) { fa = widen(wa[j]); fb = widen(wb[j]); }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (NT > 1 && !(mask >> nt & 1)) continue;
          uint4 v;
          if constexpr (STAGED) {
            v = *reinterpret_cast<const uint4*>((j & 1 ? xb[nt] : xa[nt]) + blk + (j & 2) * 64);
          } else {
            v = make_uint4(0, 0, 0, 0);
            if (at + j * 64 + q * 16 < row_bytes)
              v = *reinterpret_cast<const uint4*>(xg[nt] + (at + j * 64) / 2);
          }
          auto& c0 = acc[2 * j % kN][nt];
          auto& c1 = acc[(2 * j + 1) % kN][nt];
          if constexpr (WT == kBf16) chunk_mma_bf16(c0, c1, wa[j], wb[j], v);
          if constexpr (WT == kInt8) chunk_mma_s8(c0, c1, wa[j], wb[j], v);
          if constexpr (WT == kFp8) chunk_mma_fp8(acc, nt, fa, fb, v);
        }
      }
      push();      // into the stage just read, whose vectors the products have taken
      blk += a.T * 256;
    }
    // Adapters: one more product for each adapted column, B13's rows with u in that column
    // alone.  Gate and up have different u, so each takes its half of the 16 rows.
    float add[LORA ? NT : 1][4] = {};
    if constexpr (LORA) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      if (cols && !waited) {
        grid_dependency_wait();
        waited = true;
      }
      if (cols && !ahead) read_u(__ffs(cols) - 1, 0, u);
      for (; cols; cols &= cols - 1) {
        const int t = __ffs(cols) - 1;
        const unsigned rest = cols & (cols - 1);
        float one[4] = {};
        for (int at = 0; at < lora_bytes; at += KB * 64) {
          const unsigned f = fifo.front();
#pragma unroll
          for (int j = 0; j < KB; ++j) {
            if (at + j * 64 >= lora_bytes) break;
            uint4 v[4];
            if (j == 0 && at == 0) {
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] = u[i];
              if (rest) read_u(__ffs(rest) - 1, 0, u);
            } else {
              read_u(t, at + j * 64, v);
            }
            const uint4 wa = load_shared(f + j * 1024), wb = load_shared(f + j * 1024 + 512);
            chunk_mma_bf16(one, one, wa, zero, v[0]);
            chunk_mma_bf16(one, one, wa, zero, v[1]);
            chunk_mma_bf16(one, one, zero, wb, v[2]);
            chunk_mma_bf16(one, one, zero, wb, v[3]);
          }
          push();
        }
        // (only the column itself: a row of B13 with an infinity or a NaN is one in them all)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t == nt * 8 + 2 * q + (i & 1)) add[nt][i] = one[i];
      }
    }
    if (!mine) continue;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (NT > 1 && !(mask >> nt & 1)) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = nt * 8 + 2 * q + j, p = col[t];
        if (p < 0) continue;
        float gate = (float)whole(acc, nt, j), up = (float)whole(acc, nt, 2 + j);
        if (WT != kBf16) {
          gate *= xs[t] * sg;
          up *= xs[t] * su;
        }
        if (LORA) {
          gate += add[nt][j];
          up += add[nt][2 + j];
        }
        const float h = gate / (1.f + expf(-gate)) * up;
        const size_t at = (size_t)p * a.I + r;
        if (WT == kBf16) split(h * a.weights[p], a.h_hi + at, a.h_lo + at);
        else a.h[at] = h;
      }
    }
  }
  if (!waited) grid_dependency_wait();     // this grid's end means prep's, too
}

// ---------------------------------------------------------------------------------------
// mid: what down needs of h and cannot make itself.  With 8-bit weights the first P CTAs
// quantise a pair's h each (unless down does: `self_h`); the others, with
// adapters, compute v[p] = c weights[t,j] A2[adapter, expert] h, a warp a row.  All that does not
// hang on h is read before the wait, A2's rows too.

template <int WT, bool LORA>
__global__ void __launch_bounds__(kThreads) mid_kernel(const __grid_constant__ ExpertsArgs a) {
  release_dependents();       // down may start streaming: it waits for this kernel's end
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P = a.T * a.k;
  int block = blockIdx.x;
  if (WT != kBf16 && !a.self_h) {
    if (block < P) {
      const int p = block;
      const bool has = slot_of(a, p) >= 0;
      const float weight = a.weights[p];
      grid_dependency_wait();
      if (!has) return;
      const size_t at = (size_t)p * a.I;
      __shared__ unsigned tops[kWarps];
      unsigned top = 0;
      float4 held[4];                            // rows of up to 4096 are read once
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (tid + j * kThreads) * 4;
        held[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < a.I) held[j] = __ldcg(reinterpret_cast<const float4*>(a.h + at + i));
      }
      const auto top_of = [](const float4& v) {
        return max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
      };
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, top_of(held[j]));
      for (int i = (tid + 4 * kThreads) * 4; i < a.I; i += kThreads * 4)
        top = max(top, top_of(__ldcg(reinterpret_cast<const float4*>(a.h + at + i))));
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == 0) tops[warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max(top, tops[w]);
      const float m = clamp_top(top);
      const RowQuant rq = row_quant<WT>(m);
      if (tid == 0) a.h_scale[p] = quant_scale<WT>(m) * weight;
      const auto store = [&](int i, const float4& v) {
        *reinterpret_cast<unsigned*>(a.hq + at + i) = quantise4<WT>(v.x, v.y, v.z, v.w, rq);
      };
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((tid + j * kThreads) * 4 < a.I) store((tid + j * kThreads) * 4, held[j]);
      for (int i = (tid + 4 * kThreads) * 4; i < a.I; i += kThreads * 4)
        store(i, __ldcg(reinterpret_cast<const float4*>(a.h + at + i)));
      return;
    }
    block -= P;
  }
  if (!LORA) return;
  const int per = (a.lora.r + kWarps - 1) / kWarps;
  const int p = block / per, row = (block - p * per) * kWarps + warp;
  const int m = row < a.lora.r && slot_of(a, p) >= 0 ? matrix_of(a, p) : -1;
  constexpr int kHeld = 8;                       // rows of up to 2048 are read ahead
  uint4 w[kHeld];
  float factor = 0.f;
  const __nv_bfloat16* from = a.lora.a2 + ((long long)max(m, 0) * a.lora.r + row) * a.I;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = lane * 8 + j * 256;
    w[j] = make_uint4(0, 0, 0, 0);
    if (m >= 0 && i < a.I) w[j] = *reinterpret_cast<const uint4*>(from + i);
  }
  // bf16 weights: h already carries the routing weight
  if (m >= 0) factor = a.lora.scaling[m / a.lora.E] * (WT == kBf16 ? 1.f : a.weights[p]);
  grid_dependency_wait();
  if (m < 0) return;
  const size_t at = (size_t)p * a.I;
  float s = 0.f;
  const auto add = [&](const uint4& wv, int i) {
    if (WT == kBf16) {
      s = dot8(wv, __ldcg(reinterpret_cast<const uint4*>(a.h_hi + at + i)), s);
      s = dot8(wv, __ldcg(reinterpret_cast<const uint4*>(a.h_lo + at + i)), s);
    } else {
      const float4 h0 = __ldcg(reinterpret_cast<const float4*>(a.h + at + i));
      const float4 h1 = __ldcg(reinterpret_cast<const float4*>(a.h + at + i + 4));
      const unsigned x[4] = {wv.x, wv.y, wv.z, wv.w};
      const float h[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s = fmaf(low_bf16(x[j]), h[2 * j], s);
        s = fmaf(high_bf16(x[j]), h[2 * j + 1], s);
      }
    }
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (lane * 8 + j * 256 < a.I) add(w[j], lane * 8 + j * 256);
  for (int i = lane * 8 + kHeld * 256; i < a.I; i += 256)
    add(*reinterpret_cast<const uint4*>(from + i), i);
#pragma unroll
  for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (lane == 0) {
    const size_t to = (size_t)p * a.lora.r + row;
    split(s * factor, a.v_hi + to, a.v_lo + to);
  }
}

// ---------------------------------------------------------------------------------------
// down

// A CTA owns a range of out's columns, taken in tiles of up to 16 (rows of W2).  Within a
// tile a warp takes every kWarps-th unit: a slice of an entry's rows, its blocks one after
// the other, with the accumulators kept over all units; then every kWarps-th adapted pair.
// Entries are sliced only as far as it takes to give the warps equal shares.
struct DownUnits {
  int entries, log_slices, blocks, units;       // units of all entries
  int pairs, pair_blocks;                       // adapted pairs after them
  __device__ __forceinline__ void plan(int D, int CB, int adapted, int RB) {
    entries = D;
    blocks = CB;
    log_slices = 0;
    while ((D << log_slices) % kWarps != 0 && (D << log_slices) < 4 * kWarps &&
           (2 << log_slices) <= CB)
      ++log_slices;
    units = D << log_slices;
    pairs = adapted;
    pair_blocks = RB;
  }
  __device__ __forceinline__ int all() const { return units + pairs; }
  __device__ __forceinline__ int entry(int u) const { return u >> log_slices; }
  // First block of unit u (of u + 1: its end).
  __device__ __forceinline__ int first(int u) const {
    return (u & ((1 << log_slices) - 1)) * blocks >> log_slices;
  }
  __device__ __forceinline__ int end(int u) const {
    return ((u & ((1 << log_slices) - 1)) + 1) * blocks >> log_slices;
  }
};
__device__ __forceinline__ int tile_rows(int row, int r1) {
  const int left = r1 - row, tiles = (left + 15) / 16;
  return tiles ? (left + tiles - 1) / tiles : 0;
}

// Chunks per block: where the other operand comes from global memory, two blocks of it have
// to fit the registers.
template <int WT, int NT, bool HS>
constexpr int kDownBlock = HS ? 4 : WT == kBf16 ? 4 / NT : NT == 4 ? 2 : 4;

// h in shared memory (HS): a row of `stride` bytes (an odd number of 64: lanes of two rows
// then read all banks) for each pair's h, two for its high and low parts, zeros past a row's
// end; and such rows of zeros for the columns without a pair.
__host__ __device__ inline int h_stride(int I, int wtype) {
  return (I * (wtype == kBf16 ? 2 : 1) + 255) / 256 * 256 + 64;
}
__host__ __device__ inline int align16(int n) { return (n + 15) / 16 * 16; }
// Bytes of: the pairs' scales; the scales of the CTA's `rows` of every entry; adapters' v.
__host__ __device__ inline int pair_scale_bytes(int P, int wtype) {
  return wtype == kBf16 ? 0 : align16(P * 4);
}
__host__ __device__ inline int row_scale_bytes(int P, int rows, int wtype) {
  return wtype == kBf16 ? 0 : align16(P * rows * 4);
}
__host__ __device__ inline size_t h_bytes(int P, int I, int rows, int r, int wtype) {
  return (size_t)(P + 1) * (wtype == kBf16 ? 2 : 1) * h_stride(I, wtype) +
         pair_scale_bytes(P, wtype) + row_scale_bytes(P, rows, wtype) + (size_t)P * 2 * r * 2;
}
// Rows that down quantises itself: few enough that every CTA doing so costs less than a
// launch in between.
constexpr int kSelfWidth = 1024, kSelfValues = 16384;

// Whole CTA; ends with a barrier, all earlier copies landed.
template <int WT, bool LORA>
__device__ void stage_h(const ExpertsArgs& a, const Routing& rt, unsigned char* hs, float* scale,
                        __nv_bfloat16* v) {
  const int P = a.T * a.k, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int stride = h_stride(a.I, WT), parts = WT == kBf16 ? 2 : 1;
  if (LORA) {              // rows [2p] high, [2p + 1] low parts of v
    const int per = a.lora.r / 8;
    for (int i = tid; i < P * 2 * per; i += blockDim.x) {
      const int row = i / per, at = (i - row * per) * 8, p = row >> 1;
      if (rt.pair_slot[p] < 0 || rt.matrix[p] < 0) continue;
      copy16((unsigned)__cvta_generic_to_shared(v + (size_t)row * a.lora.r + at),
             reinterpret_cast<const uint8_t*>((row & 1 ? a.v_lo : a.v_hi) +
                                              (size_t)p * a.lora.r + at), true);
    }
    copy_commit();
  }
  for (int i = tid * 16; i < stride * parts; i += blockDim.x * 16)
    *reinterpret_cast<uint4*>(hs + (size_t)P * parts * stride + i) = make_uint4(0, 0, 0, 0);
  if (WT != kBf16 && a.self_h) {
    for (int p = warp; p < P; p += blockDim.x >> 5) {
      if (rt.pair_slot[p] < 0) continue;
      float4 x[kSelfWidth / 128];
      unsigned top = 0;
#pragma unroll
      for (int j = 0; j < kSelfWidth / 128; ++j) {
        const int i = j * 128 + lane * 4;
        x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < a.I) x[j] = __ldcg(reinterpret_cast<const float4*>(a.h + (size_t)p * a.I + i));
      }
#pragma unroll
      for (int j = 0; j < kSelfWidth / 128; ++j)
        top = max(top, max(max(abs_bits(x[j].x), abs_bits(x[j].y)),
                           max(abs_bits(x[j].z), abs_bits(x[j].w))));
      const float m = clamp_top(__reduce_max_sync(0xffffffffu, top));
      const RowQuant rq = row_quant<WT>(m);
#pragma unroll
      for (int j = 0; j < kSelfWidth / 128; ++j) {
        const int i = j * 128 + lane * 4;
        if (j * 128 >= stride - 64) break;
        if (i < stride - 64)
          *reinterpret_cast<unsigned*>(hs + (size_t)p * stride + i) =
              i < a.I ? quantise4<WT>(x[j].x, x[j].y, x[j].z, x[j].w, rq) : 0;
      }
      if (lane == 0) scale[p] = quant_scale<WT>(m) * a.weights[p];
    }
  } else {
    const int row_bytes = a.I * Kind<WT>::kItem, per = (stride - 64) / 16;
    for (int i = tid; i < P * parts * per; i += blockDim.x) {
      const int row = i / per, at = (i - row * per) * 16, p = row / parts;
      if (rt.pair_slot[p] < 0) continue;
      const uint8_t* src = WT == kBf16 ? reinterpret_cast<const uint8_t*>(row & 1 ? a.h_lo : a.h_hi)
                                       : a.hq;
      copy16((unsigned)__cvta_generic_to_shared(hs + (size_t)row * stride + at),
             src + (size_t)p * row_bytes + at, at < row_bytes);
    }
    copy_commit();
    if (WT != kBf16)
      for (int p = tid; p < P; p += blockDim.x)
        if (rt.pair_slot[p] >= 0) scale[p] = __ldcg(a.h_scale + p);
  }
  copy_wait<0>();
  __syncthreads();
}

constexpr int kDownMaxThreads = 512;          // (see alone_threads)

template <int NT>
constexpr int kRed = kWarps * 16 * 8 * NT;   // the warps' partial sums

template <int WT, int NT, bool LORA, bool HS>
__global__ void __launch_bounds__(HS && NT < 4 ? kDownMaxThreads : kThreads, 1)
    down_kernel(const __grid_constant__ ExpertsArgs a) {
  using K = Kind<WT>;
  using Acc = typename K::Acc;
  constexpr int KB = kDownBlock<WT, NT, HS>, kParts = WT == kBf16 ? 2 : 1;
  using Stream = Fifo<KB, kDownChunks[HS] / KB>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int P = a.T * a.k;
  const int r0 = (unsigned)a.H * blockIdx.x / gridDim.x;
  const int r1 = (unsigned)a.H * (blockIdx.x + 1) / gridDim.x, rows = r1 - r0;
  Stream fifo(smem);
  constexpr int kFifo = Stream::kStages * Stream::kStage;
  const Routing rt = routing_at(smem + kFifo, P, NT);
  float* red = reinterpret_cast<float*>(smem + kFifo + routing_bytes(P, NT, LORA));
  unsigned char* hs = reinterpret_cast<unsigned char*>(red + kRed<NT>);        // HS
  const int stride = h_stride(a.I, WT);
  unsigned char* after_h = hs + (size_t)(P + 1) * kParts * stride;
  float* scale = reinterpret_cast<float*>(after_h);
  float* row_scale = reinterpret_cast<float*>(after_h + pair_scale_bytes(P, WT));
  __nv_bfloat16* vs = reinterpret_cast<__nv_bfloat16*>(after_h + pair_scale_bytes(P, WT) +
                                                       row_scale_bytes(P, rows, WT));

  // Everything up to the wait reads the call's inputs only.  They are complete: this grid
  // starts once every CTA of the kernels before it has started, the first of them after its
  // own wait.
  release_dependents();
  const FirstReads first(a);
  build_routing<NT, LORA>(a, rt, first, reinterpret_cast<int*>(smem));

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int row_bytes = a.I * K::kItem, lora_bytes = LORA ? a.lora.r * 2 : 0;
  DownUnits units;
  units.plan(rt.entries[0], (row_bytes + KB * 64 - 1) / (KB * 64), LORA ? rt.entries[2] : 0,
             (lora_bytes + KB * 64 - 1) / (KB * 64));
  const int U = units.all();

  // The head of the stream: a block of unit hu of the tile at hrow.
  int hrow = warp < kWarps && warp < U ? r0 : r1, hn = tile_rows(r0, r1), hu = warp, hb = 0, hend = 0;
  int size_a = 0, size_b = 0, hbytes = 0;
  const uint8_t* src = nullptr;
  const auto head_at = [&]() {
    size_a = g < hn ? 16 : 0;
    size_b = g + 8 < hn ? 16 : 0;
    if (!LORA || hu < units.units) {
      hb = units.first(hu);
      hend = units.end(hu);
      hbytes = row_bytes;
      src = a.w2 + ((long long)rt.slot[units.entry(hu)] * a.H + hrow + g) * row_bytes;
    } else {
      hb = 0;
      hend = units.pair_blocks;
      hbytes = lora_bytes;
      src = reinterpret_cast<const uint8_t*>(a.lora.b2) +
            ((long long)rt.matrix[rt.list[hu - units.units]] * a.H + hrow + g) * lora_bytes;
    }
    src += hb * (KB * 64) + q * 16;
  };
  const auto push = [&]() {
    if (hrow < r1) {
      const uint8_t* src_b = src + 8 * hbytes;
      if ((hb + 1) * (KB * 64) <= hbytes) {
        fifo.push_whole(src, size_a, src_b, size_b);
      } else {
        const int left = hbytes - hb * (KB * 64) - q * 16;
        fifo.push(src, size_a ? left : 0, src_b, size_b ? left : 0);
      }
      src += KB * 64;
      if (++hb == hend) {
        hu += kWarps;
        if (hu >= U) {
          hu = warp;
          hrow += hn;
          hn = tile_rows(hrow, r1);
        }
        if (hrow < r1) head_at();
      }
    }
    copy_commit();
  };
  if (hrow < r1) head_at();
  for (int i = 0; i < Stream::kStages; ++i) push();
  if (HS && WT != kBf16) {
    const int n = rt.entries[0] * rows;
    for (int i = tid; i < n; i += blockDim.x) {
      const int e = i / rows;
      row_scale[i] = a.s2[(long long)rt.slot[e] * a.H + r0 + (i - e * rows)];
    }
  }

  grid_dependency_wait();
  if (HS) stage_h<WT, LORA>(a, rt, hs, scale, vs);

  for (int row = r0, n; row < r1; row += n) {
    n = tile_rows(row, r1);
    float acc[NT][4] = {};
    for (int u = warp < kWarps ? warp : U; u < U; u += kWarps) {
      if (LORA && u >= units.units) {
        // an adapted pair: B2's rows with v in its token's column
        const int p = rt.list[u - units.units], t = token_of(a, p);
        const uint4 zero = make_uint4(0, 0, 0, 0);
        float one[4] = {};
        for (int at = 0; at < lora_bytes; at += KB * 64) {
          const unsigned f = fifo.front();
#pragma unroll
          for (int j = 0; j < KB; ++j) {
            const int pos = at + j * 64 + q * 16;
            const bool in = g == (t & 7) && pos < lora_bytes;
            uint4 hi = zero, lo = zero;
            if (HS) {
              if (in) {
                const __nv_bfloat16* from = vs + (size_t)p * 2 * a.lora.r + pos / 2;
                hi = *reinterpret_cast<const uint4*>(from);
                lo = *reinterpret_cast<const uint4*>(from + a.lora.r);
              }
            } else {
              hi = load_or_zero(a.v_hi + (size_t)p * a.lora.r + pos / 2, in);
              lo = load_or_zero(a.v_lo + (size_t)p * a.lora.r + pos / 2, in);
            }
            const uint4 wa = load_shared(f + j * 1024), wb = load_shared(f + j * 1024 + 512);
            chunk_mma_bf16(one, one, wa, wb, hi);
            chunk_mma_bf16(one, one, wa, wb, lo);
          }
          push();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t == nt * 8 + 2 * q + (i & 1)) acc[nt][i] += one[i];
        continue;
      }
      const int e = units.entry(u), end = units.end(u);
      int b = units.first(u);
      const unsigned mask = rt.mask[e];
      const short* col = rt.col + (size_t)e * 8 * NT;
      // 8-bit: scales of rows g, g + 8 and of columns 2q, 2q + 1
      float rf[2] = {}, cf[NT][2] = {};
      if (WT != kBf16) {
        const float* from = HS ? row_scale + e * rows + (row - r0)
                               : a.s2 + (long long)rt.slot[e] * a.H + row;
        if (g < n) rf[0] = from[g];
        if (g + 8 < n) rf[1] = from[g + 8];
      }
      // column g's h (its low part at `low` bytes), in shared or in global memory
      const unsigned char* from[NT];
      bool has[NT], kept[NT][2];     // column g has a pair; columns 2q, 2q + 1
      const long long low = HS ? stride
                               : reinterpret_cast<const unsigned char*>(a.h_lo) -
                                     reinterpret_cast<const unsigned char*>(a.h_hi);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int p = col[nt * 8 + g];
        has[nt] = p >= 0;
        if (HS)
          from[nt] = hs + (p >= 0 ? p : P) * kParts * stride + b * (KB * 64) + q * 16;
        else
          from[nt] = (WT == kBf16 ? reinterpret_cast<const unsigned char*>(a.h_hi) : a.hq) +
                     (long long)p * row_bytes + b * (KB * 64) + q * 16;
        const int p0 = col[nt * 8 + 2 * q], p1 = col[nt * 8 + 2 * q + 1];
        kept[nt][0] = p0 >= 0;
        kept[nt][1] = p1 >= 0;
        if (WT != kBf16) {
          if (p0 >= 0) cf[nt][0] = HS ? scale[p0] : __ldcg(a.h_scale + p0);
          if (p1 >= 0) cf[nt][1] = HS ? scale[p1] : __ldcg(a.h_scale + p1);
        }
      }
      // not HS: the operand of the next block is on its way while this one is multiplied
      uint4 next[HS ? 1 : NT][HS ? 1 : KB][HS ? 1 : kParts];
      const auto fetch = [&](int b) {
#pragma unroll
        for (int nt = 0; nt < (HS ? 0 : NT); ++nt) {
          if (NT > 1 && !(mask >> nt & 1)) continue;
          const int left = has[nt] && b < end ? row_bytes - b * (KB * 64) - q * 16 : 0;
#pragma unroll
          for (int j = 0; j < KB; ++j)
#pragma unroll
            for (int part = 0; part < kParts; ++part)
              next[nt][j][part] = load_or_zero(from[nt] + part * low + j * 64, left > j * 64);
          from[nt] += KB * 64;
        }
      };
      if (!HS) fetch(b);
      constexpr int kN = kSumParts<WT, NT>;
      Acc sum[kN][NT][4] = {};
      for (; b < end; ++b) {
        uint4 now[HS ? 1 : NT][HS ? 1 : KB][HS ? 1 : kParts];
        if (!HS) {
#pragma unroll
          for (int nt = 0; nt < (HS ? 0 : NT); ++nt)
#pragma unroll
            for (int j = 0; j < KB; ++j)
#pragma unroll
              for (int part = 0; part < kParts; ++part) now[nt][j][part] = next[nt][j][part];
          fetch(b + 1);
        }
        const unsigned f = fifo.front();
        uint4 wa[KB], wb[KB];
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          wa[j] = load_shared(f + j * 1024);
          wb[j] = load_shared(f + j * 1024 + 512);
        }
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          Wide fa, fb;
          if (WT == kFp8) { fa = widen(wa[j]); fb = widen(wb[j]); }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (NT > 1 && !(mask >> nt & 1)) continue;
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              uint4 v;
              if constexpr (HS) v = *reinterpret_cast<const uint4*>(from[nt] + part * stride + j * 64);
              else v = now[nt][j][part];
              const int c = 2 * (WT == kBf16 ? part : j & 1);
              if constexpr (WT == kBf16) chunk_mma_bf16(sum[c][nt], sum[c + 1][nt], wa[j], wb[j], v);
              if constexpr (WT == kInt8)
                chunk_mma_s8(sum[c % kN][nt], sum[(c + 1) % kN][nt], wa[j], wb[j], v);
              if constexpr (WT == kFp8) chunk_mma_fp8(sum, nt, fa, fb, v);
            }
          }
        }
        if (HS)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            if (has[nt]) from[nt] += KB * 64;
        push();
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (NT > 1 && !(mask >> nt & 1)) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (a column without a pair is zeros, but zero times an infinite weight is a NaN)
          if (!kept[nt][i & 1]) continue;
          const Acc v = whole(sum, nt, i);
          acc[nt][i] += WT == kBf16 ? (float)v : (float)v * (rf[i >> 1] * cf[nt][i & 1]);
        }
      }
    }
    float* mine = red + warp * 16 * 8 * NT;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (warp >= kWarps) break;
      const int col = nt * 8 + 2 * q;
      mine[g * 8 * NT + col] = acc[nt][0];
      mine[g * 8 * NT + col + 1] = acc[nt][1];
      mine[(g + 8) * 8 * NT + col] = acc[nt][2];
      mine[(g + 8) * 8 * NT + col + 1] = acc[nt][3];
    }
    __syncthreads();
    for (int o = tid; o < 16 * a.T; o += blockDim.x) {
      const int i = o & 15, t = o >> 4;
      if (i >= n) continue;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) s += red[(k * 16 + i) * 8 * NT + t];
      a.out[t * a.ldo + row + i] = __float2bfloat16(s);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// route: a cluster of CTAs takes TT tokens.  Each CTA scores its share of the experts, a warp
// EX at a time, straight from the router's weight; the scores meet in the first CTA's shared
// memory, where a warp per token picks.  One launch, bound by latency: reading x and the
// weight, summing, k dependent choices.
//
// Scores are sums in 64 bits of exact products, in one order for every call: only experts whose
// scores agree to some 15 digits could change places with another order.  A bf16 becomes a
// double by moving its bits: shifted by 3 into a double's high word, its exponent reads as
// e - 896 (subnormals included).  x is brought back to its own exponent when it is staged, the
// weights are not: sums are multiplied by 2^896 at the end, which is exact.  (The conversion
// instruction runs at a quarter of the 64-bit products' rate.)  A sum is done again with plain
// conversions where the move does not hold: with an infinity or a NaN among its operands, a
// subnormal in x, or a result so small that products may have underflowed.

constexpr int kRouteThreads = 512, kRouteWarps = kRouteThreads / 32;
constexpr int kRouteStages = 8;                  // of a warp, 256 columns of its experts each

struct RouteArgs {
  const __nv_bfloat16 *x, *gate;
  const float* bias;
  float* weights;
  int* ids;
  long long ldx;
  int T, H, E, k, sigmoid, renorm;
  float scale;
};

// The two bf16 of `u` times 2^-896 (low half, high half).
__device__ __forceinline__ double moved_low(unsigned u) {
  return __hiloint2double(((int)(u << 16) >> 3) & 0x8fffffff, 0);
}
__device__ __forceinline__ double moved_high(unsigned u) {
  return __hiloint2double(((int)u >> 3) & 0x8fffe000, 0);
}
// The high word of the double that the bf16 in the high half of `u` is (normal or zero).
__device__ __forceinline__ unsigned high_word(unsigned u) {
  return (u & 0x7f800000u) ? (((int)u >> 3) & 0x8fffe000) + (896 << 20) : 0;
}

// One dot product with plain conversions: the warp's.
__device__ __noinline__ double plain_dot(const __nv_bfloat16* w, const __nv_bfloat16* x, int H) {
  double s = 0.0;
  for (int i = (threadIdx.x & 31); i < H; i += 32)
    s += (double)__bfloat162float(w[i]) *
         (double)__bfloat162float(x[i]);
#pragma unroll
  for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  return s;
}

__device__ __forceinline__ unsigned remote_shared(const void* p, int rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(r)
      : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_remote(unsigned at, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory");
}

template <int TT, int EX>
__global__ void __launch_bounds__(kRouteThreads, 1) route_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  using Stream = Fifo<1, kRouteStages, kRouteThreads>;
  Stream fifo(smem);
  unsigned* xs = reinterpret_cast<unsigned*>(smem + kRouteStages * Stream::kStage);  // [TT][H]
  double* score = reinterpret_cast<double*>(xs + TT * a.H);        // [TT][E], first CTA
  unsigned long long* key = reinterpret_cast<unsigned long long*>(score + TT * a.E);  // likewise
  __shared__ int odd[TT], some[TT];       // x has an inf, a NaN or a subnormal; x is not all zeros
  unsigned rank, size;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int t0 = blockIdx.x / size * TT;
  const int n = min(TT, a.T - t0);

  grid_dependency_wait();
  release_dependents();

  // The warp's experts, EX at a time, 256 columns at a step, through its FIFO.
  const int share = (a.E + (int)size - 1) / (int)size;
  const int e0 = (int)rank * share, e1 = min(a.E, e0 + share);
  int he = e0 + warp * EX, hi = 0;
  const auto push = [&]() {
    if (he < e1) {
      const uint8_t* w = reinterpret_cast<const uint8_t*>(a.gate + (long long)he * a.H + hi + lane * 8);
      const int left = hi + lane * 8 < a.H ? 16 : 0;
      fifo.push(w, left, w + (he + 1 < e1 ? 2LL * a.H : 0), EX == 2 ? left : 0);
      hi += 256;
      if (hi >= a.H) {
        hi = 0;
        he += kRouteWarps * EX;
      }
    }
    copy_commit();
  };
  for (int i = 0; i < kRouteStages; ++i) push();
  // the first CTA's shared memory is there to be written once its threads run
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  if (tid < TT) odd[tid] = some[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    for (int i = tid * 8; i < a.H; i += kRouteThreads * 8) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (t < n) v = *reinterpret_cast<const uint4*>(a.x + (t0 + t) * a.ldx + i);
      const unsigned u[4] = {v.x, v.y, v.z, v.w};
      unsigned to[8];
      bool special = top_bits(v) >= 0x7f800000u;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        to[2 * m] = high_word(u[m] << 16);
        to[2 * m + 1] = high_word(u[m] & 0xffff0000u);
        special |= ((u[m] & 0x7f80u) == 0 && (u[m] & 0x7fu)) ||
                   ((u[m] & 0x7f800000u) == 0 && (u[m] & 0x7f0000u));
      }
      // of every eight columns four in either half of the row: lanes read 16 bytes apart
      unsigned* at = xs + t * a.H + i / 2;
      *reinterpret_cast<uint4*>(at) = make_uint4(to[0], to[1], to[2], to[3]);
      *reinterpret_cast<uint4*>(at + a.H / 2) = make_uint4(to[4], to[5], to[6], to[7]);
      if (special) odd[t] = 1;
      if (top_bits(v)) some[t] = 1;
    }
  }
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");

  for (int e = e0 + warp * EX; e < e1; e += kRouteWarps * EX) {
    const bool two = e + 1 < e1;
    double acc[EX][TT][2] = {};                  // (even and odd columns: shorter chains)
    unsigned top[EX] = {};
    for (int i = lane * 8; i - lane * 8 < a.H; i += 256) {
      const unsigned f = fifo.front();
      unsigned u[EX][4];
#pragma unroll
      for (int x = 0; x < EX; ++x) {
        const uint4 w = load_shared(f + x * 512);
        u[x][0] = w.x; u[x][1] = w.y; u[x][2] = w.z; u[x][3] = w.w;
#pragma unroll
        for (int m = 0; m < 4; ++m) top[x] = __vmaxu2(top[x], u[x][m] & 0x7fff7fffu);
      }
      unsigned v[TT][8];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        // (past a row's end the weights are zeros and x must be finite: any of its words)
        const unsigned* from = xs + t * a.H + (i < a.H ? i : 0) / 2;
        const uint4 v0 = *reinterpret_cast<const uint4*>(from);
        const uint4 v1 = *reinterpret_cast<const uint4*>(from + a.H / 2);
        v[t][0] = v0.x; v[t][1] = v0.y; v[t][2] = v0.z; v[t][3] = v0.w;
        v[t][4] = v1.x; v[t][5] = v1.y; v[t][6] = v1.z; v[t][7] = v1.w;
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
#pragma unroll
        for (int x = 0; x < EX; ++x) {
          const double lo = moved_low(u[x][m]), hi = moved_high(u[x][m]);
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            acc[x][t][0] = fma(__hiloint2double(v[t][2 * m], 0), lo, acc[x][t][0]);
            acc[x][t][1] = fma(__hiloint2double(v[t][2 * m + 1], 0), hi, acc[x][t][1]);
          }
        }
      }
      push();
    }
#pragma unroll
    for (int x = 0; x < EX; ++x) {
      const bool bad = __any_sync(0xffffffffu, (top[x] & 0x7fffu) >= 0x7f80u || top[x] >= 0x7f800000u);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        double s = acc[x][t][0] + acc[x][t][1];
#pragma unroll
        for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= 0x1p896;
        if (t < n && (bad || odd[t] || (fabs(s) < 0x1p-64 && some[t])))
          s = plain_dot(a.gate + (long long)(e + (two ? x : 0)) * a.H, a.x + (t0 + t) * a.ldx, a.H);
        if (lane == 0 && (x == 0 || two))
          store_remote(remote_shared(score + t * a.E + e + x, 0), s + 0.0);   // -0 becomes 0
      }
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned; barrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
  if (rank != 0) return;

  // ---- a warp picks for its token ------------------------------------------------------
  // What is compared: the value's bits, made to order as unsigned; 0 = not to be picked.
  for (int i = tid; i < n * a.E; i += kRouteThreads) {
    double v = score[i];
    if (a.sigmoid) v = 1.0 / (1.0 + exp(-v)) + (a.bias ? (double)a.bias[i % a.E] : 0.0);
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    const bool never = v != v || v == -INFINITY;
    key[i] = never ? 0 : b >> 63 ? ~b : b | 1ull << 63;
  }
  __syncthreads();
  if (warp >= n) return;
  const int tok = t0 + warp;
  score += warp * a.E;
  key += warp * a.E;
  // A lane's best two of its experts; they are looked for again when both are picked.
  unsigned long long best = 0, second = 0;
  int best_e = INT_MAX, second_e = INT_MAX;
  const auto scan = [&]() {
    best = second = 0;
    best_e = second_e = INT_MAX;
    for (int e = lane; e < a.E; e += 32) {             // ascending: the first of equals stays
      const unsigned long long o = key[e];
      if (o > best) {
        second = best;
        second_e = best_e;
        best = o;
        best_e = e;
      } else if (o > second) {
        second = o;
        second_e = e;
      }
    }
  };
  scan();
  int mine = -1;                // lane r < k: the r-th pick
  for (int r = 0; r < a.k; ++r) {
    const unsigned hi = (unsigned)(best >> 32), top_hi = __reduce_max_sync(0xffffffffu, hi);
    const bool in = hi == top_hi;
    const unsigned lo = in ? (unsigned)best : 0, top_lo = __reduce_max_sync(0xffffffffu, lo);
    if ((top_hi | top_lo) == 0) break;
    const int e = (int)__reduce_min_sync(0xffffffffu,
                                         in && lo == top_lo ? (unsigned)best_e : 0xffffffffu);
    if (lane == r) mine = e;
    if ((e & 31) == lane) {
      key[e] = 0;               // picked
      best = second;
      best_e = second_e;
      second = 0;
      second_e = INT_MAX;
      if (best == 0) scan();
    }
  }
  const double s = mine >= 0 ? score[mine] : 0.0;
  double weight = 0.0;
  if (a.sigmoid) {
    if (mine >= 0) weight = 1.0 / (1.0 + exp(-s));
  } else {
    // the first pick is the largest; renormalised, the sum over all experts cancels
    const double top = __shfl_sync(0xffffffffu, s, 0);
    if (mine >= 0) weight = exp(s - top);
    if (!a.renorm) {
      double all = 0.0;
      for (int e = lane; e < a.E; e += 32)
        if (score[e] == score[e]) all += exp(score[e] - top);
#pragma unroll
      for (int off = 16; off; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
      weight /= all;
    }
  }
  if (a.renorm) {
    double total = weight;
#pragma unroll
    for (int off = 16; off; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (total != 0.0) weight /= total;           // (a NaN, from a score of +inf, is one in all)
  }
  if (lane < a.k) {
    a.weights[(long long)tok * a.k + lane] = mine >= 0 ? (float)(weight * (double)a.scale) : 0.f;
    a.ids[(long long)tok * a.k + lane] = mine;
  }
}

// ---------------------------------------------------------------------------------------
// host side

std::atomic<int> g_sms[kMaxDevices];

int device_sms(int* dev, int* sms) {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= kMaxDevices)
    return (int)cudaErrorInvalidDevice;
  int n = g_sms[d].load(std::memory_order_relaxed);
  if (n == 0) {
    const cudaError_t err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d);
    if (err != cudaSuccess) return (int)err;
    g_sms[d].store(n, std::memory_order_relaxed);
  }
  *dev = d;
  *sms = n;
  return 0;
}

// Raise a kernel's dynamic shared memory limit once per device (`done`: its own flags).
template <typename Kernel>
cudaError_t allow_smem(Kernel fn, std::atomic<bool>* done, int dev) {
  if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  int optin = 0;
  cudaError_t err = cudaDeviceGetAttribute(&optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
  if (err != cudaSuccess) return err;
  cudaFuncAttributes fa{};
  err = cudaFuncGetAttributes(&fa, fn);
  if (err != cudaSuccess) return err;
  err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             optin - (int)fa.sharedSizeBytes);
  // An SM is not repartitioned while a CTA is on it: without this the partition that up needs
  // keeps down off the SM until up has left.
  if (err == cudaSuccess)
    err = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                               cudaSharedmemCarveoutMaxShared);
  if (err == cudaSuccess) done[dev].store(true, std::memory_order_release);
  return err;
}

template <typename... Params, typename... Args>
int launch(void (*fn)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
           int cluster, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, fn, Params(args)...);
}

// An SM takes one CTA of up and one of down, and not two of a kind (two on one SM and none on
// another was 25 us to 18 for one token in bf16): two of up do not fit its shared memory, two
// of down not its registers, for which down is launched with idle warps beside its kWarps
// (they help to stage h).
constexpr size_t kUpAlone = (228 * 1024) / 2 - 1024 + 16;

template <typename Kernel>
int alone_threads(Kernel fn, std::atomic<int>& known, int* threads) {
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaFuncAttributes fa{};
    const cudaError_t err = cudaFuncGetAttributes(&fa, fn);
    if (err != cudaSuccess) return (int)err;
    n = (32768 / ((fa.numRegs + 7) / 8 * 8) / 32 + 1) * 32;
    n = n < kThreads ? kThreads : n > kDownMaxThreads ? kDownMaxThreads : n;
    known.store(n, std::memory_order_relaxed);
  }
  *threads = n;
  return 0;
}

int chunk_columns(int wtype) { return wtype == kBf16 ? 32 : 64; }

size_t staged_bytes(int T, int H, int wtype) {
  const int cc = 4 * chunk_columns(wtype);
  return (size_t)((H + cc - 1) / cc) * 256 * T;
}

int column_tiles(int T) { return T <= 8 ? 1 : T <= 16 ? 2 : 4; }

// Shared memory of up_kernel without the copy of x, and of down_kernel without h.
size_t up_bytes(int P, int NT, bool lora) {
  return kUpFifo + routing_bytes(P, NT, lora) + kMaxTokens * 4;
}
size_t down_bytes(int P, int NT, bool lora, bool hs) {
  return down_fifo(hs) + routing_bytes(P, NT, lora) + (size_t)kWarps * 16 * 8 * NT * 4;
}

// Does the copy of x fit beside it?  bf16 rows are read from L1 / L2 where it does not.
bool fits_staged(int T, int k, int H, int wtype) {
  const int NT = column_tiles(T);
  return up_bytes(T * k, NT, true) + staged_bytes(T, H, wtype) + 2 * kMaxTokens * 4 <= kSmem;
}

// Tokens of one launch: as many as fit the column tiles, the pair tables and (8-bit
// weights, which are multiplied by staged rows only) the shared memory.
int tokens_per_launch(int T, int k, int H, int wtype) {
  int n = T < kMaxTokens ? T : kMaxTokens;
  while (n > 1 && (n * k > kMaxPairs || n * k * 8 * column_tiles(n) > kMaxCols ||
                   (wtype != kBf16 && !fits_staged(n, k, H, wtype))))
    --n;
  return n;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// The workspace's parts for `tokens` tokens of k experts; returns its size.
size_t carve(ExpertsArgs* a, unsigned char* base, int tokens, int k, int H, int I, int wtype,
             int r) {
  const size_t pairs = (size_t)tokens * k;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    unsigned char* p = base ? base + at : nullptr;
    at += align256(bytes);
    return p;
  };
  if (wtype == kBf16) {
    a->h_hi = reinterpret_cast<__nv_bfloat16*>(take(pairs * I * 2));
    a->h_lo = reinterpret_cast<__nv_bfloat16*>(take(pairs * I * 2));
  } else {
    a->h = reinterpret_cast<float*>(take(pairs * I * 4));
    a->hq = take(pairs * I);
    a->h_scale = reinterpret_cast<float*>(take(pairs * 4));
    a->xq = take((size_t)tokens * H);
    a->x_scale = reinterpret_cast<float*>(take((size_t)tokens * 4));
  }
  if (r) {
    a->u_hi = reinterpret_cast<__nv_bfloat16*>(take(pairs * 2 * r * 2));
    a->u_lo = reinterpret_cast<__nv_bfloat16*>(take(pairs * 2 * r * 2));
    a->v_hi = reinterpret_cast<__nv_bfloat16*>(take(pairs * r * 2));
    a->v_lo = reinterpret_cast<__nv_bfloat16*>(take(pairs * r * 2));
  }
  return at;
}

template <int WT, int NT, bool LORA>
int run_layer(ExpertsArgs a, cudaStream_t stream) {
  static std::atomic<bool> done_up[2][kMaxDevices], done_down[2][kMaxDevices];
  static std::atomic<int> alone[kMaxDevices];
  int dev = 0, sms = 0;
  int rc = device_sms(&dev, &sms);
  if (rc != 0) return rc;
  // only bf16 rows may be read where they are
  const bool staged = WT != kBf16 || fits_staged(a.T, a.k, a.H, WT);
  const auto up = staged ? up_kernel<WT, NT, LORA, true> : up_kernel<WT, NT, LORA, WT != kBf16>;
  cudaError_t err = allow_smem(up, done_up[staged], dev);
  const int P = a.T * a.k;
  size_t down_smem = down_bytes(P, NT, LORA, true) + h_bytes(P, a.I, (a.H + sms - 1) / sms, a.lora.r, WT);
  const bool hs = down_smem <= kSmem;
  a.self_h = WT != kBf16 && hs && a.I <= kSelfWidth && P * a.I <= kSelfValues;
  if (!hs) down_smem = down_bytes(P, NT, LORA, false);
  const auto down = hs ? down_kernel<WT, NT, LORA, true> : down_kernel<WT, NT, LORA, false>;
  if (err == cudaSuccess) err = allow_smem(down, done_down[hs], dev);
  if (err != cudaSuccess) return (int)err;
  if (LORA || a.prepared) {
    const int grid = (a.prepared ? a.T : 0) +
                     (LORA ? P * ((2 * a.lora.r + kWarps - 1) / kWarps) : 0);
    rc = launch(prep_kernel<WT, LORA>, dim3(grid), kThreads, 0, stream, 1, a);
    if (rc != 0) return rc;
  }
  rc = launch(up, dim3(sms), kThreads,
              max(kUpAlone, up_bytes(P, NT, LORA) + (staged ? staged_bytes(a.T, a.H, WT) : 0)),
              stream, 1, a);
  if (rc != 0) return rc;
  const bool quantise = WT != kBf16 && !a.self_h;
  if (LORA || quantise) {
    const int grid = (quantise ? P : 0) + (LORA ? P * ((a.lora.r + kWarps - 1) / kWarps) : 0);
    rc = launch(mid_kernel<WT, LORA>, dim3(grid), kThreads, 0, stream, 1, a);
    if (rc != 0) return rc;
  }
  int threads = kThreads;
  if (hs && NT < 4) {
    rc = alone_threads(down, alone[dev], &threads);
    if (rc != 0) return rc;
  }
  return launch(down, dim3(sms), threads, down_smem, stream, 1, a);
}

template <int WT, bool LORA>
int run_tiles(const ExpertsArgs& a, cudaStream_t stream) {
  switch (column_tiles(a.T)) {
    case 1: return run_layer<WT, 1, LORA>(a, stream);
    case 2: return run_layer<WT, 2, LORA>(a, stream);
    default: return run_layer<WT, 4, LORA>(a, stream);
  }
}

template <int WT>
int run_type(const ExpertsArgs& a, cudaStream_t stream) {
  return a.lora.r ? run_tiles<WT, true>(a, stream) : run_tiles<WT, false>(a, stream);
}

size_t route_bytes(int TT, int H, int E) {
  return (size_t)kRouteStages * kRouteThreads * 32 + (size_t)TT * (H * 4 + 16 * (size_t)E);
}

template <int TT, int EX>
int run_route(const RouteArgs& a, cudaStream_t stream, int cluster) {
  static std::atomic<bool> done[kMaxDevices];
  static std::atomic<int> wide[kMaxDevices];     // 1: clusters of 16 run here, 2: they do not
  int dev = 0, sms = 0;
  const int rc = device_sms(&dev, &sms);
  if (rc != 0) return rc;
  const auto fn = route_kernel<TT, EX>;
  cudaError_t err = allow_smem(fn, done, dev);
  if (err != cudaSuccess) return (int)err;
  const size_t smem = route_bytes(TT, a.H, a.E);
  if (cluster > 8 && wide[dev].load(std::memory_order_relaxed) == 0) {
    err = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (err != cudaSuccess) return (int)err;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(kRouteThreads);
    cfg.dynamicSmemBytes = kSmem - 64;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    wide[dev].store(n > 0 ? 1 : 2, std::memory_order_relaxed);
  }
  if (cluster > 8 && wide[dev].load(std::memory_order_relaxed) == 2) cluster = 8;
  const long long groups = ((long long)a.T + TT - 1) / TT;
  return launch(fn, dim3((unsigned)(groups * cluster)), kRouteThreads, smem, stream, cluster, a);
}

template <int EX>
int run_tokens(const RouteArgs& a, cudaStream_t stream, int tt, int cluster) {
  return tt == 1   ? run_route<1, EX>(a, stream, cluster)
         : tt == 2 ? run_route<2, EX>(a, stream, cluster)
                   : run_route<4, EX>(a, stream, cluster);
}

bool misaligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

bool shape_ok(int T, int k, int H, int I, int wtype) {
  if (T < 0 || k <= 0 || k > EXPERT_CACHE_EXPERTS_MAX_TOPK) return false;
  if (wtype < kBf16 || wtype > kFp8) return false;
  const int vec = wtype == kBf16 ? 8 : 16;
  return H > 0 && H <= EXPERT_CACHE_EXPERTS_MAX_DIM && H % vec == 0 && I > 0 &&
         I <= EXPERT_CACHE_EXPERTS_MAX_DIM && I % vec == 0;
}

int experts_checked(ExpertsArgs a, int wtype, void* workspace, long workspace_bytes,
                    cudaStream_t stream) {
  const int T = a.T, r = a.lora.r;
  if (!shape_ok(T, a.k, a.H, a.I, wtype)) return -1;
  if (a.S <= 0 || a.S > EXPERT_CACHE_MAX_SLOTS || a.n_map < 0 || (a.map && a.n_map == 0))
    return -1;
  if (a.ldx < a.H || a.ldx % 8 || a.ldo < a.H) return -1;
  if (T == 0) return 0;
  if (!a.x || !a.ids || !a.weights || !a.w13 || !a.w2 || !a.out) return -1;
  if ((wtype != kBf16) != (a.s13 != nullptr) || (wtype != kBf16) != (a.s2 != nullptr)) return -1;
  if (misaligned(a.x, 16) || misaligned(a.w13, 16) || misaligned(a.w2, 16) ||
      misaligned(a.out, 2) || misaligned(a.s13, 4) || misaligned(a.s2, 4) ||
      misaligned(a.ids, 4) || misaligned(a.weights, 4) || misaligned(a.map, 4))
    return -1;
  const int per = tokens_per_launch(T, a.k, a.H, wtype);
  const size_t need = carve(&a, nullptr, per, a.k, a.H, a.I, wtype, r);
  if (!workspace || misaligned(workspace, 256) || workspace_bytes < (long)need) return -1;
  carve(&a, static_cast<unsigned char*>(workspace), per, a.k, a.H, a.I, wtype, r);
  const ExpertsArgs all = a;
  for (long long t = 0; t < T; t += per) {       // (T may lie next to the end of int)
    a.T = T - t < per ? (int)(T - t) : per;
    a.x = all.x + t * all.ldx;
    a.out = all.out + t * all.ldo;
    a.ids = all.ids + t * all.k;
    a.weights = all.weights + t * all.k;
    if (r) a.lora.index = all.lora.index + t;
    a.prepared = wtype != kBf16 && (long long)a.T * a.H > kSelfX;
    const int rc = wtype == kBf16   ? run_type<kBf16>(a, stream)
                   : wtype == kInt8 ? run_type<kInt8>(a, stream)
                                    : run_type<kFp8>(a, stream);
    if (rc != 0) return rc;
  }
  return 0;
}

ExpertsArgs experts_args(const void* x, int T, int ldx, int H, const int* ids,
                         const float* weights, int k, const int* expert_map, int n_map,
                         const void* w13, const float* w13_scale, const void* w2,
                         const float* w2_scale, int S, int I, void* out, int ldo) {
  ExpertsArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.ids = ids;
  a.weights = weights;
  a.map = expert_map;
  a.w13 = static_cast<const uint8_t*>(w13);
  a.w2 = static_cast<const uint8_t*>(w2);
  a.s13 = w13_scale;
  a.s2 = w2_scale;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ldx = ldx;
  a.ldo = ldo;
  a.T = T;
  a.k = k;
  a.per_k = k > 0 ? 1.f / (float)k : 0.f;
  a.H = H;
  a.I = I;
  a.S = S;
  a.n_map = n_map;
  return a;
}

}  // namespace

extern "C" {

int expert_cache_experts_workspace(int T, int k, int H, int I, int wtype, int r, long* bytes) {
  if (!shape_ok(T, k, H, I, wtype) || bytes == nullptr) return -1;
  if (r < 0 || r > EXPERT_CACHE_LORA_MAX_RANK || r % 8) return -1;
  ExpertsArgs a{};
  *bytes = T == 0 ? 0
                  : (long)carve(&a, nullptr, tokens_per_launch(T, k, H, wtype), k, H, I, wtype, r);
  return 0;
}

int expert_cache_experts(const void* x, int T, int ldx, int H, const int* ids,
                         const float* weights, int k, const int* expert_map, int n_map,
                         const void* w13, const float* w13_scale, const void* w2,
                         const float* w2_scale, int wtype, int S, int I, void* out, int ldo,
                         void* workspace, long workspace_bytes, cudaStream_t stream) {
  return experts_checked(experts_args(x, T, ldx, H, ids, weights, k, expert_map, n_map, w13,
                                      w13_scale, w2, w2_scale, S, I, out, ldo),
                         wtype, workspace, workspace_bytes, stream);
}

int expert_cache_experts_lora(const void* x, int T, int ldx, int H, const int* ids,
                              const float* weights, int k, const int* expert_map, int n_map,
                              const void* w13, const float* w13_scale, const void* w2,
                              const float* w2_scale, int wtype, int S, int I,
                              const int* adapter, const void* a13, const void* b13,
                              const void* a2, const void* b2, const float* scaling, int L,
                              int E, int r, void* out, int ldo, void* workspace,
                              long workspace_bytes, cudaStream_t stream) {
  ExpertsArgs a = experts_args(x, T, ldx, H, ids, weights, k, expert_map, n_map, w13, w13_scale,
                               w2, w2_scale, S, I, out, ldo);
  if (L <= 0 || E <= 0 || (long long)L * E > INT_MAX || r <= 0 || r > EXPERT_CACHE_LORA_MAX_RANK || r % 8) return -1;
  if (!adapter || !a13 || !b13 || !a2 || !b2 || !scaling) return -1;
  if (misaligned(a13, 16) || misaligned(b13, 16) || misaligned(a2, 16) || misaligned(b2, 16) ||
      misaligned(adapter, 4) || misaligned(scaling, 4))
    return -1;
  a.lora.index = adapter;
  a.lora.a13 = static_cast<const __nv_bfloat16*>(a13);
  a.lora.b13 = static_cast<const __nv_bfloat16*>(b13);
  a.lora.a2 = static_cast<const __nv_bfloat16*>(a2);
  a.lora.b2 = static_cast<const __nv_bfloat16*>(b2);
  a.lora.scaling = scaling;
  a.lora.L = L;
  a.lora.E = E;
  a.lora.r = r;
  return experts_checked(a, wtype, workspace, workspace_bytes, stream);
}

int expert_cache_route(const void* x, int T, int ldx, int H, const void* gate_w, int E, int k,
                       int scoring, int renormalize, const float* bias, float scale,
                       float* out_weights, int* out_ids, cudaStream_t stream) {
  if (T < 0 || H <= 0 || H % 8 || H > EXPERT_CACHE_PREGATE_MAX_HIDDEN || ldx < H || ldx % 8)
    return -1;
  if (E <= 0 || E > EXPERT_CACHE_PREGATE_MAX_EXPERTS || k <= 0 || k > E ||
      k > EXPERT_CACHE_EXPERTS_MAX_TOPK)
    return -1;
  if (scoring < 0 || scoring > 1 || (scoring == 0 && bias != nullptr)) return -1;
  if (misaligned(x, 16) || misaligned(gate_w, 16) || misaligned(bias, 4) ||
      misaligned(out_weights, 4) || misaligned(out_ids, 4))
    return -1;
  if (T == 0) return 0;
  if (!x || !gate_w || !out_weights || !out_ids) return -1;
  RouteArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.gate = static_cast<const __nv_bfloat16*>(gate_w);
  a.bias = bias;
  a.weights = out_weights;
  a.ids = out_ids;
  a.ldx = ldx;
  a.T = T;
  a.H = H;
  a.E = E;
  a.k = k;
  a.sigmoid = scoring;
  a.renorm = renormalize != 0;
  a.scale = scale;
  // Tokens a cluster: as few as keep the clusters to one wave, of which the device holds 15
  // with 8 CTAs each (32 tokens of 256 experts of 4096: 28.4 us in 16 clusters, 21.5 in 8).
  // Clusters of 16 CTAs, of which it holds 7, while there are few and experts for them (one
  // token of 128 experts 7.2 -> 6.1 us; 53 tokens of 61 experts 8.2 -> 9.2).  An expert a
  // warp at a time where that is enough for the CTA's share.
  int tt = T <= 4 ? 1 : T <= 30 ? 2 : 4;
  while (tt > 1 && route_bytes(tt, H, E) > kSmem - 64) tt /= 2;
  const long long groups = ((long long)T + tt - 1) / tt;
  if (groups * 8 > INT_MAX) return -1;           // CTAs of one launch
  const int cluster = E >= 128 && groups <= 4 ? 16 : 8;
  return E <= cluster * kRouteWarps ? run_tokens<1>(a, stream, tt, cluster)
                                    : run_tokens<2>(a, stream, tt, cluster);
}

}  // extern "C"
