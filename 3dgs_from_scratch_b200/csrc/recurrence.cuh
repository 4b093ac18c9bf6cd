// recurrence.cuh -- the gated linear recurrence's pieces, shared by its forward
// and backward kernels (recurrence_forward.cu, recurrence_backward.cu).
//
// The operator: over every sequence of a packed (rows, C) tensor,
//   h_t = g_t h_{t-1} + x_t,  h_{-1} = initial,
// each gate shared by D = C / G consecutive channels. It is linear, so a run
// of rows acts on the state before it as h -> P h + L (P the product of its
// gates, L its result from a zero state), and runs compose:
//   (P2, L2) after (P1, L1) = (P1 P2, P2 L1 + L2).
// Gates may lie above 1, and a few hundred of 2 take P out of fp32's range
// although no state is anywhere near (a state of 0, or a small one), where
// inf * 0 would make a NaN of it. So each chunk's P is also kept with an
// exponent of its own, and the scan over the chunks goes by that form wherever a
// chunk's product passes 1, or 2^11 on its way. Where none does, products under
// 2^-126 count as 0, and nothing makes what is lost of a state larger again than
// 2^-115 of it.
//
// Memory is what bounds both directions (a handful of operations an element).
// So a thread does nothing but walk rows: it owns V channels of a chunk of
// rows, keeps the state in registers and reads and writes each row
// once, a batch of rows in flight at a time. Chunks are as long as leaves
// enough threads to fill the device. Sequence bounds need no chunks of their
// own: at a sequence's first row the initial state takes the place of the
// state so far, so ragged sequences cost what their rows cost.
//
// Where a sequence reaches over a chunk's end, the state that enters the next
// chunk has to be known first. That takes two small launches before the walk:
// the map (P, L) of what the chunk holds of its last sequence, which reads those
// rows once more (nothing where sequences end with chunks, few rows where
// sequences are short), and a scan over the chunks' maps. Even sequences are cut
// into chunks of whole sequences where there are enough of them. An earlier
// form kept tiles in registers and chained them in one launch, which reads
// everything once; its folds, barriers and waits cost more than the second read
// (8 x 2048 rows x 1024 channels, bf16 with fp32 gates: forward 74 us, backward
// 183 us in one kernel each, against 48 and 85 us in three).
// What the walks reach of the 6.46 TB/s that a copy reaches: 262,144 rows x 64
// channels fp32 forward 31 us (0.66), backward 51 us (0.69); 65,536 sequences of
// 30 rows x 16 channels 63 (0.72) and 113 us (0.68).
//
// Nothing here depends on the order in which blocks run, so every run of the
// program rounds alike.
//
// "Logical" rows run in the direction of the recurrence: with `reverse` the
// logical row t is the row rows - 1 - t of the tensor. The backward's chain runs
// against it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cfloat>

#include "gs_common.cuh"

namespace gs {
namespace scan {

constexpr int kThreads = 256;
constexpr int kBatch = 8;  // rows in flight, and from one kept state to the next
// Threads on an SM that a chunk length aims at: with 640 too few loads are in
// flight, with 2560 chunks are so short that the chain costs more (forward and
// backward of 8 x 2048 x 1024: 212, 184 and 189 us, of 524,288 x 35: 410, 402 and
// 495 us with 640, 1280 and 2560).
constexpr int kFill = 1280;
// Rows that a thread walks in the time that the chain's two launches take (12 us).
constexpr int kShort = 128;

// How a problem is cut. It depends on the sizes and types alone, never on
// pointers, so that the backward finds the states that the forward kept.
struct Plan {
  int vec;             // channels of a thread: adjacent ones, read as one vector,
  int step;            // or (step > 0) apart by so many: where rows are no whole vectors
  int tx, cy;          // threads across the channels of a block, chunks in it
  int width;           // channels of a block
  int channel_blocks;  // blocks across the channels
  int chunk;           // rows of a chunk
  int64_t chunks;
  int kept;            // states kept of a chunk
  bool whole;          // sequences end with chunks: nothing passes from one to the next
  int slots;           // blocks that hold a part of one gate's channels
};

// Where a sequence begins in a run, nothing of the state before it passes through:
// the run is cut, which stands in the place of P.
constexpr uint32_t kCut = 0xffffc0deu;  // as fp32 a NaN that no product here is

// m 2^e, 1 <= |m| < 2 or 0 with e = 0.
struct alignas(8) Wide {
  float m;
  int e;
};

struct Args {
  int64_t rows;
  int sequences, channels, gates, per_gate;  // per_gate = channels / gates
  int64_t period;                            // rows of a sequence when offsets == nullptr
  const int32_t *offsets;                    // sequences + 1 row numbers, or nullptr
  int reverse;
  Plan plan;
  const void *x, *gate, *dh;
  int64_t x_stride, gate_stride, dh_stride;  // elements from row to row
  const float *initial, *dfinal;
  void *h, *dx, *dgate;
  float *final_state, *dinitial;
  float *saved;      // (chunks, kept, channels): the state before each batch of rows
  int *hints;        // (chunks): the sequence of the row where the chain leaves each chunk; null:
                     // no state passes between chunks, or even sequences
  float2 *maps;      // (chunks, channels): P and L
  Wide *products;    // (chunks, channels): P with its exponent, where maps holds 0 or infinity
  float *carry;      // (chunks, channels): the state that enters each chunk; null: none does
  const float *empty_src;  // what leaves an empty sequence: copied to empty_dst, zeros where null
  float *empty_dst;
  float *partial;    // (slots, rows, gates): gate gradients of channel blocks, or nullptr
  uint32_t *status;
};

int type_bytes(int type);
Plan make_plan(int64_t rows, int sequences, bool even, int channels, int gates, int x_type, int gate_type);
int check_shape(int64_t rows, int sequences, int channels, int gates, int x_type, int gate_type, int even);
bool suits(const void *p, int64_t stride, int bytes, int vec);
int launch_carry(const Args &A, bool back, cudaStream_t st);

inline size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }
inline size_t chain_bytes(const Plan &p, int channels) {
  const size_t n = (size_t)p.chunks, c = (size_t)channels;
  return p.whole ? 0 : round16(n * 4) + 2 * round16(n * c * 8) + round16(n * c * 4);
}
inline void place_chain(Args &A, void *scratch) {
  const size_t n = (size_t)A.plan.chunks, c = (size_t)A.channels;
  if (A.plan.whole) return;
  char *b = static_cast<char *>(scratch);
  if (A.offsets != nullptr) A.hints = reinterpret_cast<int *>(b);
  b += round16(n * 4);
  A.maps = reinterpret_cast<float2 *>(b);
  b += round16(n * c * 8);
  A.products = reinterpret_cast<Wide *>(b);
  b += round16(n * c * 8);
  A.carry = reinterpret_cast<float *>(b);
}

// ---- loads and stores of V adjacent elements ---------------------------------------

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

template <typename T, int V>
struct alignas(V * sizeof(T) >= 16 ? 16 : V * sizeof(T)) Pack {
  T e[V];
};

// The place of a thread: its channels and its chunk's logical rows t0..t1-1. ST:
// its channels lie apart; where the block has no second one for it, the first
// stands in, and the thread writes the same values twice.
template <int V, bool ST>
struct Place {
  int tx, cy, c, g;  // c, g: its first channel and that channel's gate
  int to[V];         // ST: from there to its others
  int64_t chunk, t0, t1;
  bool on;
  __device__ __forceinline__ int at(int v) const { return ST ? to[v] : v; }
};

template <typename T, int V, bool ST, typename P>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p, const P &at) {
  if (!ST) return *reinterpret_cast<const Pack<T, V> *>(p);
  Pack<T, V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.e[v] = p[at.at(v)];
  return o;
}

template <typename T, int V, bool ST>
__device__ __forceinline__ void store_pack(T *p, const float (&x)[V], const Place<V, ST> &at) {
  Pack<T, V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.e[v] = from_f32<T>(x[v]);
  if (!ST) {
    *reinterpret_cast<Pack<T, V> *>(p) = o;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) p[at.at(v)] = o.e[v];
  }
}

// The gates of a thread's channels: one each, or one for the whole vector (the
// plan cuts vectors at gate bounds).
template <typename GT, int V, bool SHARED, bool ST>
struct Gates {
  Pack<GT, SHARED ? 1 : V> g;
  __device__ __forceinline__ float operator()(int v) const { return to_f32<GT>(g.e[SHARED ? 0 : v]); }
  __device__ __forceinline__ void load(const GT *p, const Place<V, ST> &at) {
    if (SHARED)
      g.e[0] = p[0];
    else
      g = load_pack<GT, SHARED ? 1 : V, ST>(p, at);
  }
};

// Row `row` of a (n, channels) fp32 tensor (zeros without one).
template <int V, bool ST>
__device__ __forceinline__ void load_state(const float *__restrict__ p, const Args &A, int64_t row,
                                           const Place<V, ST> &at, float (&out)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v)
    out[v] = p != nullptr ? p[row * A.channels + at.c + at.at(v)] : 0.f;
}
template <int V, bool ST>
__device__ __forceinline__ void store_state(float *__restrict__ p, const Args &A, int64_t row,
                                            const Place<V, ST> &at, const float (&in)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) p[row * A.channels + at.c + at.at(v)] = in[v];
}

// The same in buffers of our own, whose rows start at whole vectors.
template <int V, bool ST>
__device__ __forceinline__ void load_kept(const float *__restrict__ p, const Args &A, int64_t row,
                                          const Place<V, ST> &at, float (&out)[V]) {
  const Pack<float, V> q = load_pack<float, V, ST>(p + row * A.channels + at.c, at);
#pragma unroll
  for (int v = 0; v < V; ++v) out[v] = q.e[v];
}
template <int V, bool ST>
__device__ __forceinline__ void store_kept(float *__restrict__ p, const Args &A, int64_t row,
                                           const Place<V, ST> &at, const float (&in)[V]) {
  store_pack<float, V, ST>(p + row * A.channels + at.c, in, at);
}

// ---- where a row belongs ----------------------------------------------------------------

// A sequence and its rows lo..hi-1 (of the tensor; rows <= INT32_MAX). Offsets
// that do not ascend give wrong sequences, but never an index outside
// [0, sequences).
struct Cursor {
  int s, lo, hi;
  // Moves to the sequence of row p. Rows outside every sequence leave it at a
  // neighbour that does not hold them.
  __device__ __forceinline__ void seek(const Args &A, int p) {
    if (A.offsets == nullptr) {
      const int n = (int)A.period;
      s = (int)((uint32_t)p / (uint32_t)n);
      lo = s * n;
      hi = lo + n;
      return;
    }
    // A step at a time, and leaps that double while they succeed and halve when
    // they do not: a million empty sequences between two rows take about 100 reads.
    for (int leap = 1; s + 1 < A.sequences && p >= A.offsets[s + 1];) {
      ++s;
      const int far = min(s + leap, A.sequences - 1);
      const bool over = p >= A.offsets[far];  // all sequences before it are over
      s = over ? far : s;
      leap = over ? leap * 2 : max(leap / 2, 1);
    }
    for (int leap = 1; s > 0 && p < A.offsets[s];) {
      --s;
      const int far = max(s - leap, 0);
      const bool behind = p < A.offsets[far + 1];  // it ends behind the row, and so do those after it
      s = behind ? far : s;
      leap = behind ? leap * 2 : max(leap / 2, 1);
    }
    lo = A.offsets[s];
    hi = A.offsets[s + 1];
  }
  __device__ __forceinline__ bool holds(int p) const { return p >= lo && p < hi; }
  // Rows p..p+n-1 are all inside and neither its first nor its last.
  __device__ __forceinline__ bool plain(int p, int n) const { return p > lo && p < hi && hi - p > n; }
  // Logical rows from row p on to the end of what p is in: its sequence, or the
  // rows outside of every sequence. At least 1. The cursor has sought p.
  __device__ __forceinline__ int rest(const Args &A, int p) const {
    int n = INT32_MAX / 2;
    if (holds(p)) n = A.reverse ? p - lo + 1 : hi - p;
    else if (!A.reverse && p < lo) n = lo - p;
    else if (A.reverse && p >= hi) n = p - hi + 1;
    return n < 1 ? 1 : n;
  }
  __device__ __forceinline__ bool first(const Args &A, int p) const { return p == (A.reverse ? hi - 1 : lo); }
};

// The sequence where a chunk's walk begins, given whether it walks against the
// logical rows: the one that the chain left the neighbouring chunk with, or the
// outermost one.
template <bool BACK>
__device__ __forceinline__ int first_hint(const Args &A, int64_t chunk) {
  const int64_t next = chunk + (BACK ? 1 : -1);
  if (A.hints != nullptr && next >= 0 && next < A.plan.chunks) return A.hints[next];
  return (A.reverse != 0) == BACK ? 0 : A.sequences - 1;
}

// Blocks behind those of the first launch's chunks: a warp for each sequence
// copies what passes an empty one by and checks that the offsets ascend within
// [0, rows].
constexpr int kSequences = kThreads / 32;
inline unsigned extra_blocks(const Args &A) {
  return A.offsets == nullptr && A.rows > 0 ? 0u : (unsigned)((A.sequences + kSequences - 1) / kSequences);
}
__device__ __forceinline__ void look_at_sequences(const Args &A, int64_t block) {
  const int64_t s = block * kSequences + threadIdx.x / 32;
  if (s >= A.sequences) return;
  const int64_t a = A.offsets != nullptr ? A.offsets[s] : 0, b = A.offsets != nullptr ? A.offsets[s + 1] : 0;
  if (a == b && A.empty_dst != nullptr)
    for (int c = (int)lane_id(); c < A.channels; c += 32)
      A.empty_dst[s * A.channels + c] = A.empty_src != nullptr ? A.empty_src[s * A.channels + c] : 0.f;
  if ((a < 0 || a > b || b > A.rows) && lane_id() == 0)
    atomicCAS(A.status, 0u, (uint32_t)GS_ERR_INVALID_ARGUMENT);
}

inline unsigned grid_of(const Plan &p) {
  return (unsigned)(((p.chunks + p.cy - 1) / p.cy) * p.channel_blocks);
}

// The walk after the two launches of the chain, or alone.
template <typename Kernel>
inline int launch_walk(Kernel kernel, const Args &A, cudaStream_t st) {
  const unsigned blocks = grid_of(A.plan);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr = overlapping();
  cfg.attrs = &attr;
  cfg.numAttrs = A.carry != nullptr ? 1 : 0;
  cfg.gridDim = dim3(blocks + (A.carry == nullptr ? extra_blocks(A) : 0));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  const int rc = cuda_status(cudaLaunchKernelEx(&cfg, kernel, A, blocks));
  if (rc) return rc;
  count_launch();
  return GS_OK;
}

template <int V, bool SHARED, bool ST>
__device__ __forceinline__ Place<V, ST> place_of(const Args &A, int64_t group, int cblk) {
  Place<V, ST> p;
  p.tx = threadIdx.x % A.plan.tx;
  p.cy = threadIdx.x / A.plan.tx;
  p.c = cblk * A.plan.width + p.tx * (ST ? 1 : V);
  const int end = (cblk + 1) * A.plan.width < A.channels ? (cblk + 1) * A.plan.width : A.channels;
  p.g = SHARED ? p.c / A.per_gate : p.c;
#pragma unroll
  for (int v = 0; v < V; ++v) p.to[v] = ST && p.c + v * A.plan.step < end ? v * A.plan.step : 0;
  p.chunk = group * A.plan.cy + p.cy;
  p.on = p.cy < A.plan.cy && p.chunk < A.plan.chunks && p.c < end;
  p.t0 = p.chunk * A.plan.chunk;
  p.t1 = p.t0 + A.plan.chunk < A.rows ? p.t0 + A.plan.chunk : A.rows;
  return p;
}

__device__ __forceinline__ int64_t row_at(const Args &A, int64_t t) { return A.reverse ? A.rows - 1 - t : t; }
// Elements from one logical row to the next.
__device__ __forceinline__ int64_t along(const Args &A, int64_t stride) { return A.reverse ? -stride : stride; }

// ---- products of gates with an exponent of their own -------------------------------------

__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int within(int e, int most) { return min(max(e, -most), most); }

// v 2^e; 0 where v lies below the normal range.
__device__ __forceinline__ Wide normal(float v, int e) {
  const uint32_t bits = __float_as_uint(v);
  const int exponent = (int)(bits >> 23 & 255);
  if (exponent == 0) return Wide{0.f, 0};
  return Wide{__uint_as_float((bits & 0x807fffffu) | 0x3f800000u), e + exponent - 127};
}

// ---- the chunks' maps ----------------------------------------------------------------------
//
// What passes from a chunk to the one after it along the chain (BACK: against
// the logical rows, with v = g (dh + v) in place of h = g h + x): the map of the
// rows of the sequence that reaches over the chunk's end, from that sequence's
// first row along the chain where the chunk holds it (the chain is cut there).

// p times the gates of n rows, one by one: where their product leaves the range.
// What is not finite needs no care here: the run's result is not finite then.
template <typename GT>
__device__ __forceinline__ void multiply_rows(Wide &p, const GT *gate, int64_t step, int n) {
#pragma unroll 1
  for (int k = 0; k < n; ++k) {
    const float g = to_f32<GT>(gate[k * step]);
    const bool large = fabsf(g) >= 1.f;
    p = normal(p.m * (large ? g * 0.5f : g * 0x1p100f), p.e + (large ? 1 : -100));
  }
}

// Four blocks an SM (two where a thread holds more loads): with three, or as many
// registers as the compiler likes, too few loads are in flight (16,384 x 1024 fp32:
// forward 60 us, 68 and 73).
template <typename XT, typename GT, int V, bool SHARED, bool ST, bool BACK>
__global__ void __launch_bounds__(kThreads, ST || (V == 4 && !SHARED) ? 2 : 4) maps_kernel(const __grid_constant__ Args A, unsigned blocks) {
  start_next();
  if (blockIdx.x >= blocks) {
    look_at_sequences(A, blockIdx.x - blocks);
    return;
  }
  const int cblk = blockIdx.x % A.plan.channel_blocks;
  const auto p = place_of<V, SHARED, ST>(A, blockIdx.x / A.plan.channel_blocks, cblk);
  if (!p.on) return;
  const int64_t t_end = BACK ? p.t0 : p.t1 - 1;  // the chunk's last row along the chain
  const int row_end = (int)row_at(A, t_end);
  Cursor q;
  q.s = 0;
  if (A.offsets != nullptr) {  // the first sequence that ends behind the row, or the last
    int hi = A.sequences - 1;
    while (q.s < hi) {
      const int mid = q.s + (hi - q.s) / 2;
      if (A.offsets[mid + 1] <= row_end) q.s = mid + 1;
      else hi = mid;
    }
    if (cblk == 0 && p.tx == 0) A.hints[p.chunk] = q.s;
  }
  q.seek(A, row_end);
  // Rows of the tensor run up along the chain, or down.
  const bool up = (A.reverse != 0) == BACK;
  int n = (int)(p.t1 - p.t0);  // rows of the chunk that the map covers
  bool cut = false, needed = true;
  if (!q.holds(row_end) || row_end == (up ? q.hi - 1 : q.lo)) {
    cut = true;   // the sequence ends with the chunk, or the row is outside
    needed = false;
  } else {
    const int first = up ? q.lo : q.hi - 1;  // the sequence's first row along the chain
    const int before = up ? row_end - first : first - row_end;
    if (before < n) n = before + 1, cut = true;
  }
  constexpr int kGates = SHARED ? 1 : V;
  Wide P[kGates];
  float L[V];
  int peak = 0;  // of the exponents
#pragma unroll
  for (int v = 0; v < kGates; ++v) P[v] = Wide{1.f, 0};
#pragma unroll
  for (int v = 0; v < V; ++v) L[v] = 0.f;
  if (needed) {
    if (cut) load_state(BACK ? A.dfinal : A.initial, A, q.s, p, L);
    const int64_t row = up ? row_end - (n - 1) : row_end + (n - 1);
    const int64_t xs = BACK ? A.dh_stride : A.x_stride;
    const XT *from = reinterpret_cast<const XT *>(BACK ? A.dh : A.x) + row * xs + p.c;
    const GT *gate = reinterpret_cast<const GT *>(A.gate) + row * A.gate_stride + p.g;
    const int64_t step = up ? xs : -xs, gstep = up ? A.gate_stride : -A.gate_stride;
    const bool some = !BACK || A.dh != nullptr;
    constexpr int kAhead = ST || V == 1 ? 2 * kBatch : kBatch;
    for (int left = n; left > 0; left -= kAhead) {
      Pack<XT, V> x[kAhead];
      Gates<GT, V, SHARED, ST> g[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k < left) {
          if (some) x[k] = load_pack<XT, V, ST>(from + k * step, p);
          g[k].load(gate + k * gstep, p);
        }
      float product[kGates];
#pragma unroll
      for (int v = 0; v < kGates; ++v) product[v] = P[v].m;
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k < left) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float e = some ? to_f32<XT>(x[k].e[v]) : 0.f;
            L[v] = BACK ? g[k](v) * (e + L[v]) : fmaf(g[k](v), L[v], e);
          }
        }
      // Cut runs need no product. Where threads are bound by their loads alone, a
      // branch around it costs more than it (bf16 with fp32 gates, 8 x 2048 x 1024:
      // forward 57 us with, 48 without; bf16, 49,152 x 333: 55 and 59).
      if (!ST || !cut) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (k < left)
#pragma unroll
            for (int v = 0; v < kGates; ++v) product[v] *= g[k](v);
#pragma unroll
        for (int v = 0; v < kGates; ++v) {
          if (fabsf(product[v]) >= 0x1p-110f && fabsf(product[v]) <= 0x1p110f)
            P[v] = normal(product[v], P[v].e);
          else if (!cut && P[v].m != 0.f) {
            bool zero = false;  // most often a reset
#pragma unroll
            for (int k = 0; k < kAhead; ++k) zero = zero || (k < left && g[k](v) == 0.f);
            if (zero) P[v] = Wide{0.f, 0};
            else multiply_rows(P[v], gate + p.at(v), gstep, left < kAhead ? left : kAhead);
          }
          peak = max(peak, P[v].e);
        }
      }
      from += kAhead * step;
      gate += kAhead * gstep;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Wide w = P[SHARED ? 0 : v];
    const int64_t at = p.chunk * A.channels + p.c + p.at(v);
    const bool held = w.e >= -126 && peak <= 10 && w.m != 0.f;
    const float P32 = held ? w.m * power_of_2(w.e) : peak > 10 ? INFINITY : 0.f;
    A.maps[at] = make_float2(cut ? __uint_as_float(kCut) : P32, L[v]);
    if (!held) A.products[at] = w;
  }
}

}  // namespace scan
}  // namespace gs
