// recurrence.cuh -- the gated linear recurrence's tiles, shared by its
// forward and backward kernels (recurrence_forward.cu, recurrence_backward.cu).
//
// The operator: over every sequence of a packed (rows, C) tensor,
//   h_t = g_t h_{t-1} + x_t,  h_{-1} = initial,
// each gate shared by D = C / G consecutive channels. It is linear, so a run
// of rows acts on the state before it as h -> P h + L (P the product of its
// gates, L its result from a zero state), and runs compose:
//   (P2, L2) after (P1, L1) = (P1 P2, P2 L1 + L2).
//
// Every kernel works on tiles of rows x channels: a block of 256 threads holds
// SEG segments of R consecutive rows each (TX threads across the channels, V
// channels per thread), reads the tile once into registers, reduces each
// segment to its (P, L), folds the segments through shared memory and then
// walks its rows again from the state before them. Sequence bounds need no
// tiles of their own: at a sequence's first row the chain from the row before
// is cut and the initial state enters, so ragged sequences cost what their rows
// cost.
//
// Memory is what bounds both directions (a handful of operations an element):
// forward x and the gates in, h out; backward x, the gates and dh in, dx and the
// gates' gradient out. What kept the first kernels from it were instructions:
// rows are therefore walked by pointer, and a segment without sequence bounds
// takes a path that looks at none.
//
// "Logical" rows run in the direction of the recurrence: with `reverse` the
// logical row t is the row rows - 1 - t of the tensor, and everything below
// is the same.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gs_common.cuh"

namespace gs {
namespace scan {

constexpr int kThreads = 256;

struct Args {
  int64_t rows;
  int sequences, channels, gates, per_gate;  // per_gate = channels / gates
  int64_t period;                            // rows of a sequence when offsets == nullptr
  const int32_t *offsets;                    // sequences + 1 row numbers, or nullptr
  int reverse;
  int tx, seg, tile_rows, channel_blocks;    // the plan below
  int64_t tiles;
  const void *x, *gate, *dh;
  int64_t x_stride, gate_stride, dh_stride;  // elements from row to row
  const float *initial, *dfinal;
  void *h, *dx, *dgate;
  float *final_state, *dinitial;
  float *saved;      // (backward's tiles, channels): the state before each of them
  int saved_rows;    // rows of the backward's tiles: tile_rows, or half of the forward's
  uint32_t *ticket;  // hands out the tiles in the chain's order; null: one tile
  uint2 *groups;     // (groups, channels): the state after a group of tiles, and whether it is there
  ulonglong2 *maps;  // (tiles, channels): each tile's P and L, each with whether it is there
  float *partial;    // (slots, rows, gates): gate gradients of channel blocks, or nullptr
  int slots;
  uint32_t *status;
};

// How a problem is cut. It depends on the sizes and types alone, never on
// pointers, so that the backward finds the states that the forward kept.
struct Plan {
  int vec, tx, seg, tile_rows, back_rows, channel_blocks, slots;
  int64_t tiles, back_tiles;
};

// Rows of a segment: of single channels and of vectors of them, forward and
// backward (which holds three tensors and the states in registers).
constexpr int segment_rows(int vec, bool back) { return vec == 1 ? 8 : back || vec == 8 ? 2 : 4; }
// Blocks on an SM, which their registers are held to.
constexpr int kResident = 3;

int type_bytes(int type);
Plan make_plan(int64_t rows, int channels, int gates, int x_type, int gate_type);
int check_shape(int64_t rows, int sequences, int channels, int gates, int x_type, int gate_type,
                const int32_t *offsets);
bool suits(const void *p, int64_t stride, int bytes, int vec);
void fill_plan(Args &A, const Plan &p, bool back);

// Tiles of a group, whose last one passes the state on to the next group.
constexpr int kGroup = 64;

// The scratch of the tiles' chain, zeroed before every launch: ticket, group
// states, maps.
inline size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }
inline size_t groups_bytes(int64_t tiles, int channels) {
  return round16((size_t)((tiles + kGroup - 1) / kGroup) * channels * 8);
}
inline size_t chain_bytes(int64_t tiles, int channels) {
  return tiles == 1 ? 0 : 16 + groups_bytes(tiles, channels) + (size_t)tiles * channels * 16;
}
inline int place_chain(Args &A, void *scratch, cudaStream_t st) {
  if (A.tiles == 1) return GS_OK;
  char *b = static_cast<char *>(scratch);
  A.ticket = reinterpret_cast<uint32_t *>(b);
  A.groups = reinterpret_cast<uint2 *>(b + 16);
  A.maps = reinterpret_cast<ulonglong2 *>(b + 16 + groups_bytes(A.tiles, A.channels));
  return zero_async(scratch, chain_bytes(A.tiles, A.channels), st);
}

// ---- loads and stores of V consecutive elements ---------------------------------

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

// V elements as they lie in memory: aligned to what one load can move.
template <typename T, int V>
struct alignas(V * sizeof(T) >= 16 ? 16 : V * sizeof(T)) Pack {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
  return *reinterpret_cast<const Pack<T, V> *>(p);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const float (&v)[V]) {
  Pack<T, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) o.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<Pack<T, V> *>(p) = o;
}

// ---- where the rows of a tile belong ----------------------------------------------

// First index in [0, n) of the ascending a with a[i] > v, n if there is none;
// every lane of the warp takes part, 32 probes a round.
__device__ __forceinline__ int warp_upper_bound(const int32_t *__restrict__ a, int n, int64_t v) {
  const int lane = (int)lane_id();
  int lo = 0;
  while (n > 0) {
    const int step = (n + 31) / 32;
    const int64_t at = (int64_t)(lane + 1) * step - 1;
    const bool below = at < n && (int64_t)a[lo + at] <= v;
    const int whole = __popc(__ballot_sync(0xffffffffu, below));
    const int skip = whole * step < n ? whole * step : n;
    lo += skip;
    const int rest = n - skip;
    n = rest < step - 1 ? rest : step - 1;
  }
  return lo;
}

// What is known of a logical row: 4 * sequence + 2 * (last row of it) + (first
// row of it), "first" and "last" in logical order; kOutside outside every
// sequence. Offsets that do not ascend give wrong sequences, but never an
// index outside [0, sequences).
constexpr int kOutside = -1;

__device__ __forceinline__ int row_info(const Args &A, int s, bool begins, bool ends) {
  return s * 4 + ((A.reverse ? begins : ends) ? 2 : 0) + ((A.reverse ? ends : begins) ? 1 : 0);
}

// The rows of a tile, where sequences are given by offsets. All threads call
// it; it synchronises.
__device__ __forceinline__ void tile_info(const Args &A, int64_t tile, int *info) {
  __shared__ int bounds[2];
  const int64_t t0 = tile * A.tile_rows;
  const int64_t t1 = t0 + A.tile_rows < A.rows ? t0 + A.tile_rows : A.rows;
  const int64_t p0 = A.reverse ? A.rows - t1 : t0, p1 = p0 + (t1 - t0) - 1;  // rows p0..p1
  const int warp = threadIdx.x / 32;
  if (warp < 2) {
    const int s = warp_upper_bound(A.offsets + 1, A.sequences, warp ? p1 : p0);
    if (lane_id() == 0) bounds[warp] = s;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < t1 - t0; i += kThreads) {
    const int64_t p = A.reverse ? A.rows - 1 - (t0 + i) : t0 + i;
    int lo = bounds[0], hi = bounds[1] > bounds[0] ? bounds[1] : bounds[0];
    while (lo < hi) {  // the bounds' own sequences hold the answer
      const int mid = lo + (hi - lo) / 2;
      if ((int64_t)A.offsets[1 + mid] <= p) lo = mid + 1;
      else hi = mid;
    }
    info[i] = lo >= A.sequences || p < (int64_t)A.offsets[lo]
                  ? kOutside
                  : row_info(A, lo, p == (int64_t)A.offsets[lo], p + 1 == (int64_t)A.offsets[lo + 1]);
  }
  __syncthreads();
}

// The sequences without rows, shared out over the tiles: what leaves them is
// what enters them (src -> dst, zero where src is null), for this block's
// channels. The same walk checks that the offsets ascend within [0, rows].
__device__ __forceinline__ void empty_sequences(const Args &A, int64_t tile, int c0, int c1,
                                                const float *__restrict__ src,
                                                float *__restrict__ dst) {
  if (A.offsets == nullptr) return;
  bool good = true;
  for (int64_t s = tile * kThreads + threadIdx.x; s < A.sequences; s += A.tiles * kThreads) {
    const int32_t a = A.offsets[s], b = A.offsets[s + 1];
    good = good && a >= 0 && a <= b && (int64_t)b <= A.rows;
    if (a == b && dst != nullptr)
      for (int c = c0; c < c1; ++c)
        dst[s * A.channels + c] = src != nullptr ? src[s * A.channels + c] : 0.f;
  }
  if (!good) atomicCAS(A.status, 0u, (uint32_t)GS_ERR_INVALID_ARGUMENT);
}

// The place of a thread in its tile.
struct Place {
  int tx, sg, c, g;   // channel vector and segment in the tile, first channel and its gate
  int64_t tile, t0;   // tile and its first logical row
  int64_t row;        // the segment's first row in the tensor
  int rows;           // rows of the tensor in this thread's segment (0: nothing to do)
  bool plain;         // whole, and without a sequence's first or last row
};

template <int V, int R, bool SHARED>
__device__ __forceinline__ Place place_of(const Args &A, int64_t tile, int cblk) {
  Place p;
  p.tile = tile;
  p.tx = threadIdx.x % A.tx;
  p.sg = threadIdx.x / A.tx;
  p.c = (cblk * A.tx + p.tx) * V;
  p.g = SHARED ? p.c / A.per_gate : p.c;
  p.t0 = tile * A.tile_rows;
  const int64_t t = p.t0 + p.sg * R, left = A.rows - t;
  p.row = A.reverse ? A.rows - 1 - t : t;
  p.rows = p.sg >= A.seg || p.c >= A.channels || left <= 0 ? 0 : left < R ? (int)left : R;
  p.plain = false;
  return p;
}

// Elements from one logical row to the next.
__device__ __forceinline__ int64_t along(const Args &A, int64_t stride) {
  return A.reverse ? -stride : stride;
}

// Logical row t of even sequences.
__device__ __forceinline__ int even_info(const Args &A, int64_t t) {
  const uint32_t p = (uint32_t)(A.reverse ? A.rows - 1 - t : t), n = (uint32_t)A.period;
  const uint32_t s = p / n, at = p - s * n;
  return row_info(A, (int)s, at == 0, at == n - 1);
}

// What is known of the thread's rows, and whether the segment is plain.
template <int R>
__device__ __forceinline__ void segment_info(const Args &A, Place &p, const int *info, int (&in)[R]) {
  if (p.rows == 0) return;
  if (A.offsets != nullptr) {
    int any = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      in[i] = info[p.sg * R + i];
      any |= in[i];
    }
    p.plain = p.rows == R && (any & (int)0x80000003) == 0;
  } else {
    const uint32_t n = (uint32_t)A.period, q = (uint32_t)p.row;
    uint32_t s = q / n, at = q - s * n;
    p.plain = p.rows == R && (A.reverse ? at + 1 < n && at >= R : at > 0 && at + R < n);
    if (p.plain) return;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      in[i] = row_info(A, (int)s, at == 0, at == n - 1);
      if (A.reverse) {
        if (at == 0) at = n - 1, --s;
        else --at;
      } else if (++at == n) {
        at = 0, ++s;
      }
    }
  }
}

// The gate of a thread's channel v: one for each channel, or one for the
// whole vector (the plan cuts vectors at gate bounds).
template <typename GT, int V, bool SHARED>
struct Gates {
  Pack<GT, SHARED ? 1 : V> g;
  __device__ __forceinline__ float operator()(int v) const { return to_f32<GT>(g.e[SHARED ? 0 : v]); }
  __device__ __forceinline__ void load(const GT *p) { g = load_pack<GT, SHARED ? 1 : V>(p); }
};

// The state that enters a sequence, channels c.. of sequence s (zero without one).
template <int V>
__device__ __forceinline__ void load_state(const float *__restrict__ p, const Args &A, int s, int c,
                                           float (&out)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) out[v] = p != nullptr ? p[(int64_t)s * A.channels + c + v] : 0.f;
}

template <int V>
__device__ __forceinline__ void store_state(float *__restrict__ p, const Args &A, int s, int c,
                                            const float (&in)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) p[(int64_t)s * A.channels + c + v] = in[v];
}

// A segment's rows as one map h -> P h + L in the direction of the recurrence.
// A row outside every sequence clears the state, the rows behind the tensor's
// end (p.rows) leave it alone.
template <typename XT, typename GT, int V, int R, bool SHARED>
__device__ __forceinline__ void reduce_segment(const Args &A, const Place &p, const int (&ins)[R],
                                               const Pack<XT, V> (&x)[R],
                                               const Gates<GT, V, SHARED> (&g)[R], float (&P)[V],
                                               float (&L)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) P[v] = 1.f, L[v] = 0.f;
  if (p.plain) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        L[v] = fmaf(g[i](v), L[v], to_f32<XT>(x[i].e[v]));
        P[v] *= g[i](v);
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i >= p.rows) break;
    const int in = ins[i];
    if (in < 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 0.f, L[v] = 0.f;
      continue;
    }
    if (in & 1) {
      load_state<V>(A.initial, A, in >> 2, p.c, L);
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      L[v] = fmaf(g[i](v), L[v], to_f32<XT>(x[i].e[v]));
      P[v] *= g[i](v);
    }
  }
}

// The same against the direction, for the gradient that a row hands to the
// row before it, v = g (dh + v_after): a segment's rows as v -> P v + L. At a
// sequence's last row the final state's gradient enters.
template <typename XT, typename GT, int V, int R, bool SHARED>
__device__ __forceinline__ void reduce_segment_back(const Args &A, const Place &p, const int (&ins)[R],
                                                    const Pack<XT, V> (&dh)[R],
                                                    const Gates<GT, V, SHARED> (&g)[R],
                                                    float (&P)[V], float (&L)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) P[v] = 1.f, L[v] = 0.f;
  if (p.plain) {
#pragma unroll
    for (int i = R - 1; i >= 0; --i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        L[v] = g[i](v) * (to_f32<XT>(dh[i].e[v]) + L[v]);
        P[v] *= g[i](v);
      }
    return;
  }
#pragma unroll
  for (int i = R - 1; i >= 0; --i) {
    if (i >= p.rows) continue;
    const int in = ins[i];
    if (in < 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 0.f, L[v] = 0.f;
      continue;
    }
    if (in & 2) {
      load_state<V>(A.dfinal, A, in >> 2, p.c, L);
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      L[v] = g[i](v) * (to_f32<XT>(dh[i].e[v]) + L[v]);
      P[v] *= g[i](v);
    }
  }
}

// Whether the chain is cut somewhere in the thread's segment: at a sequence's
// first row (its last one, against the direction) or outside every sequence.
// A cut is kept apart from P = 0, so that an infinite or NaN state neither
// leaks into the next sequence nor vanishes at a gate that happens to be 0.
template <int R>
__device__ __forceinline__ bool segment_cut(const Place &p, const int (&in)[R], int bit) {
  bool cut = false;
  if (p.plain) return false;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < p.rows) cut = cut || in[i] < 0 || (in[i] & bit);
  return cut;
}

__device__ __forceinline__ float pass(bool cut, float P, float L, float h) {
  return cut ? L : fmaf(P, h, L);
}

// A tile in shared memory: its segments' maps by channel and where the chain
// is cut. Segments are folded in runs, run q of them by thread q * width + c for
// channel c of the block's width = tx * V (256 / width runs): map[segment] then
// is the map of what lies before the segment in its run, `runs` that of whole
// runs. In the order of segments and runs, so every run of the program rounds
// alike.
template <int V>
struct Tile {
  float2 map[kThreads * V];  // [segment][channel of the block]
  float2 runs[kThreads];     // [run][channel]
  float2 chain[kThreads];    // [run of tiles][channel]
  float carry[kThreads];     // [channel]: the state that enters the tile
  uint8_t cut[kThreads], cut_before[kThreads], cut_run[kThreads];
};

// Puts a thread's segment map in place.
template <int V>
__device__ __forceinline__ void put_segment(const Args &A, const Place &p, Tile<V> &S, bool cut,
                                            const float (&P)[V], const float (&L)[V]) {
  if (p.sg >= A.seg) return;
#pragma unroll
  for (int v = 0; v < V; ++v)
    S.map[(p.sg * A.tx + p.tx) * V + v] = make_float2(P[v], L[v]);
  if (p.tx == 0) S.cut[p.sg] = cut;
}

// Segment k of the fold (BACK: from the last segment on).
template <bool BACK>
__device__ __forceinline__ int fold_at(const Args &A, int k) { return BACK ? A.seg - 1 - k : k; }

template <int V, bool BACK>
__device__ __forceinline__ void fold_runs(const Args &A, Tile<V> &S) {
  const int width = A.tx * V, runs = kThreads / width, run = threadIdx.x / width, c = threadIdx.x % width;
  if (run >= runs) return;
  float P = 1.f, L = 0.f;
  bool cut = false;
  for (int k = A.seg * run / runs; k < A.seg * (run + 1) / runs; ++k) {
    const int sg = fold_at<BACK>(A, k);
    const float2 m = S.map[sg * width + c];
    const bool here = S.cut[sg];
    S.map[sg * width + c] = make_float2(P, L);
    if (c == 0) S.cut_before[sg] = cut;
    L = pass(here, m.x, m.y, L);
    P *= m.x;
    cut = cut || here;
  }
  S.runs[threadIdx.x] = make_float2(P, L);
  if (c == 0) S.cut_run[run] = cut;
}

// The whole tile's map of channel c of the block, and whether it is cut.
template <int V>
__device__ __forceinline__ bool whole_tile(const Args &A, const Tile<V> &S, int c, float &P, float &L) {
  const int width = A.tx * V, runs = kThreads / width;
  bool cut = false;
  P = 1.f, L = 0.f;
  for (int q = 0; q < runs; ++q) {
    const float2 m = S.runs[q * width + c];
    L = pass(S.cut_run[q], m.x, m.y, L);
    P *= m.x;
    cut = cut || S.cut_run[q];
  }
  return cut;
}

// A segment's state before it, from the state that enters the tile.
template <int V, bool BACK>
__device__ __forceinline__ void enter_segment(const Args &A, const Place &p, const Tile<V> &S,
                                              float (&h)[V]) {
  const int width = A.tx * V, runs = kThreads / width, at = p.tx * V;
  const int k = fold_at<BACK>(A, p.sg);
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = S.carry[at + v];
  for (int q = 0; q < runs && k >= A.seg * (q + 1) / runs; ++q) {
    const bool cut = S.cut_run[q];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = S.runs[q * width + at + v];
      h[v] = pass(cut, m.x, m.y, h[v]);
    }
  }
  const bool cut = S.cut_before[p.sg];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float2 m = S.map[p.sg * width + at + v];
    h[v] = pass(cut, m.x, m.y, h[v]);
  }
}

// ---- the chain from tile to tile ---------------------------------------------------
//
// Blocks take their tiles by ticket, in the chain's order (position k counts
// along it), so every tile that a block waits for is held by a block that runs
// already. A tile puts its own map in place as soon as it has it. The state that enters tile k
// is then: the state after the group of kGroup tiles before k's own group, and
// the maps of the tiles between, folded in order; of the tiles only those count
// that hold rows of the sequence that reaches into k. A group's last tile passes
// the state on. What is added to what depends on positions alone, so every run
// rounds alike. A number and whether it is there travel in one 8-byte word, so
// nothing has to be ordered. Waits are bounded; one that gives up records
// GS_ERR_DEVICE_TIMEOUT.

__device__ __forceinline__ uint64_t word_of(float v) { return (uint64_t)__float_as_uint(v) | (1ull << 32); }
__device__ __forceinline__ float value_of(uint64_t w) { return __uint_as_float((uint32_t)w); }
__device__ __forceinline__ uint64_t load_word(const void *p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_word(void *p, float v) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(word_of(v)) : "memory");
}
__device__ __forceinline__ ulonglong2 load_map(const ulonglong2 *p) {
  ulonglong2 v;
  asm volatile("ld.relaxed.gpu.global.v2.u64 {%0, %1}, [%2];" : "=l"(v.x), "=l"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_map(ulonglong2 *p, float P, float L) {
  asm volatile("st.relaxed.gpu.global.v2.u64 [%0], {%1, %2};" ::"l"(p), "l"(word_of(P)), "l"(word_of(L))
               : "memory");
}
__device__ __forceinline__ bool there(const ulonglong2 &w) { return ((w.x & w.y) >> 32) != 0; }

// The tile that this block takes: (position in the chain, channel block).
__device__ __forceinline__ void take_tile(const Args &A, int64_t &position, int &cblk) {
  __shared__ uint32_t mine;
  uint32_t t = blockIdx.x;
  if (A.ticket != nullptr) {
    if (threadIdx.x == 0) mine = atomicAdd(A.ticket, 1u);
    __syncthreads();
    t = mine;
  }
  position = t / A.channel_blocks;
  cblk = t % A.channel_blocks;
}

// First position of the chain of `in`, the info of the row at which the chain
// enters position k (BACK: its last row): that of its sequence's first row, k
// where nothing enters.
template <bool BACK>
__device__ __forceinline__ int64_t chain_start(const Args &A, int64_t k, int in) {
  if (in < 0 || (in & (BACK ? 2 : 1))) return k;
  const int s = in >> 2;
  const int64_t a = A.offsets != nullptr ? A.offsets[s] : s * A.period;      // rows a..b-1
  const int64_t b = A.offsets != nullptr ? A.offsets[s + 1] : (s + 1) * A.period;
  const int64_t t = (A.reverse != 0) != BACK ? A.rows - b : a;                // along the chain
  // Against the direction tiles are counted from the end of whole tiles.
  const int64_t shift = BACK ? A.tiles * A.tile_rows - A.rows : 0;
  const int64_t at = (t + shift) / A.tile_rows;
  return at < 0 ? 0 : at < k ? at : k;
}

// Puts the tile's map in place (position k; its runs are folded) and finds the
// state that enters it, into S.carry. in: see chain_start. All threads call it;
// it synchronises.
template <int V, bool BACK>
__device__ __forceinline__ void join_chain(const Args &A, Tile<V> &S, int64_t k, int cblk, int in) {
  const int width = A.tx * V, c = threadIdx.x, at = cblk * width + c;
  const bool mine = c < width && at < A.channels;
  if (A.ticket == nullptr) {
    if (c < width) S.carry[c] = 0.f;
    __syncthreads();
    return;
  }
  float P, L;
  bool cut = false;
  if (mine) {
    cut = whole_tile<V>(A, S, c, P, L);
    store_map(A.maps + k * A.channels + at, P, L);
  }
  const int64_t group = k / kGroup, start = chain_start<BACK>(A, k, in);
  const bool from_group = start < group * kGroup;
  const int64_t base = from_group ? group * kGroup : start;
  const int count = (int)(k - base);  // < kGroup
  uint32_t spins = 0;
  // The maps between, folded in runs of tiles.
  const int runs = kThreads / width, run = c / width, cc = c % width;
  if (run < runs && count > 0) {
    const int j0 = count * run / runs, j1 = count * (run + 1) / runs;
    float p = 1.f, l = 0.f;
    if (cblk * width + cc < A.channels) {
      const ulonglong2 *m = A.maps + base * A.channels + cblk * width + cc;
      for (int j = j0; j < j1; j += 4) {
        ulonglong2 w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (j + q < j1) w[q] = load_map(m + (int64_t)(j + q) * A.channels);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (j + q < j1) {
            while (!there(w[q]) && spins < kSpinLimit) {
              w[q] = load_map(m + (int64_t)(j + q) * A.channels);
              ++spins;
            }
            // the chain's first tile holds the cut: only its L counts
            const bool first = !from_group && j + q == 0;
            const float fp = value_of(w[q].x), fl = value_of(w[q].y);
            l = first ? fl : fmaf(fp, l, fl);
            p = first ? 0.f : p * fp;
          }
      }
    }
    S.chain[run * width + cc] = make_float2(p, l);
  }
  __syncthreads();
  if (mine) {
    float h = 0.f;
    if (from_group) {
      const uint2 *word = A.groups + (group - 1) * A.channels + at;
      uint64_t v = load_word(word);
      while (!(v >> 32) && spins < kSpinLimit) {
        v = load_word(word);
        ++spins;
      }
      h = value_of(v);
    }
    if (count > 0)
      for (int q = 0; q < runs; ++q) {
        const float2 f = S.chain[q * width + c];
        const bool first = !from_group && count * q / runs == 0 && count * (q + 1) / runs > 0;
        h = first ? f.y : fmaf(f.x, h, f.y);
      }
    if (k % kGroup == kGroup - 1) store_word(&A.groups[group * A.channels + at], pass(cut, P, L, h));
    S.carry[c] = h;
  } else if (c < width) {
    S.carry[c] = 0.f;
  }
  if (spins >= kSpinLimit) atomicCAS(A.status, 0u, (uint32_t)GS_ERR_DEVICE_TIMEOUT);
  __syncthreads();
}

}  // namespace scan
}  // namespace gs
