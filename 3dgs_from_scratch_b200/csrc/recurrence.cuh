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
// Every kernel works on tiles of kept rows x channels: a block of 256 threads
// holds SEG segments of R consecutive rows each (TX threads across the
// channels, V channels per thread), reads the tile once into registers,
// reduces each segment to its (P, L), folds the segments through shared
// memory and then walks its rows again from the state before them. Sequence
// bounds need no tiles of their own: at a sequence's first row the chain from
// the row before is cut (P becomes 0) and the initial state enters, so ragged
// sequences cost what their rows cost.
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
  float *saved;      // (tiles, channels): the state before each tile
  uint32_t *ticket;  // hands out the tiles in the chain's order; null: one tile
  uint32_t *flags;   // (tiles, channel blocks): the tile's map is in place
  uint2 *groups;     // (groups, channels): the state after a group of tiles, and whether it is there
  float2 *maps;      // (tiles, channels): each tile's (P, L)
  float *partial;    // (slots, rows, gates): gate gradients of channel blocks, or nullptr
  int slots;
  uint32_t *status;
};

// How a problem is cut. It depends on the sizes and types alone, never on
// pointers, so that the backward finds the states that the forward kept.
struct Plan {
  int vec, tx, seg, tile_rows, channel_blocks, slots;
  int64_t tiles;
};

// Rows of a segment: of single channels, and of vectors of them.
constexpr int kRowsScalar = 8, kRowsVector = 4;

int type_bytes(int type);
Plan make_plan(int64_t rows, int channels, int gates, int x_type, int gate_type);
int check_shape(int64_t rows, int sequences, int channels, int gates, int x_type, int gate_type,
                const int32_t *offsets);
bool suits(const void *p, int64_t stride, int bytes, int vec);
void fill_plan(Args &A, const Plan &p);

// Tiles of a group, whose last one passes the state on to the next group.
constexpr int kGroup = 64;

// The scratch of the tiles' chain: ticket, flags and group states (zeroed
// before every launch), then the maps.
inline size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }
inline int64_t groups_of(const Plan &p) { return (p.tiles + kGroup - 1) / kGroup; }
inline size_t zeroed_bytes(const Plan &p, int channels) {
  return 16 + round16((size_t)p.tiles * p.channel_blocks * 4) + round16((size_t)groups_of(p) * channels * 8);
}
inline size_t chain_bytes(const Plan &p, int channels) {
  return p.tiles == 1 ? 0 : zeroed_bytes(p, channels) + round16((size_t)p.tiles * channels * 8);
}
inline int place_chain(Args &A, const Plan &p, void *scratch, cudaStream_t st) {
  char *b = static_cast<char *>(scratch);
  A.ticket = reinterpret_cast<uint32_t *>(b);
  A.flags = reinterpret_cast<uint32_t *>(b + 16);
  A.groups = reinterpret_cast<uint2 *>(b + 16 + round16((size_t)p.tiles * p.channel_blocks * 4));
  A.maps = reinterpret_cast<float2 *>(b + zeroed_bytes(p, A.channels));
  return zero_async(scratch, zeroed_bytes(p, A.channels), st);
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

// What a tile knows of a logical row: 4 * sequence + 2 * (last row of it) +
// (first row of it), "first" and "last" in logical order; -1 outside every
// sequence. Offsets that do not ascend give wrong sequences, but never an
// index outside [0, sequences).
__device__ __forceinline__ void tile_info(const Args &A, int64_t tile, int *info) {
  __shared__ int bounds[2];
  const int64_t t0 = tile * A.tile_rows;
  const int64_t t1 = t0 + A.tile_rows < A.rows ? t0 + A.tile_rows : A.rows;
  const int64_t p0 = A.reverse ? A.rows - t1 : t0, p1 = p0 + (t1 - t0) - 1;  // rows p0..p1
  if (A.offsets != nullptr) {
    const int warp = threadIdx.x / 32;
    if (warp < 2) {
      const int s = warp_upper_bound(A.offsets + 1, A.sequences, warp ? p1 : p0);
      if (lane_id() == 0) bounds[warp] = s;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < t1 - t0; i += kThreads) {
    const int64_t p = A.reverse ? A.rows - 1 - (t0 + i) : t0 + i;
    int s;
    bool begins, ends;
    if (A.offsets == nullptr) {
      s = (int)(p / A.period);
      const int64_t at = p - (int64_t)s * A.period;
      begins = at == 0;
      ends = at == A.period - 1;
    } else {
      int lo = bounds[0], hi = bounds[1] > bounds[0] ? bounds[1] : bounds[0];
      while (lo < hi) {  // the bounds' own sequences hold the answer
        const int mid = lo + (hi - lo) / 2;
        if ((int64_t)A.offsets[1 + mid] <= p) lo = mid + 1;
        else hi = mid;
      }
      s = lo;
      if (s >= A.sequences || p < (int64_t)A.offsets[s]) {
        info[i] = -1;
        continue;
      }
      begins = p == (int64_t)A.offsets[s];
      ends = p + 1 == (int64_t)A.offsets[s + 1];
    }
    const bool first = A.reverse ? ends : begins, last = A.reverse ? begins : ends;
    info[i] = s * 4 + (last ? 2 : 0) + (first ? 1 : 0);
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
  bool on;            // holds channels of the tensor
  int64_t tile, t0;   // tile and its first logical row
  int rows;           // rows of the tensor in this thread's segment
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
  p.on = p.sg < A.seg && p.c < A.channels;
  const int64_t left = A.rows - p.t0 - (int64_t)p.sg * R;
  p.rows = !p.on || left <= 0 ? 0 : left < R ? (int)left : R;
  return p;
}

// Row number in the tensor of row i of the thread's segment.
template <int R>
__device__ __forceinline__ int64_t row_of(const Args &A, const Place &p, int i) {
  const int64_t t = p.t0 + (int64_t)p.sg * R + i;
  return A.reverse ? A.rows - 1 - t : t;
}

// The gate of a thread's channel v: one for each channel, or one for the
// whole vector (the plan cuts vectors at gate bounds).
template <typename GT, int V, bool SHARED>
struct Gates {
  Pack<GT, SHARED ? 1 : V> g;
  __device__ __forceinline__ float operator()(int v) const { return to_f32<GT>(g.e[SHARED ? 0 : v]); }
  __device__ __forceinline__ void load(const Args &A, int64_t row, int at) {
    g = load_pack<GT, SHARED ? 1 : V>(reinterpret_cast<const GT *>(A.gate) + row * A.gate_stride + at);
  }
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
__device__ __forceinline__ void reduce_segment(const Args &A, const Place &p, const int *info,
                                               const Pack<XT, V> (&x)[R],
                                               const Gates<GT, V, SHARED> (&g)[R], float (&P)[V],
                                               float (&L)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) P[v] = 1.f, L[v] = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i >= p.rows) break;
    const int in = info[p.sg * R + i];
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
__device__ __forceinline__ void reduce_segment_back(const Args &A, const Place &p, const int *info,
                                                    const Pack<XT, V> (&dh)[R],
                                                    const Gates<GT, V, SHARED> (&g)[R],
                                                    float (&P)[V], float (&L)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) P[v] = 1.f, L[v] = 0.f;
#pragma unroll
  for (int i = R - 1; i >= 0; --i) {
    if (i >= p.rows) continue;
    const int in = info[p.sg * R + i];
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
__device__ __forceinline__ bool segment_cut(const Place &p, const int *info, int bit) {
  bool cut = false;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < p.rows) {
      const int in = info[p.sg * R + i];
      cut = cut || in < 0 || (in & bit);
    }
  return cut;
}

__device__ __forceinline__ float pass(bool cut, float P, float L, float h) {
  return cut ? L : fmaf(P, h, L);
}

// A tile in shared memory: its rows' info, its segments' maps by channel, and
// where the chain is cut (in a segment, and anywhere before it).
template <int V, int R>
struct Tile {
  int info[kThreads * R];
  float2 map[kThreads * V];  // [segment][channel of the block]
  uint8_t cut[kThreads], cut_before[kThreads];
};

// Folds the tile's segments: map[segment] becomes the map of everything
// before the segment (BACK: behind it). Thread c of the block gets the whole
// tile's map for its channel c (c < tx * V <= 256). In the order of the
// segments, so every run rounds alike. The caller synchronises before and
// after.
template <int V, int R, bool BACK>
__device__ __forceinline__ bool fold_segments(const Args &A, Tile<V, R> &S, float &P, float &L) {
  const int width = A.tx * V, c = threadIdx.x;
  P = 1.f, L = 0.f;
  bool cut = false;
  if (c < width)
    for (int k = 0; k < A.seg; ++k) {
      const int sg = BACK ? A.seg - 1 - k : k;
      const float2 m = S.map[sg * width + c];
      const bool here = S.cut[sg];
      S.map[sg * width + c] = make_float2(P, L);
      if (c == 0) S.cut_before[sg] = cut;
      L = pass(here, m.x, m.y, L);
      P *= m.x;
      cut = cut || here;
    }
  return cut;
}

// Puts a thread's segment map where fold_segments finds it.
template <int V, int R>
__device__ __forceinline__ void put_segment(const Args &A, const Place &p, Tile<V, R> &S, bool cut,
                                            const float (&P)[V], const float (&L)[V]) {
  if (p.sg >= A.seg) return;
#pragma unroll
  for (int v = 0; v < V; ++v)
    S.map[(p.sg * A.tx + p.tx) * V + v] = make_float2(P[v], L[v]);
  if (p.tx == 0) S.cut[p.sg] = cut;
}

// A segment's state before it, from the state that enters the tile
// (carry[channel of the block]).
template <int V, int R>
__device__ __forceinline__ void enter_segment(const Args &A, const Place &p, const Tile<V, R> &S,
                                              const float *carry, float (&h)[V]) {
  const bool cut = S.cut_before[p.sg];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float2 m = S.map[(p.sg * A.tx + p.tx) * V + v];
    h[v] = pass(cut, m.x, m.y, carry[p.tx * V + v]);
  }
}

// ---- the chain from tile to tile ---------------------------------------------------
//
// Blocks take their tiles by ticket, in the chain's order (position k counts
// along it), so every tile that a block waits for is held by a block that runs
// already. A tile puts its own map in place as soon as it has it. The state
// that enters tile k is then: the state after the group of kGroup tiles before
// k's own group, and the maps of the tiles between, folded in order; of the
// tiles only those count that hold rows of the sequence that reaches into k. A
// group's last tile passes the state on. What is added to what depends on
// positions alone, so every run rounds alike. Waits are bounded; one that gives
// up records GS_ERR_DEVICE_TIMEOUT.

__device__ __forceinline__ uint32_t load_acquire(const uint32_t *p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(uint32_t *p, uint32_t v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// A state and its flag in one 8-byte word, which arrives whole.
__device__ __forceinline__ uint2 load_word(const uint2 *p) {
  uint64_t v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}
__device__ __forceinline__ void store_word(uint2 *p, float state) {
  const uint64_t v = (uint64_t)__float_as_uint(state) | (1ull << 32);
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}

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

// Publishes the tile's map (P, L; thread c for channel c of the block) and
// finds the state that enters it, into carry[c]. All threads call it; it
// synchronises.
template <bool BACK>
__device__ __forceinline__ void join_chain(const Args &A, int64_t k, int cblk, int width, int in,
                                           bool cut, float P, float L, float *carry,
                                           float2 *parts) {
  const int c = threadIdx.x, at = cblk * width + c;
  const bool mine = c < width && at < A.channels;
  if (A.ticket == nullptr) {
    if (c < width) carry[c] = 0.f;
    __syncthreads();
    return;
  }
  if (mine) A.maps[k * A.channels + at] = make_float2(P, L);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) store_release(&A.flags[k * A.channel_blocks + cblk], 1u);
  const int64_t group = k / kGroup, start = chain_start<BACK>(A, k, in);
  const bool from_group = start < group * kGroup;
  const int64_t base = from_group ? group * kGroup : start;
  const int count = (int)(k - base);
  bool late = false;
  if (threadIdx.x < count) {  // count < kGroup <= threads
    uint32_t spins = 0;
    while (load_acquire(&A.flags[(base + threadIdx.x) * A.channel_blocks + cblk]) == 0u)
      if (++spins == kSpinLimit) {
        late = true;
        break;
      }
  }
  __syncthreads();
  // The maps between, folded in up to threads / width runs of tiles.
  const int runs = kThreads / width, run = c / width, cc = c % width;
  if (run < runs) {
    const int j0 = count * run / runs, j1 = count * (run + 1) / runs;
    float p = 1.f, l = 0.f;
    if (cblk * width + cc < A.channels) {
      const float2 *m = A.maps + base * A.channels + cblk * width + cc;
#pragma unroll 8
      for (int j = j0; j < j1; ++j) {
        const float2 f = __ldcg(m + (int64_t)j * A.channels);
        // the chain's first tile holds the cut: only its L counts
        const bool first = !from_group && j == 0;
        l = first ? f.y : fmaf(f.x, l, f.y);
        p = first ? 0.f : p * f.x;
      }
    }
    parts[run * width + cc] = make_float2(p, l);
  }
  __syncthreads();
  if (mine) {
    float h = 0.f;
    if (from_group) {
      const uint2 *word = A.groups + (group - 1) * A.channels + at;
      uint2 v = load_word(word);
      uint32_t spins = 0;
      while (v.y == 0u) {
        if (++spins == kSpinLimit) {
          late = true;
          break;
        }
        v = load_word(word);
      }
      h = __uint_as_float(v.x);
    }
    for (int q = 0; q < runs; ++q) {
      const float2 f = parts[q * width + c];
      const bool first = !from_group && count > 0 && count * q / runs == 0 && count * (q + 1) / runs > 0;
      h = first ? f.y : fmaf(f.x, h, f.y);
    }
    if (k % kGroup == kGroup - 1) store_word(&A.groups[group * A.channels + at], pass(cut, P, L, h));
    carry[c] = h;
  } else if (c < width) {
    carry[c] = 0.f;
  }
  if (late) atomicCAS(A.status, 0u, (uint32_t)GS_ERR_DEVICE_TIMEOUT);
  __syncthreads();
}

}  // namespace scan
}  // namespace gs
