// recurrence_forward.cu -- h_t = g_t h_{t-1} + x_t over packed sequences (see
// recurrence.cuh).
#include "cluster.cuh"
#include "recurrence.cuh"

namespace gs {
namespace scan {

int type_bytes(int type) {
  return type == GS_TYPE_F32 ? 4 : type == GS_TYPE_BF16 || type == GS_TYPE_F16 ? 2 : 0;
}

Plan make_plan(int64_t rows, int sequences, bool even, int channels, int gates, int x_type, int gate_type) {
  Plan p;
  const int xb = type_bytes(x_type), gb = type_bytes(gate_type), per = channels / gates;
  const bool shared = per > 1;
  // 8 bytes of the wider type a row and thread: 16 leave too few threads, and
  // the backward short of registers.
  const int wide = 8 / (shared ? xb : xb > gb ? xb : gb);
  if ((shared ? per : channels) % wide == 0) {
    p.vec = wide;
    p.step = 0;
  } else {
    // In 16 bits two channels a thread, tx apart, so that the threads of a row
    // still read adjacent ones (bf16, 65,536 rows x 333 channels: forward 76 us
    // against 146 with one, with the backward 197 against 264; 524,288 x 35: 64
    // against 83, 158 against 175; few rows even out, 4096 x 35: 13.1 against
    // 13.9, 32 against 28). One a thread in 32 bits (524,288 x 35: 80 and 191
    // against 93 and 212 with two), where channels share gates (333 with one
    // gate: 205 against 213 with the backward) and up to a warp's channels
    // (2,097,152 x 3: 230 against 258).
    p.step = !shared && xb == 2 && gb == 2 && channels > 32;
    p.vec = p.step ? 2 : 1;
  }
  const int most = kThreads * p.vec, one = shared ? per : 1;  // channels of a block, of a gate
  p.channel_blocks = (channels + most - 1) / most;
  p.width = (channels + p.channel_blocks - 1) / p.channel_blocks;
  if (!p.step) p.width = (p.width + p.vec - 1) / p.vec * p.vec;
  if (one <= most) {  // whole gates in a block, where they fit
    p.width = (p.width + one - 1) / one * one;
    if (p.width > most) p.width = most / one * one;
  }
  p.channel_blocks = (channels + p.width - 1) / p.width;
  p.tx = (p.width + p.vec - 1) / p.vec;
  p.step *= p.tx;
  p.cy = kThreads / p.tx;
  const int vectors = (channels + p.vec - 1) / p.vec;
  // Rows of a chunk: about kFill threads on each of 148 SMs.
  const int64_t want = rows * vectors / (148 * kFill);
  const int64_t period = even ? rows / sequences : 0;
  // Sequences stay whole, without the chain's launches, where they are short or
  // enough to give 256 threads an SM: fewer lose more by the threads that are
  // missing (512 rows x 64 channels fp32, forward and backward: 137 us whole and 92
  // cut at 64 threads an SM, 156 and 168 at 128, 217 and 300 at 256, 513 and 694 at
  // 640; 2048 rows 816 and 1125 at 256).
  p.whole = even && period > 0 && (period <= kShort || (int64_t)sequences * vectors >= 148 * 256);
  if (p.whole) {
    const int64_t k = want / period;
    p.chunk = (int)(period * (k < 1 ? 1 : k > 64 ? 64 : k));
  } else {
    int64_t chunk = 32;
    while (chunk < want && chunk < 512) chunk *= 2;
    p.chunk = (int)chunk;
    if (rows <= kShort) p.chunk = kShort;
    p.whole = rows <= p.chunk;
  }
  p.chunks = rows > 0 ? (rows + p.chunk - 1) / p.chunk : 0;
  p.kept = (p.chunk + kBatch - 1) / kBatch;
  p.slots = shared && p.width % per != 0 ? (per + p.width - 2) / p.width + 1 : 1;
  return p;
}

// The state that enters each chunk, from the chunks' maps: 4 channels a block,
// 128 threads a channel with a run of chunks each. The runs' maps are scanned in
// shared memory, then each thread goes through its run once more from the state
// before it. Many chunks are shared out over a cluster of blocks, which read
// each other's maps.
constexpr int kCarryChannels = 4, kRuns = 128, kCarryBlocks = 8;

// A run's map with P in fp32, for products of at most 1, and in the form that
// holds any product.
struct Narrow {
  static constexpr int kAhead = 16;  // chunks on their way at a time; a run of no more is read once
  float P, L;
  __device__ static Narrow nothing() { return {1.f, 0.f}; }
  __device__ static Narrow of(const Args &A, int64_t at) {
    const float2 m = A.maps[at];
    return {m.x, m.y};
  }
  __device__ bool cut() const { return __float_as_uint(P) == kCut; }
  // What leaves the run that a state enters.
  __device__ float through(float state) const { return cut() ? L : fmaf(P, state, L); }
  // Becomes the map of `before` and then this.
  __device__ void follow(const Narrow &before) {
    L = through(before.L);
    P = cut() ? P : before.cut() ? before.P : P * before.P;
  }
  __device__ bool grown() const { return !cut() && !(fabsf(P) <= 1.f); }
};
struct Broad {
  static constexpr int kAhead = 4;
  static constexpr int kCutExponent = INT32_MIN, kFarOut = 1 << 20;  // sums of two exponents stay integers
  Wide P;
  float L;
  __device__ static Broad nothing() { return {{1.f, 0}, 0.f}; }
  __device__ static Broad of(const Args &A, int64_t at) {
    const float2 m = A.maps[at];
    if (__float_as_uint(m.x) == kCut) return {{0.f, kCutExponent}, m.y};
    const float size = fabsf(m.x);
    return {size >= FLT_MIN && size <= FLT_MAX ? normal(m.x, 0) : A.products[at], m.y};
  }
  __device__ bool cut() const { return P.e == kCutExponent; }
  // In three factors of 2^100 at most, which take any state of fp32 to 0 or to
  // infinity, and a zero state to 0.
  __device__ float through(float state) const {
    const int e1 = within(P.e, 100), e2 = within(P.e - e1, 100), e3 = within(P.e - e1 - e2, 100);
    return cut() ? L : fmaf(state * power_of_2(e1) * power_of_2(e2), P.m * power_of_2(e3), L);
  }
  __device__ void follow(const Broad &before) {
    L = through(before.L);
    if (cut()) return;
    if (before.cut()) P = before.P;
    else P = normal(P.m * before.P.m, within(P.e + before.P.e, kFarOut));
  }
  __device__ bool grown() const { return false; }
};

// What a block keeps in shared memory. More than these 9 KB keep the walk, which
// starts before the scan has ended, off the same SM for longer (25 KB: 1,300
// chunks x 200 channels 36 us in place of 34).
template <class M>
struct Scanned {
  static constexpr int kBuffers = sizeof(M) == 8 ? 2 : 1;
  M maps[kBuffers][kRuns][kCarryChannels];
  M others[kCarryBlocks][kCarryChannels];
  int grown;
};

// Returns whether (in the cluster) a chunk's product has grown; nothing is written then.
template <bool BACK, class M>
__device__ __forceinline__ bool carry_chunks(const Args &A, int blocks, Scanned<M> &S) {
  const int lane = threadIdx.x % kCarryChannels, run = threadIdx.x / kCarryChannels;
  const int rank = blocks > 1 ? (int)cluster_rank() : 0;
  const int c = blockIdx.x / blocks * kCarryChannels + lane;
  const bool on = c < A.channels;
  const int64_t n = A.plan.chunks, b0 = n * rank / blocks, b1 = n * (rank + 1) / blocks;
  const int64_t k0 = b0 + (b1 - b0) * run / kRuns, k1 = b0 + (b1 - b0) * (run + 1) / kRuns;
  const int64_t step = BACK ? -1 : 1, first = BACK ? n - 1 - k0 : k0;
  float *__restrict__ to = A.carry + first * A.channels + c;
  const int len = (int)(k1 - k0);
  M m[M::kAhead];
  const auto load = [&](int from) {
#pragma unroll
    for (int k = 0; k < M::kAhead; ++k)
      if (from + k < len) m[k] = M::of(A, (first + (from + k) * step) * A.channels + (on ? c : 0));
  };
  M mine = M::nothing();
  bool grown = false;
  for (int from = 0; from < len; from += M::kAhead) {
    load(from);
#pragma unroll
    for (int k = 0; k < M::kAhead; ++k)
      if (from + k < len) {
        M now = m[k];
        now.follow(mine);
        mine = now;
        grown = grown || m[k].grown();
      }
  }
  // Inclusive scan of the runs' maps, doubling the reach.
  S.maps[0][run][lane] = mine;
  __syncthreads();
  int at = 0;
  for (int reach = 1; reach < kRuns; reach *= 2) {
    if (run >= reach) mine.follow(S.maps[at][run - reach][lane]);
    at = (at + 1) % S.kBuffers;
    if (S.kBuffers == 1) __syncthreads();
    S.maps[at][run][lane] = mine;
    if (reach * 2 < kRuns) __syncthreads();
  }
  grown = __syncthreads_or(grown);
  float h = 0.f;  // the state that enters the block's chunks, then the run's
  if (blocks > 1) {
    if (threadIdx.x == 0) S.grown = grown;
    cluster_sync();
    int theirs = 0;
    if ((int)threadIdx.x < blocks * kCarryChannels) {
      const int q = threadIdx.x / kCarryChannels;
      const uint32_t from = cluster_addr(&S.maps[at][kRuns - 1][lane], q);
      uint32_t w[sizeof(M) / 4];
#pragma unroll
      for (int k = 0; k < (int)(sizeof(M) / 4); ++k) w[k] = cluster_load_u32(from + 4 * k);
      memcpy(&S.others[q][lane], w, sizeof(M));
      theirs = (int)cluster_load_u32(cluster_addr(&S.grown, q));
    }
    cluster_sync();  // no block leaves while another may read its maps
    grown = __syncthreads_or(theirs);
    for (int q = 0; q < rank; ++q) h = S.others[q][lane].through(h);
  }
  if (grown) return true;
  if (!on) return false;
  if (run > 0) h = S.maps[at][run - 1][lane].through(h);
  for (int from = 0; from < len; from += M::kAhead) {
    if (len > M::kAhead) load(from);
#pragma unroll
    for (int k = 0; k < M::kAhead; ++k)
      if (from + k < len) {
        to[(from + k) * step * A.channels] = h;
        h = m[k].through(h);
      }
  }
  return false;
}

// Out of line, so that the registers of the usual form stay its own.
template <bool BACK>
__device__ __noinline__ void carry_grown_chunks(const Args &A, int blocks, Scanned<Broad> &S) {
  carry_chunks<BACK>(A, blocks, S);
}

template <bool BACK>
__global__ void __launch_bounds__(kCarryChannels *kRuns) carry_kernel(const __grid_constant__ Args A, int blocks) {
  __shared__ union {
    Scanned<Narrow> narrow;
    Scanned<Broad> broad;
  } shared;
  start_next();
  wait_for_previous();
  if (carry_chunks<BACK>(A, blocks, shared.narrow)) {
    __syncthreads();  // the narrow form's maps are no longer read
    carry_grown_chunks<BACK>(A, blocks, shared.broad);
  }
}

int launch_carry(const Args &A, bool back, cudaStream_t st) {
  // The whole forward in fp32 with one block, and with a cluster: 941 chunks of 32
  // rows x 64 channels 12.1 and 16.2 us, x 200 19.6 and 26.7; 4096 x 64 33.0 and
  // 27.8, 4096 x 4 25.9 and 20.0. Between, few channels gain by a cluster (2048 x 4
  // 20.5 and 19.8) and more lose (2048 x 64 15.6 and 18.8).
  const int blocks = A.plan.chunks > 12 * kRuns ? kCarryBlocks : 1;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0] = overlapping();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = blocks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = blocks > 1 ? 2 : 1;
  cfg.gridDim = dim3((unsigned)((A.channels + kCarryChannels - 1) / kCarryChannels) * blocks);
  cfg.blockDim = dim3(kCarryChannels * kRuns);
  cfg.stream = st;
  const int rc = cuda_status(back ? cudaLaunchKernelEx(&cfg, carry_kernel<true>, A, blocks)
                                  : cudaLaunchKernelEx(&cfg, carry_kernel<false>, A, blocks));
  if (rc) return rc;
  count_launch();
  return GS_OK;
}

template <typename XT, typename GT, int V, bool SHARED, bool ST>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ Args A, unsigned blocks) {
  if (blockIdx.x >= blocks) {
    look_at_sequences(A, blockIdx.x - blocks);
    return;
  }
  const auto p =
      place_of<V, SHARED, ST>(A, blockIdx.x / A.plan.channel_blocks, blockIdx.x % A.plan.channel_blocks);
  if (!p.on) return;
  int row = (int)row_at(A, p.t0);
  const int64_t xs = along(A, A.x_stride), gs = along(A, A.gate_stride), hs = along(A, A.channels);
  const int one = A.reverse ? -1 : 1;
  const XT *from = reinterpret_cast<const XT *>(A.x) + row * A.x_stride + p.c;
  const GT *gate = reinterpret_cast<const GT *>(A.gate) + row * A.gate_stride + p.g;
  XT *to = reinterpret_cast<XT *>(A.h) + (int64_t)row * A.channels + p.c;
  wait_for_previous();
  Cursor q;
  q.s = first_hint<false>(A, p.chunk);
  q.seek(A, row);
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = 0.f;
  if (A.carry != nullptr) load_kept(A.carry, A, p.chunk, p, h);
  int64_t kept = p.chunk * A.plan.kept;
  // Rows to the next event: the first row of a sequence, or of rows outside.
  bool inside = q.holds(row);
  int event = inside && q.first(A, row) || !inside ? 0 : q.rest(A, row);
  for (int left = (int)(p.t1 - p.t0); left > 0; left -= kBatch) {
    Pack<XT, V> x[kBatch];
    Gates<GT, V, SHARED, ST> g[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (k < left) {
        x[k] = load_pack<XT, V, ST>(from, p);
        g[k].load(gate, p);
        from += xs;
        gate += gs;
      }
    if (A.saved != nullptr) store_kept(A.saved, A, kept++, p, h);
    if (inside && event > kBatch && left >= kBatch) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(g[k](v), h[v], to_f32<XT>(x[k].e[v]));
        store_pack<XT, V, ST>(to, h, p);
        to += hs;
      }
    } else {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (k >= left) break;
        if (k == event) {
          const int at = row + k * one;
          q.seek(A, at);
          inside = q.holds(at);
          event += q.rest(A, at);
          if (inside) load_state(A.initial, A, q.s, p, h);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[v] = fmaf(g[k](v), h[v], to_f32<XT>(x[k].e[v]));
          if (!inside) h[v] = 0.f;
        }
        if (k + 1 == event && inside && A.final_state != nullptr)
          store_state(A.final_state, A, q.s, p, h);
        store_pack<XT, V, ST>(to, h, p);
        to += hs;
      }
    }
    row += kBatch * one;
    event -= kBatch;
  }
}

template <typename XT, typename GT, int V, bool SHARED, bool ST>
static int launch_forward(const Args &A, cudaStream_t st) {
  if (A.carry != nullptr) {
    const unsigned blocks = grid_of(A.plan);
    maps_kernel<XT, GT, V, SHARED, ST, false><<<blocks + extra_blocks(A), kThreads, 0, st>>>(A, blocks);
    count_launch();
    const int rc = launch_carry(A, false, st);
    if (rc) return rc;
  }
  return launch_walk(forward_kernel<XT, GT, V, SHARED, ST>, A, st);
}

template <typename XT, typename GT>
static int pick_forward(const Args &A, cudaStream_t st) {
  constexpr int kPer = 8 / (int)(sizeof(XT) > sizeof(GT) ? sizeof(XT) : sizeof(GT));
  constexpr int kShared = 8 / (int)sizeof(XT);
  constexpr bool kApart = sizeof(XT) == 2 && sizeof(GT) == 2;
  const bool shared = A.per_gate > 1;
  if (A.plan.step) return launch_forward<XT, GT, kApart ? 2 : 1, false, kApart>(A, st);
  if (A.plan.vec == 1)
    return shared ? launch_forward<XT, GT, 1, true, false>(A, st) : launch_forward<XT, GT, 1, false, false>(A, st);
  return shared ? launch_forward<XT, GT, kShared, true, false>(A, st)
                : launch_forward<XT, GT, kPer, false, false>(A, st);
}

// What both directions check of their sizes and types.
int check_shape(int64_t rows, int sequences, int channels, int gates, int x_type, int gate_type, int even) {
  if (rows < 0 || rows > INT32_MAX || sequences < 1 || sequences > (1 << 28) || channels < 1 ||
      channels > (1 << 30) || gates < 1 || channels % gates != 0 || !type_bytes(x_type) ||
      (gate_type != x_type && gate_type != GS_TYPE_F32))
    return GS_ERR_INVALID_ARGUMENT;
  if (even && rows % sequences != 0) return GS_ERR_INVALID_ARGUMENT;
  const Plan p = make_plan(rows, sequences, even, channels, gates, x_type, gate_type);
  if ((p.chunks / p.cy + 1) * p.channel_blocks > INT32_MAX / 2) return GS_ERR_CAPACITY;
  return GS_OK;
}

// Whether a row pointer and stride suit the plan's vectors.
bool suits(const void *p, int64_t stride, int bytes, int vec) {
  return ((uintptr_t)p % (bytes * vec)) == 0 && stride % vec == 0;
}

}  // namespace scan
}  // namespace gs

using namespace gs;
using namespace gs::scan;

extern "C" size_t gs_gated_scan_saved_bytes(int64_t rows, int sequences, int even, int channels, int gates,
                                            int x_type, int gate_type) {
  if (check_shape(rows, sequences, channels, gates, x_type, gate_type, even)) return 0;
  const Plan p = make_plan(rows, sequences, even, channels, gates, x_type, gate_type);
  return (size_t)p.chunks * p.kept * channels * 4;
}

extern "C" size_t gs_gated_scan_scratch_bytes(int64_t rows, int sequences, int even, int channels, int gates,
                                              int x_type, int gate_type, int backward) {
  if (check_shape(rows, sequences, channels, gates, x_type, gate_type, even)) return 0;
  const Plan p = make_plan(rows, sequences, even, channels, gates, x_type, gate_type);
  size_t bytes = chain_bytes(p, channels);
  if (backward && p.slots > 1) bytes += (size_t)p.slots * rows * gates * 4;
  return bytes;
}

extern "C" int gs_gated_scan_forward(int64_t rows, int sequences, int channels, int gates, int x_type,
                                     int gate_type, const void *x, int64_t x_row_stride,
                                     const void *gate, int64_t gate_row_stride,
                                     const float *initial, const int32_t *offsets, int reverse,
                                     void *h, float *final_state, float *saved, void *scratch,
                                     size_t scratch_bytes, void *stream) {
  const int even = offsets == nullptr;
  int rc = check_shape(rows, sequences, channels, gates, x_type, gate_type, even);
  if (rc) return rc;
  if (rows > 0 && (x == nullptr || gate == nullptr || h == nullptr)) return GS_ERR_INVALID_ARGUMENT;
  Args A{};
  A.plan = make_plan(rows, sequences, even, channels, gates, x_type, gate_type);
  const int xb = type_bytes(x_type), gb = type_bytes(gate_type), vec = A.plan.step ? 1 : A.plan.vec;
  const bool shared = channels != gates;
  if (!suits(x, x_row_stride, xb, vec) || !suits(h, channels, xb, vec) ||
      !suits(gate, gate_row_stride, gb, shared ? 1 : vec) ||
      (((uintptr_t)initial | (uintptr_t)final_state | (uintptr_t)offsets) & 3) ||
      ((uintptr_t)saved & 15))
    return GS_ERR_INVALID_ARGUMENT;
  A.rows = rows;
  A.sequences = sequences;
  A.channels = channels;
  A.gates = gates;
  A.per_gate = channels / gates;
  A.period = even ? rows / sequences : 0;
  A.offsets = offsets;
  A.reverse = reverse != 0;
  A.x = x;
  A.x_stride = x_row_stride;
  A.gate = gate;
  A.gate_stride = gate_row_stride;
  A.initial = initial;
  A.h = h;
  A.final_state = final_state;
  A.saved = saved;
  const size_t need = gs_gated_scan_scratch_bytes(rows, sequences, even, channels, gates, x_type, gate_type, 0);
  if (need > 0) {
    if (scratch == nullptr || ((uintptr_t)scratch & 15)) return GS_ERR_INVALID_ARGUMENT;
    if (scratch_bytes < need) return GS_ERR_CAPACITY;
    place_chain(A, scratch);
  }
  A.status = device_status_word();
  if (A.status == nullptr) return GS_ERR_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  A.empty_src = initial;
  A.empty_dst = final_state;
  const bool same = x_type == gate_type;
  if (x_type == GS_TYPE_F32) return pick_forward<float, float>(A, st);
  if (x_type == GS_TYPE_BF16)
    return same ? pick_forward<__nv_bfloat16, __nv_bfloat16>(A, st) : pick_forward<__nv_bfloat16, float>(A, st);
  return same ? pick_forward<__half, __half>(A, st) : pick_forward<__half, float>(A, st);
}
