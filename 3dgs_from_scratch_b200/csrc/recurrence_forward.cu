// recurrence_forward.cu -- h_t = g_t h_{t-1} + x_t over packed sequences (see
// recurrence.cuh for the tiles).
#include "recurrence.cuh"

namespace gs {
namespace scan {

int type_bytes(int type) {
  return type == GS_TYPE_F32 ? 4 : type == GS_TYPE_BF16 || type == GS_TYPE_F16 ? 2 : 0;
}

Plan make_plan(int64_t rows, int channels, int gates, int x_type, int gate_type) {
  Plan p;
  const int xb = type_bytes(x_type), gb = type_bytes(gate_type), per = channels / gates;
  const bool shared = per > 1;
  const int wide = 16 / (shared ? xb : xb > gb ? xb : gb);
  p.vec = (shared ? per : channels) % wide == 0 ? wide : 1;
  const int vectors = channels / p.vec, most = p.vec == 1 ? 64 : 8;
  int tx = vectors < most ? vectors : most;
  if (shared && per / p.vec <= most) {  // whole gates in a block, where they fit
    const int one = per / p.vec;
    tx = most / one * one;
    if (tx > vectors) tx = vectors;
  }
  p.tx = tx;
  p.channel_blocks = (vectors + tx - 1) / tx;
  p.seg = kThreads / tx;
  p.tile_rows = p.seg * segment_rows(p.vec, false);
  p.back_rows = p.seg * segment_rows(p.vec, true);
  p.tiles = rows > 0 ? (rows + p.tile_rows - 1) / p.tile_rows : 1;
  p.back_tiles = rows > 0 ? (rows + p.back_rows - 1) / p.back_rows : 1;
  // Blocks that hold a part of one gate's channels (1: none is split).
  const int width = tx * p.vec;
  p.slots = 1;
  if (shared && width % per != 0) p.slots = (per + width - 2) / width + 1;
  return p;
}

template <typename XT, typename GT, int V, int R, bool SHARED>
__global__ void __launch_bounds__(kThreads, kResident) forward_kernel(const __grid_constant__ Args A) {
  __shared__ Tile<V> S;
  __shared__ int info[kThreads * R];
  int64_t tile;
  int cblk;
  take_tile(A, tile, cblk);
  Place p = place_of<V, R, SHARED>(A, tile, cblk);
  Pack<XT, V> x[R];
  Gates<GT, V, SHARED> g[R];
  {  // all loads in flight before the first use
    const XT *from = reinterpret_cast<const XT *>(A.x) + p.row * A.x_stride + p.c;
    const GT *gate = reinterpret_cast<const GT *>(A.gate) + p.row * A.gate_stride + p.g;
    const int64_t xs = along(A, A.x_stride), gs = along(A, A.gate_stride);
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < p.rows) {
        x[i] = load_pack<XT, V>(from);
        g[i].load(gate);
        from += xs;
        gate += gs;
      }
  }
  if (A.offsets != nullptr) tile_info(A, tile, info);
  int in[R];
  segment_info<R>(A, p, info, in);
  {
    float P[V], L[V];
    reduce_segment<XT, GT, V, R, SHARED>(A, p, in, x, g, P, L);
    put_segment<V>(A, p, S, segment_cut<R>(p, in, 1), P, L);
  }
  __syncthreads();
  fold_runs<V, false>(A, S);
  __syncthreads();
  const int width = A.tx * V, c0 = cblk * width;
  join_chain<V, false>(A, S, tile, cblk,
                       A.offsets != nullptr ? info[0] : A.rows > 0 ? even_info(A, p.t0) : kOutside);
  empty_sequences(A, tile, c0, c0 + width < A.channels ? c0 + width : A.channels, A.initial, A.final_state);
  if (p.rows == 0) return;
  float h[V];
  enter_segment<V, false>(A, p, S, h);
  XT *to = reinterpret_cast<XT *>(A.h) + p.row * A.channels + p.c;
  const int64_t hs = along(A, A.channels);
  // The backward's tiles begin in the middle of these, too.
  const int at = p.sg * R, halves = A.tile_rows / A.saved_rows;
  if (A.saved != nullptr && at == 0) store_state<V>(A.saved, A, tile * halves, p.c, h);
  const bool middle = A.saved != nullptr && at <= A.saved_rows && A.saved_rows < at + R;
  if (p.plain && !middle) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = fmaf(g[i](v), h[v], to_f32<XT>(x[i].e[v]));
      store_pack<XT, V>(to, h);
      to += hs;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i >= p.rows) break;
    if (middle && at + i == A.saved_rows) store_state<V>(A.saved, A, tile * halves + 1, p.c, h);
    const int row = p.plain ? 0 : in[i];
    if (row < 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = 0.f;
    } else {
      if (row & 1) load_state<V>(A.initial, A, row >> 2, p.c, h);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = fmaf(g[i](v), h[v], to_f32<XT>(x[i].e[v]));
      if ((row & 2) && A.final_state != nullptr) store_state<V>(A.final_state, A, row >> 2, p.c, h);
    }
    store_pack<XT, V>(to, h);
    to += hs;
  }
}

template <typename XT, typename GT, int V, int R, bool SHARED>
static void launch_forward(const Args &A, cudaStream_t st) {
  forward_kernel<XT, GT, V, R, SHARED><<<(unsigned)(A.tiles * A.channel_blocks), kThreads, 0, st>>>(A);
  count_launch();
}

template <typename XT, typename GT>
static void pick_forward(const Args &A, int vec, cudaStream_t st) {
  constexpr int kPer = 16 / (int)(sizeof(XT) > sizeof(GT) ? sizeof(XT) : sizeof(GT));
  constexpr int kShared = 16 / (int)sizeof(XT);
  const bool shared = A.per_gate > 1;
  if (vec == 1 && shared) launch_forward<XT, GT, 1, segment_rows(1, false), true>(A, st);
  else if (vec == 1) launch_forward<XT, GT, 1, segment_rows(1, false), false>(A, st);
  else if (shared) launch_forward<XT, GT, kShared, segment_rows(kShared, false), true>(A, st);
  else launch_forward<XT, GT, kPer, segment_rows(kPer, false), false>(A, st);
}

void run_forward(const Args &A, const Plan &p, int x_type, int gate_type, cudaStream_t st) {
  const bool same = x_type == gate_type;
  if (x_type == GS_TYPE_F32) pick_forward<float, float>(A, p.vec, st);
  else if (x_type == GS_TYPE_BF16 && same) pick_forward<__nv_bfloat16, __nv_bfloat16>(A, p.vec, st);
  else if (x_type == GS_TYPE_BF16) pick_forward<__nv_bfloat16, float>(A, p.vec, st);
  else if (same) pick_forward<__half, __half>(A, p.vec, st);
  else pick_forward<__half, float>(A, p.vec, st);
}

}  // namespace scan
}  // namespace gs

using namespace gs;

// What both directions check of their sizes, types and rows.
int gs::scan::check_shape(int64_t rows, int sequences, int channels, int gates, int x_type,
                          int gate_type, const int32_t *offsets) {
  if (rows < 0 || rows > INT32_MAX || sequences < 1 || sequences > (1 << 28) || channels < 1 ||
      gates < 1 || channels % gates != 0 || !type_bytes(x_type) ||
      (gate_type != x_type && gate_type != GS_TYPE_F32))
    return GS_ERR_INVALID_ARGUMENT;
  if (offsets == nullptr && rows % sequences != 0) return GS_ERR_INVALID_ARGUMENT;
  const Plan p = make_plan(rows, channels, gates, x_type, gate_type);
  if (p.back_tiles * p.channel_blocks > INT32_MAX / 2) return GS_ERR_CAPACITY;
  return GS_OK;
}

// Whether a row pointer and stride suit the plan's vectors.
bool gs::scan::suits(const void *p, int64_t stride, int bytes, int vec) {
  const int64_t align = (int64_t)bytes * vec > 16 ? 16 : (int64_t)bytes * vec;
  return ((uintptr_t)p % align) == 0 && (stride * bytes) % align == 0;
}

void gs::scan::fill_plan(Args &A, const Plan &p, bool back) {
  A.tx = p.tx;
  A.seg = p.seg;
  A.tile_rows = back ? p.back_rows : p.tile_rows;
  A.saved_rows = p.back_rows;
  A.channel_blocks = p.channel_blocks;
  A.tiles = back ? p.back_tiles : p.tiles;
  A.slots = p.slots;
}

using namespace gs::scan;

extern "C" size_t gs_gated_scan_saved_bytes(int64_t rows, int channels, int gates, int x_type,
                                            int gate_type) {
  if (check_shape(rows, 1, channels, gates, x_type, gate_type, nullptr)) return 0;
  return (size_t)make_plan(rows, channels, gates, x_type, gate_type).back_tiles * channels * 4;
}

extern "C" size_t gs_gated_scan_scratch_bytes(int64_t rows, int channels, int gates, int x_type,
                                              int gate_type, int backward) {
  if (check_shape(rows, 1, channels, gates, x_type, gate_type, nullptr)) return 0;
  const Plan p = make_plan(rows, channels, gates, x_type, gate_type);
  size_t bytes = chain_bytes(backward ? p.back_tiles : p.tiles, channels);
  if (backward && p.slots > 1) bytes += (size_t)p.slots * rows * gates * 4;
  return bytes;
}

extern "C" int gs_gated_scan_forward(int64_t rows, int sequences, int channels, int gates, int x_type,
                                     int gate_type, const void *x, int64_t x_row_stride,
                                     const void *gate, int64_t gate_row_stride,
                                     const float *initial, const int32_t *offsets, int reverse,
                                     void *h, float *final_state, float *saved, void *scratch,
                                     size_t scratch_bytes, void *stream) {
  const int rc = check_shape(rows, sequences, channels, gates, x_type, gate_type, offsets);
  if (rc) return rc;
  if (rows > 0 && (x == nullptr || gate == nullptr || h == nullptr)) return GS_ERR_INVALID_ARGUMENT;
  const Plan p = make_plan(rows, channels, gates, x_type, gate_type);
  const int xb = type_bytes(x_type), gb = type_bytes(gate_type);
  const bool shared = channels != gates;
  if (!suits(x, x_row_stride, xb, p.vec) || !suits(h, channels, xb, p.vec) ||
      !suits(gate, gate_row_stride, gb, shared ? 1 : p.vec) ||
      (((uintptr_t)initial | (uintptr_t)final_state | (uintptr_t)offsets | (uintptr_t)saved) & 3))
    return GS_ERR_INVALID_ARGUMENT;
  Args A{};
  fill_plan(A, p, false);
  A.rows = rows;
  A.sequences = sequences;
  A.channels = channels;
  A.gates = gates;
  A.per_gate = channels / gates;
  A.period = offsets == nullptr ? rows / sequences : 0;
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
  if (p.tiles > 1) {
    if (scratch == nullptr || ((uintptr_t)scratch & 15)) return GS_ERR_INVALID_ARGUMENT;
    if (scratch_bytes < chain_bytes(p.tiles, channels)) return GS_ERR_CAPACITY;
  }
  A.status = device_status_word();
  if (A.status == nullptr) return GS_ERR_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int failed = place_chain(A, scratch, st);
  if (failed) return failed;
  run_forward(A, p, x_type, gate_type, st);
  return launch_status();
}
