// recurrence_backward.cu -- the gated recurrence's gradients (see
// recurrence.cuh for the tiles).
//
// With u_t = dh_t + g_{t+1} u_{t+1} the gradient that reaches h_t, the chain
// runs over v_t = g_t u_t, what row t hands to row t - 1, so that a row needs
// only its own gate:
//   v_t = g_t (dh_t + v_{t+1}), v after the last row = dfinal;
//   dx_t = u_t = dh_t + v_{t+1};  dg_t = sum over the gate's channels of u_t h_{t-1};
//   dinitial = v of the first row.
// The states h_{t-1} are recomputed in 32 bits from x, the gates and the state
// that the forward kept before each tile: the rounded h of a 16-bit run would
// cost the gates' gradient its last bits, and reading it costs as much as
// reading x.
#include "recurrence.cuh"

namespace gs {
namespace scan {

template <typename XT, typename GT, int V, int R, bool SHARED>
__global__ void __launch_bounds__(kThreads, kResident) backward_kernel(const __grid_constant__ Args A) {
  __shared__ Tile<V> S;
  __shared__ int info[kThreads * R];
  __shared__ float sums[SHARED ? kThreads * R : 1];
  int64_t position;
  int cblk;
  take_tile(A, position, cblk);
  const int64_t tile = A.tiles - 1 - position;
  const int width = A.tx * V, c0 = cblk * width, c1 = c0 + width < A.channels ? c0 + width : A.channels;
  Place p = place_of<V, R, SHARED>(A, tile, cblk);
  Pack<XT, V> x[R], dh[R];
  Gates<GT, V, SHARED> g[R];
  {  // all loads in flight before the first use
    const XT *from = reinterpret_cast<const XT *>(A.x) + p.row * A.x_stride + p.c;
    const XT *grad = reinterpret_cast<const XT *>(A.dh) + p.row * A.dh_stride + p.c;
    const GT *gate = reinterpret_cast<const GT *>(A.gate) + p.row * A.gate_stride + p.g;
    const int64_t xs = along(A, A.x_stride), gs = along(A, A.gate_stride), ds = along(A, A.dh_stride);
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < p.rows) {
        x[i] = load_pack<XT, V>(from);
        g[i].load(gate);
        if (A.dh != nullptr) {
          dh[i] = load_pack<XT, V>(grad);
          grad += ds;
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) dh[i].e[v] = from_f32<XT>(0.f);
        }
        from += xs;
        gate += gs;
      }
  }
  if (threadIdx.x < width)
    S.carry[threadIdx.x] = c0 + threadIdx.x < A.channels ? A.saved[tile * A.channels + c0 + threadIdx.x] : 0.f;
  if (A.offsets != nullptr) tile_info(A, tile, info);
  int in[R];
  segment_info<R>(A, p, info, in);
  float before[R][V];  // the state before each row
  {
    float P[V], L[V];
    reduce_segment<XT, GT, V, R, SHARED>(A, p, in, x, g, P, L);
    put_segment<V>(A, p, S, segment_cut<R>(p, in, 1), P, L);
  }
  __syncthreads();
  fold_runs<V, false>(A, S);
  __syncthreads();
  if (p.rows > 0) {
    float h[V];
    enter_segment<V, false>(A, p, S, h);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= p.rows) break;
      const int row = p.plain ? 0 : in[i];
      if (row > 0 && (row & 1)) load_state<V>(A.initial, A, row >> 2, p.c, h);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        before[i][v] = h[v];
        h[v] = row < 0 ? 0.f : fmaf(g[i](v), h[v], to_f32<XT>(x[i].e[v]));
      }
    }
  }
  {
    float P[V], L[V];
    reduce_segment_back<XT, GT, V, R, SHARED>(A, p, in, dh, g, P, L);
    __syncthreads();
    put_segment<V>(A, p, S, segment_cut<R>(p, in, 2), P, L);
  }
  __syncthreads();
  fold_runs<V, true>(A, S);
  __syncthreads();
  const int64_t left = A.rows - p.t0;
  const int rows = left < A.tile_rows ? (int)left : A.tile_rows;
  join_chain<V, true>(A, S, position, cblk,
                      rows <= 0              ? kOutside
                      : A.offsets != nullptr ? info[rows - 1]
                                             : even_info(A, p.t0 + rows - 1));
  empty_sequences(A, tile, c0, c1, A.dfinal, A.dinitial);
  if (p.rows > 0) {
    float after[V];
    enter_segment<V, true>(A, p, S, after);
    const int64_t last = p.row + along(A, p.rows - 1);
    XT *to = reinterpret_cast<XT *>(A.dx) + last * A.channels + p.c;
    GT *gate = reinterpret_cast<GT *>(A.dgate) + last * A.gates + p.c;
    const int64_t ts = along(A, A.channels), gs = along(A, A.gates);
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      if (i >= p.rows) continue;
      const int row = p.plain ? 0 : in[i];
      float u[V], dg[V], sum = 0.f;
      if (row < 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) u[v] = dg[v] = after[v] = 0.f;
      } else {
        if (row & 2) load_state<V>(A.dfinal, A, row >> 2, p.c, after);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          u[v] = to_f32<XT>(dh[i].e[v]) + after[v];
          dg[v] = u[v] * before[i][v];
          after[v] = g[i](v) * u[v];
          sum += dg[v];
        }
        if ((row & 1) && A.dinitial != nullptr) store_state<V>(A.dinitial, A, row >> 2, p.c, after);
      }
      store_pack<XT, V>(to, u);
      to -= ts;
      if (SHARED) {
        sums[(p.sg * R + i) * A.tx + p.tx] = sum;
      } else {
        store_pack<GT, V>(gate, dg);
        gate -= gs;
      }
    }
  }
  if (!SHARED) return;
  // The sums of the threads that share a gate, in their order.
  __syncthreads();
  const int first = c0 / A.per_gate, count = (c1 - 1) / A.per_gate - first + 1;
  for (int k = threadIdx.x; k < rows * count; k += kThreads) {
    const int i = k / count, gate = first + k % count;
    const int lo = gate * A.per_gate > c0 ? gate * A.per_gate : c0;
    const int hi = (gate + 1) * A.per_gate < c1 ? (gate + 1) * A.per_gate : c1;
    float sum = 0.f;
    for (int c = lo; c < hi; c += V) sum += sums[i * A.tx + (c - c0) / V];
    const int64_t t = p.t0 + i, row = A.reverse ? A.rows - 1 - t : t;
    if (A.partial == nullptr) {
      reinterpret_cast<GT *>(A.dgate)[row * A.gates + gate] = from_f32<GT>(sum);
    } else {
      const int slot = cblk - gate * A.per_gate / width;
      A.partial[((int64_t)slot * A.rows + row) * A.gates + gate] = sum;
    }
  }
}

// The gates whose channels lie in several blocks: their parts added in order.
template <typename GT>
__global__ void __launch_bounds__(kThreads) join_gates_kernel(const Args A, int width) {
  const int64_t n = A.rows * A.gates, stride = (int64_t)gridDim.x * kThreads;
  for (int64_t k = (int64_t)blockIdx.x * kThreads + threadIdx.x; k < n; k += stride) {
    const int gate = (int)(k % A.gates);
    const int first = gate * A.per_gate / width, last = ((gate + 1) * A.per_gate - 1) / width;
    float sum = 0.f;
    for (int s = 0; s <= last - first; ++s) sum += A.partial[s * n + k];
    reinterpret_cast<GT *>(A.dgate)[k] = from_f32<GT>(sum);
  }
}

template <typename XT, typename GT, int V, int R, bool SHARED>
static void launch_backward(const Args &A, cudaStream_t st) {
  backward_kernel<XT, GT, V, R, SHARED><<<(unsigned)(A.tiles * A.channel_blocks), kThreads, 0, st>>>(A);
  count_launch();
  if (A.partial != nullptr && A.rows > 0) {
    const int64_t want = (A.rows * A.gates + kThreads - 1) / kThreads;
    join_gates_kernel<GT><<<(unsigned)(want < 1184 ? want : 1184), kThreads, 0, st>>>(A, A.tx * V);
    count_launch();
  }
}

template <typename XT, typename GT>
static void pick_backward(const Args &A, int vec, cudaStream_t st) {
  constexpr int kPer = 16 / (int)(sizeof(XT) > sizeof(GT) ? sizeof(XT) : sizeof(GT));
  constexpr int kShared = 16 / (int)sizeof(XT);
  const bool shared = A.per_gate > 1;
  if (vec == 1 && shared) launch_backward<XT, GT, 1, segment_rows(1, true), true>(A, st);
  else if (vec == 1) launch_backward<XT, GT, 1, segment_rows(1, true), false>(A, st);
  else if (shared) launch_backward<XT, GT, kShared, segment_rows(kShared, true), true>(A, st);
  else launch_backward<XT, GT, kPer, segment_rows(kPer, true), false>(A, st);
}

}  // namespace scan
}  // namespace gs

using namespace gs;
using namespace gs::scan;

extern "C" int gs_gated_scan_backward(int64_t rows, int sequences, int channels, int gates,
                                      int x_type, int gate_type, const void *x,
                                      int64_t x_row_stride, const void *gate,
                                      int64_t gate_row_stride, const float *initial,
                                      const int32_t *offsets, int reverse, const float *saved,
                                      const void *grad_h, int64_t grad_h_row_stride,
                                      const float *grad_final, void *grad_x, void *grad_gate,
                                      float *grad_initial, void *scratch, size_t scratch_bytes,
                                      void *stream) {
  const int rc = check_shape(rows, sequences, channels, gates, x_type, gate_type, offsets);
  if (rc) return rc;
  if (rows > 0 && (x == nullptr || gate == nullptr || saved == nullptr || grad_x == nullptr ||
                   grad_gate == nullptr))
    return GS_ERR_INVALID_ARGUMENT;
  const Plan p = make_plan(rows, channels, gates, x_type, gate_type);
  const int xb = type_bytes(x_type), gb = type_bytes(gate_type);
  const bool shared = channels != gates;
  if (!suits(x, x_row_stride, xb, p.vec) || !suits(grad_x, channels, xb, p.vec) ||
      !suits(grad_h, grad_h_row_stride, xb, p.vec) ||
      !suits(gate, gate_row_stride, gb, shared ? 1 : p.vec) ||
      !suits(grad_gate, gates, gb, shared ? 1 : p.vec) ||
      (((uintptr_t)initial | (uintptr_t)grad_initial | (uintptr_t)grad_final | (uintptr_t)offsets |
        (uintptr_t)saved) & 3))
    return GS_ERR_INVALID_ARGUMENT;
  Args A{};
  fill_plan(A, p, true);
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
  A.dh = grad_h;
  A.dh_stride = grad_h_row_stride;
  A.initial = initial;
  A.dfinal = grad_final;
  A.dx = grad_x;
  A.dgate = grad_gate;
  A.dinitial = grad_initial;
  A.saved = const_cast<float *>(saved);
  if (p.back_tiles > 1 || p.slots > 1) {
    if (scratch == nullptr || ((uintptr_t)scratch & 15)) return GS_ERR_INVALID_ARGUMENT;
    if (scratch_bytes < gs_gated_scan_scratch_bytes(rows, channels, gates, x_type, gate_type, 1))
      return GS_ERR_CAPACITY;
  }
  if (p.slots > 1)
    A.partial = reinterpret_cast<float *>(static_cast<char *>(scratch) + chain_bytes(p.back_tiles, channels));
  A.status = device_status_word();
  if (A.status == nullptr) return GS_ERR_CUDA;
  const bool same = x_type == gate_type;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int failed = place_chain(A, scratch, st);
  if (failed) return failed;
  if (x_type == GS_TYPE_F32) pick_backward<float, float>(A, p.vec, st);
  else if (x_type == GS_TYPE_BF16 && same) pick_backward<__nv_bfloat16, __nv_bfloat16>(A, p.vec, st);
  else if (x_type == GS_TYPE_BF16) pick_backward<__nv_bfloat16, float>(A, p.vec, st);
  else if (same) pick_backward<__half, __half>(A, p.vec, st);
  else pick_backward<__half, float>(A, p.vec, st);
  return launch_status();
}
