// recurrence_backward.cu -- the gated recurrence's gradients (see
// recurrence.cuh).
//
// With u_t = dh_t + g_{t+1} u_{t+1} the gradient that reaches h_t, the chain
// runs over v_t = g_t u_t, what row t hands to row t - 1, so that a row needs
// only its own gate:
//   v_t = g_t (dh_t + v_{t+1}), v after the last row = dfinal;
//   dx_t = u_t = dh_t + v_{t+1};  dg_t = sum over the gate's channels of u_t h_{t-1};
//   dinitial = v of the first row.
// A thread walks its chunk against the rows, a batch at a time. The states
// h_{t-1} of a batch are recomputed in 32 bits from x, the gates and the state
// that the forward kept before the batch: the rounded h of a 16-bit run would
// cost the gates' gradient its last bits, and reading it costs as much as
// reading x.
#include "recurrence.cuh"

namespace gs {
namespace scan {

template <typename XT, typename GT, int V, bool SHARED>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ Args A) {
  __shared__ float sums[SHARED ? kThreads * kBatch : 1];  // [chunk of the block][row][vector]
  const int cblk = blockIdx.x % A.plan.channel_blocks;
  const int64_t group = blockIdx.x / A.plan.channel_blocks;
  const Place p = place_of<V, SHARED>(A, group, cblk);
  if (!SHARED && !p.on) return;
  const int64_t xs = along(A, A.x_stride), gs = along(A, A.gate_stride), ds = along(A, A.dh_stride);
  const int64_t ts = along(A, A.channels), os = along(A, A.gates);
  Cursor q;
  q.s = A.hints != nullptr && p.on ? A.hints[p.chunk + A.plan.chunks] : 0;
  q.lo = q.hi = 0;
  float v_in[V];  // what the row after hands down
#pragma unroll
  for (int v = 0; v < V; ++v) v_in[v] = 0.f;
  if (A.carry != nullptr && p.on) load_kept<V>(A.carry, A, p.chunk, p.c, v_in);
  Pack<XT, V> x[kBatch], dh[kBatch];
  Gates<GT, V, SHARED> g[kBatch];
  const auto rows_of = [&](int b) {  // of batch b
    const int64_t t = p.t0 + (int64_t)b * kBatch;
    return b < 0 || !p.on || t >= p.t1 ? 0 : p.t1 - t < kBatch ? (int)(p.t1 - t) : kBatch;
  };
  const auto load = [&](int b) {
    const int n = rows_of(b);
    const int64_t row = row_at(A, p.t0 + (int64_t)b * kBatch);
    const XT *from = reinterpret_cast<const XT *>(A.x) + row * A.x_stride + p.c;
    const GT *gate = reinterpret_cast<const GT *>(A.gate) + row * A.gate_stride + p.g;
    const XT *grad = reinterpret_cast<const XT *>(A.dh) + row * A.dh_stride + p.c;
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (k < n) {
        x[k] = load_pack<XT, V>(from + k * xs);
        g[k].load(gate + k * gs);
        if (A.dh != nullptr) {
          dh[k] = load_pack<XT, V>(grad + k * ds);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) dh[k].e[v] = from_f32<XT>(0.f);
        }
      }
  };
  // Where the block adds up gates between two batches, the next one is on its
  // way meanwhile.
  if (SHARED) load(A.plan.kept - 1);
  for (int b = A.plan.kept - 1; b >= 0; --b) {
    const int n = rows_of(b);
    if (!SHARED) load(b);
    if (n > 0) {
      const int64_t row = row_at(A, p.t0 + (int64_t)b * kBatch);
      float before[kBatch][V];  // the state before each row
      float h[V];
      load_kept<V>(A.saved, A, p.chunk * A.plan.kept + b, p.c, h);
      XT *to = reinterpret_cast<XT *>(A.dx) + row * A.channels + p.c;
      GT *out = reinterpret_cast<GT *>(A.dgate) + row * A.gates + p.c;
      const auto finish = [&](int k) {  // row k, given what the row after it hands down
        float dg[V], sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float u = to_f32<XT>(dh[k].e[v]) + v_in[v];
          dg[v] = u * before[k][v];
          sum += dg[v];
          before[k][v] = u;
          v_in[v] = g[k](v) * u;
        }
        store_pack<XT, V>(to + k * ts, before[k]);
        if (SHARED) sums[(p.cy * kBatch + k) * A.plan.tx + p.tx] = sum;
        else store_pack<GT, V>(out + k * os, dg);
      };
      const int64_t low = A.reverse ? row - (n - 1) : row;  // the batch's rows of the tensor
      if (!q.holds(low)) q.seek(A, low);
      if (n == kBatch && plain_rows(q, low, kBatch)) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            before[k][v] = h[v];
            h[v] = fmaf(g[k](v), h[v], to_f32<XT>(x[k].e[v]));
          }
#pragma unroll
        for (int k = kBatch - 1; k >= 0; --k) finish(k);
      } else {
        int state[kBatch];  // 4 * sequence + 2 * (its last row) + (its first row), or -1
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (k >= n) break;
          const int64_t at = A.reverse ? row - k : row + k;
          if (!q.holds(at)) q.seek(A, at);
          const bool low_end = at == q.lo, high_end = at == q.hi - 1;
          state[k] = !q.holds(at) ? -1
                                  : q.s * 4 + ((A.reverse ? low_end : high_end) ? 2 : 0) +
                                        ((A.reverse ? high_end : low_end) ? 1 : 0);
          if (state[k] >= 0 && (state[k] & 1)) load_state<V>(A.initial, A, q.s, p.c, h);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            before[k][v] = h[v];
            h[v] = state[k] < 0 ? 0.f : fmaf(g[k](v), h[v], to_f32<XT>(x[k].e[v]));
          }
        }
#pragma unroll
        for (int k = kBatch - 1; k >= 0; --k) {
          if (k >= n) continue;
          if (state[k] < 0) {
            const float zero[V] = {};
#pragma unroll
            for (int v = 0; v < V; ++v) v_in[v] = 0.f;
            store_pack<XT, V>(to + k * ts, zero);
            if (SHARED) sums[(p.cy * kBatch + k) * A.plan.tx + p.tx] = 0.f;
            else store_pack<GT, V>(out + k * os, zero);
            continue;
          }
          if (state[k] & 2) load_state<V>(A.dfinal, A, state[k] >> 2, p.c, v_in);
          finish(k);
          if ((state[k] & 1) && A.dinitial != nullptr) store_state<V>(A.dinitial, A, state[k] >> 2, p.c, v_in);
        }
      }
    }
    if (SHARED) {
      load(b - 1);
      // The sums of the threads that share a gate, in their order.
      __syncthreads();
      const int width = A.plan.tx * V, c0 = cblk * width, c1 = c0 + width < A.channels ? c0 + width : A.channels;
      const int first = c0 / A.per_gate, count = (c1 - 1) / A.per_gate - first + 1;
      // A sum is shared out to as many adjacent lanes as there are threads for.
      const int all = A.plan.cy * kBatch * count;
      int parts = 1;
      while (parts < 32 && parts * 2 * all <= kThreads) parts *= 2;
      for (int j = threadIdx.x; j < (all * parts + 31) / 32 * 32; j += kThreads) {
        const int k = j / parts, part = j % parts, line = k / count, at = first + k % count;
        const int lo = at * A.per_gate > c0 ? at * A.per_gate : c0;
        const int hi = (at + 1) * A.per_gate < c1 ? (at + 1) * A.per_gate : c1;
        float sum = 0.f;
        if (k < all)
          for (int c = lo + part * V; c < hi; c += parts * V) sum += sums[line * A.plan.tx + (c - c0) / V];
        for (int d = parts / 2; d > 0; d /= 2) sum += __shfl_down_sync(0xffffffffu, sum, d);
        const int64_t chunk = group * A.plan.cy + line / kBatch;
        const int64_t r = chunk * A.plan.chunk + b * kBatch + line % kBatch;
        if (part != 0 || k >= all || chunk >= A.plan.chunks || r >= A.rows ||
            b * kBatch + line % kBatch >= A.plan.chunk)
          continue;
        const int64_t row = row_at(A, r);
        if (A.partial == nullptr) {
          reinterpret_cast<GT *>(A.dgate)[row * A.gates + at] = from_f32<GT>(sum);
        } else {
          const int slot = cblk - at * A.per_gate / width;
          A.partial[((int64_t)slot * A.rows + row) * A.gates + at] = sum;
        }
      }
      __syncthreads();
    }
  }
}

// The gates whose channels lie in several blocks: their parts added in order.
template <typename GT>
__global__ void __launch_bounds__(kThreads) join_gates_kernel(const __grid_constant__ Args A) {
  const int width = A.plan.tx * A.plan.vec;
  const int64_t n = A.rows * A.gates, stride = (int64_t)gridDim.x * kThreads;
  for (int64_t k = (int64_t)blockIdx.x * kThreads + threadIdx.x; k < n; k += stride) {
    const int gate = (int)(k % A.gates);
    const int first = gate * A.per_gate / width, last = ((gate + 1) * A.per_gate - 1) / width;
    float sum = 0.f;
    for (int s = 0; s <= last - first; ++s) sum += A.partial[s * n + k];
    reinterpret_cast<GT *>(A.dgate)[k] = from_f32<GT>(sum);
  }
}

template <typename XT, typename GT, int V, bool SHARED>
static int launch_backward(const Args &A, cudaStream_t st) {
  if (A.carry != nullptr) {
    maps_kernel<XT, GT, V, SHARED, true><<<grid_of(A.plan), kThreads, 0, st>>>(A);
    count_launch();
    const int rc = launch_carry(A, true, st);
    if (rc) return rc;
  }
  backward_kernel<XT, GT, V, SHARED><<<grid_of(A.plan), kThreads, 0, st>>>(A);
  count_launch();
  if (A.partial != nullptr) {
    const int64_t want = (A.rows * A.gates + kThreads - 1) / kThreads;
    join_gates_kernel<GT><<<(unsigned)(want < 1184 ? want : 1184), kThreads, 0, st>>>(A);
    count_launch();
  }
  return launch_status();
}

template <typename XT, typename GT>
static int pick_backward(const Args &A, cudaStream_t st) {
  constexpr int kPer = 8 / (int)(sizeof(XT) > sizeof(GT) ? sizeof(XT) : sizeof(GT));
  constexpr int kShared = 8 / (int)sizeof(XT);
  const bool shared = A.per_gate > 1;
  if (A.plan.vec == 1)
    return shared ? launch_backward<XT, GT, 1, true>(A, st) : launch_backward<XT, GT, 1, false>(A, st);
  return shared ? launch_backward<XT, GT, kShared, true>(A, st) : launch_backward<XT, GT, kPer, false>(A, st);
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
  const int even = offsets == nullptr;
  int rc = check_shape(rows, sequences, channels, gates, x_type, gate_type, even);
  if (rc) return rc;
  if (rows > 0 && (x == nullptr || gate == nullptr || saved == nullptr || grad_x == nullptr ||
                   grad_gate == nullptr))
    return GS_ERR_INVALID_ARGUMENT;
  Args A{};
  A.plan = make_plan(rows, sequences, even, channels, gates, x_type, gate_type);
  const int xb = type_bytes(x_type), gb = type_bytes(gate_type), vec = A.plan.vec;
  const bool shared = channels != gates;
  if (!suits(x, x_row_stride, xb, vec) || !suits(grad_x, channels, xb, vec) ||
      !suits(grad_h, grad_h_row_stride, xb, vec) ||
      !suits(gate, gate_row_stride, gb, shared ? 1 : vec) ||
      !suits(grad_gate, gates, gb, shared ? 1 : vec) ||
      (((uintptr_t)initial | (uintptr_t)grad_initial | (uintptr_t)grad_final | (uintptr_t)offsets) &
       3) ||
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
  A.dh = grad_h;
  A.dh_stride = grad_h_row_stride;
  A.initial = initial;
  A.dfinal = grad_final;
  A.dx = grad_x;
  A.dgate = grad_gate;
  A.dinitial = grad_initial;
  A.saved = const_cast<float *>(saved);
  const size_t need = gs_gated_scan_scratch_bytes(rows, sequences, even, channels, gates, x_type, gate_type, 1);
  if (need > 0) {
    if (scratch == nullptr || ((uintptr_t)scratch & 15)) return GS_ERR_INVALID_ARGUMENT;
    if (scratch_bytes < need) return GS_ERR_CAPACITY;
    place_chain(A, scratch);
    if (even) A.hints = nullptr;
    if (A.plan.slots > 1)
      A.partial = reinterpret_cast<float *>(static_cast<char *>(scratch) + chain_bytes(A.plan, channels));
  }
  A.status = device_status_word();
  if (A.status == nullptr) return GS_ERR_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = launch_setup(A, grad_final, grad_initial, st);
  if (rc || rows == 0) return rc;
  const bool same = x_type == gate_type;
  if (x_type == GS_TYPE_F32) return pick_backward<float, float>(A, st);
  if (x_type == GS_TYPE_BF16)
    return same ? pick_backward<__nv_bfloat16, __nv_bfloat16>(A, st) : pick_backward<__nv_bfloat16, float>(A, st);
  return same ? pick_backward<__half, __half>(A, st) : pick_backward<__half, float>(A, st);
}
