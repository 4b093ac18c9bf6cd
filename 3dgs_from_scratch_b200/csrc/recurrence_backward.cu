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

constexpr int kParts = 4;  // threads that share a sum over a gate's channels

template <typename XT, typename GT, int V, bool SHARED, bool ST>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ Args A, unsigned blocks) {
  if (blockIdx.x >= blocks) {
    look_at_sequences(A, blockIdx.x - blocks);
    return;
  }
  // [chunk of the block][row][vector], batches in turn: a batch's sums are read
  // while the next one's are written, with one barrier between.
  __shared__ float both[2][SHARED ? kThreads * kBatch : 1];
  const int cblk = blockIdx.x % A.plan.channel_blocks;
  const int64_t group = blockIdx.x / A.plan.channel_blocks;
  const auto p = place_of<V, SHARED, ST>(A, group, cblk);
  if (!SHARED && !p.on) return;
  const int64_t xs = along(A, A.x_stride), gs = along(A, A.gate_stride), ds = along(A, A.dh_stride);
  const int64_t ts = along(A, A.channels), os = along(A, A.gates);
  wait_for_previous();
  Cursor q;
  q.s = first_hint<true>(A, p.chunk);
  q.lo = q.hi = 0;
  const int one = A.reverse ? -1 : 1;
  float v_in[V];  // what the row after hands down
#pragma unroll
  for (int v = 0; v < V; ++v) v_in[v] = 0.f;
  if (A.carry != nullptr && p.on) load_kept(A.carry, A, p.chunk, p, v_in);
  for (int b = A.plan.kept - 1; b >= 0; --b) {
    float *sums = both[b & 1];
    const int64_t t = p.t0 + (int64_t)b * kBatch;
    const int n = !p.on || t >= p.t1 ? 0 : p.t1 - t < kBatch ? (int)(p.t1 - t) : kBatch;
    if (n > 0) {
      const int row = (int)row_at(A, t);
      Pack<XT, V> x[kBatch], dh[kBatch];
      Gates<GT, V, SHARED, ST> g[kBatch];
      {
        const XT *from = reinterpret_cast<const XT *>(A.x) + row * A.x_stride + p.c;
        const GT *gate = reinterpret_cast<const GT *>(A.gate) + row * A.gate_stride + p.g;
        const XT *grad = reinterpret_cast<const XT *>(A.dh) + row * A.dh_stride + p.c;
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (k < n) {
            x[k] = load_pack<XT, V, ST>(from, p);
            g[k].load(gate, p);
            from += xs;
            gate += gs;
            if (A.dh != nullptr) {
              dh[k] = load_pack<XT, V, ST>(grad, p);
              grad += ds;
            } else {
#pragma unroll
              for (int v = 0; v < V; ++v) dh[k].e[v] = from_f32<XT>(0.f);
            }
          }
      }
      float before[kBatch][V];  // the state before each row
      float h[V];
      load_kept(A.saved, A, p.chunk * A.plan.kept + b, p, h);
      const int last = row + (n - 1) * one, low = A.reverse ? last : row;
      XT *to = reinterpret_cast<XT *>(A.dx) + (int64_t)last * A.channels + p.c;
      GT *out = reinterpret_cast<GT *>(A.dgate) + (int64_t)last * A.gates + p.c;
      float *sum_at = sums + (SHARED ? p.cy * kBatch * A.plan.tx + p.tx : 0);
      const auto finish = [&](int k, bool inside) {  // row k, given what the row after it hands down
        float dg[V], sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float u = inside ? to_f32<XT>(dh[k].e[v]) + v_in[v] : 0.f;
          dg[v] = inside ? u * before[k][v] : 0.f;
          sum += dg[v];
          before[k][v] = u;
          v_in[v] = inside ? g[k](v) * u : 0.f;
        }
        store_pack<XT, V, ST>(to, before[k], p);
        to -= ts;
        if (SHARED) {
          sum_at[k * A.plan.tx] = sum;
        } else {
          store_pack<GT, V, ST>(out, dg, p);
          out -= os;
        }
      };
      if (n == kBatch && q.plain(low, kBatch)) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            before[k][v] = h[v];
            h[v] = fmaf(g[k](v), h[v], to_f32<XT>(x[k].e[v]));
          }
#pragma unroll
        for (int k = kBatch - 1; k >= 0; --k) finish(k, true);
      } else {
        // Bit k: row k is its sequence's first, its last, outside every sequence.
        uint32_t firsts = 0, lasts = 0, outside = 0;
        for (int k = 0; k < n;) {
          const int at = row + k * one;
          q.seek(A, at);
          const int rest = q.rest(A, at), end = rest < n - k ? k + rest : n;
          if (!q.holds(at)) {
            outside |= (1u << end) - (1u << k);
          } else {
            if (q.first(A, at)) firsts |= 1u << k;
            if (rest <= n - k) lasts |= 1u << (end - 1);
          }
          k = end;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (k >= n) break;
          if (firsts >> k & 1) {
            q.seek(A, row + k * one);
            load_state(A.initial, A, q.s, p, h);
          }
#pragma unroll
          for (int v = 0; v < V; ++v) {
            before[k][v] = h[v];
            h[v] = outside >> k & 1 ? 0.f : fmaf(g[k](v), h[v], to_f32<XT>(x[k].e[v]));
          }
        }
#pragma unroll
        for (int k = kBatch - 1; k >= 0; --k) {
          if (k >= n) continue;
          if ((firsts | lasts) >> k & 1) q.seek(A, row + k * one);
          if (lasts >> k & 1) load_state(A.dfinal, A, q.s, p, v_in);
          finish(k, !(outside >> k & 1));
          if ((firsts >> k & 1) && A.dinitial != nullptr) store_state(A.dinitial, A, q.s, p, v_in);
        }
      }
    }
    if (SHARED) {
      // The sums of the threads that share a gate, in their order.
      __syncthreads();
      const int width = A.plan.width, c0 = cblk * width, c1 = c0 + width < A.channels ? c0 + width : A.channels;
      const int first = c0 / A.per_gate, count = (c1 - 1) / A.per_gate - first + 1;
      // kParts adjacent lanes share a sum.
      const int all = A.plan.cy * kBatch * count;
      for (int j = threadIdx.x / kParts; j < (all + 7) / 8 * 8; j += kThreads / kParts) {
        const int line = count == 1 ? j : j / count, at = first + (count == 1 ? 0 : j % count);
        const int lo = at * A.per_gate > c0 ? at * A.per_gate : c0;
        const int hi = (at + 1) * A.per_gate < c1 ? (at + 1) * A.per_gate : c1;
        float sum = 0.f;
        if (j < all) {
          const float *from = sums + line * A.plan.tx, *end = from + (hi - c0) / V;
#pragma unroll 4
          for (from += (lo - c0) / V + threadIdx.x % kParts; from < end; from += kParts) sum += *from;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int64_t chunk = group * A.plan.cy + line / kBatch;
        const int in_chunk = b * kBatch + line % kBatch;
        const int64_t r = chunk * A.plan.chunk + in_chunk;
        if (threadIdx.x % kParts != 0 || j >= all || chunk >= A.plan.chunks || r >= A.rows ||
            in_chunk >= A.plan.chunk)
          continue;
        const int64_t row = row_at(A, r);
        if (A.partial == nullptr) {
          reinterpret_cast<GT *>(A.dgate)[row * A.gates + at] = from_f32<GT>(sum);
        } else {
          const int slot = cblk - at * A.per_gate / width;
          A.partial[((int64_t)slot * A.rows + row) * A.gates + at] = sum;
        }
      }
    }
  }
}

// The gates whose channels lie in several blocks: their parts added in order.
template <typename GT>
__global__ void __launch_bounds__(kThreads) join_gates_kernel(const __grid_constant__ Args A) {
  const int width = A.plan.width;
  const int64_t n = A.rows * A.gates, stride = (int64_t)gridDim.x * kThreads;
  for (int64_t k = (int64_t)blockIdx.x * kThreads + threadIdx.x; k < n; k += stride) {
    const int gate = (int)(k % A.gates);
    const int first = gate * A.per_gate / width, last = ((gate + 1) * A.per_gate - 1) / width;
    float sum = 0.f;
    for (int s = 0; s <= last - first; ++s) sum += A.partial[s * n + k];
    reinterpret_cast<GT *>(A.dgate)[k] = from_f32<GT>(sum);
  }
}

template <typename XT, typename GT, int V, bool SHARED, bool ST>
static int launch_backward(const Args &A, cudaStream_t st) {
  if (A.carry != nullptr) {
    const unsigned blocks = grid_of(A.plan);
    maps_kernel<XT, GT, V, SHARED, ST, true><<<blocks + extra_blocks(A), kThreads, 0, st>>>(A, blocks);
    count_launch();
    const int rc = launch_carry(A, true, st);
    if (rc) return rc;
  }
  const int rc = launch_walk(backward_kernel<XT, GT, V, SHARED, ST>, A, st);
  if (rc) return rc;
  if (A.partial != nullptr && A.rows > 0) {
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
  constexpr bool kApart = sizeof(XT) == 2 && sizeof(GT) == 2;
  const bool shared = A.per_gate > 1;
  if (A.plan.step) return launch_backward<XT, GT, kApart ? 2 : 1, false, kApart>(A, st);
  if (A.plan.vec == 1)
    return shared ? launch_backward<XT, GT, 1, true, false>(A, st) : launch_backward<XT, GT, 1, false, false>(A, st);
  return shared ? launch_backward<XT, GT, kShared, true, false>(A, st)
                : launch_backward<XT, GT, kPer, false, false>(A, st);
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
  const int xb = type_bytes(x_type), gb = type_bytes(gate_type), vec = A.plan.step ? 1 : A.plan.vec;
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
    if (A.plan.slots > 1)
      A.partial = reinterpret_cast<float *>(static_cast<char *>(scratch) + chain_bytes(A.plan, channels));
  }
  A.status = device_status_word();
  if (A.status == nullptr) return GS_ERR_CUDA;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  A.empty_src = grad_final;
  A.empty_dst = grad_initial;
  const bool same = x_type == gate_type;
  if (x_type == GS_TYPE_F32) return pick_backward<float, float>(A, st);
  if (x_type == GS_TYPE_BF16)
    return same ? pick_backward<__nv_bfloat16, __nv_bfloat16>(A, st) : pick_backward<__nv_bfloat16, float>(A, st);
  return same ? pick_backward<__half, __half>(A, st) : pick_backward<__half, float>(A, st);
}
