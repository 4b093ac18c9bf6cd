// orthogonalize.cu -- an update matrix brought near its orthogonal factor by
// Newton-Schulz products, and the optimizer step built on it.
//
// X0 = U / max(|U|_F, eps) (transposed where U is tall, so that X is m x n
// with m <= n), then `steps` times
//   A = X X^T;  B = b A + c A A;  X = a X + B X,
// an odd quintic p(s) = a s + b s^3 + c s^5 on X's singular values.
//
// Numbers. The products run on the tensor cores with fp16 operands and fp32
// accumulators. A value is held as hi + lo, two fp16 numbers (22 bits), scaled
// by 2^12 so that neither leaves fp16's range, which ends at 15.99: |X|_2 and
// |B|_2 stay below 8 and |A|_2 = |X|_2^2 below 15 (checked by the host for the
// given coefficients), and a typical entry of even the largest matrix is far
// above the smallest normal number.
//   full (fp32 and fp16 results): every product is hi hi + hi lo + lo hi. The
//     tensor core cuts its fp32 sums off instead of rounding them, a bias that
//     grows with the number of additions (2.6e-5 of the result at 4096 x 4096
//     with one accumulator for all of K); so each 256 elements of K start a
//     fresh accumulator, and these parts are added in registers, rounded.
//     half products start one every 8192 elements (a bias of 2e-5), which also
//     keeps the longest wait for an accumulator short.
//   half (bf16 results, 2^-9 a rounding): A and B are computed from and held
//     as hi alone. Their errors (2^-12) multiply each singular direction by
//     1 + small and mix left directions only, so a small singular value keeps
//     its relative accuracy; X's own rounding would not do that (it adds to
//     every direction alike, and the small ones grow 3.4-fold a step), so X
//     keeps hi + lo in a X + B X. Two products there, one in A and in A A.
//
// Layout. Every matrix lies in the workspace as 128 x 64 blocks of fp16, each
// the 16 KB image of 128 rows of 128 bytes in the tensor core's 128-byte
// swizzle (16-byte chunk j of row r at chunk j ^ (r & 7)). A block is fetched
// with one contiguous bulk copy, and the same image serves as a K-major
// operand (rows along M or N) and, 64 of its rows at a time, as an MN-major
// one (rows along K): X needs no transposed copy, and of the symmetric A and
// B only the blocks on and above the diagonal are computed and stored, the
// others read as their mirror images.
//
// Padding to whole blocks is zero from the start and stays zero.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "tcgen05.cuh"

namespace gs {
namespace ns {

constexpr int kBlockBytes = 128 * 64 * 2;
constexpr int kMaxStages = 8;
constexpr float kScale = 4096.f, kUnscale = 1.f / 4096.f;

enum Kind { kGram, kSquare, kApply };

struct Matrix {        // planes of blocks [row block][column block]
  char *hi, *lo;       // lo may be null
  int64_t batch_bytes;
  int column_blocks;
};

struct Out {
  void *p;             // the result, or the weights that it updates; null: none
  int type;            // GS_TYPE_*
  int update;          // p = decay p - step X instead of p = X, unless the call's gate is closed
  int tall;            // X is the transpose
  int rows, cols;      // of X
  int64_t batch_stride;
  float decay, step;
};

struct Args {
  Matrix x, y, sq, poly;  // X, the next X, A, B
  int tiles, row_tiles, batches;  // of a product: tiles of a matrix, rows of them, matrices
  int k_blocks_n, k_blocks_m;     // 64-wide K blocks that hold data
  int stages;
  float a, b, c;
  Out out;
  uint32_t *status;
  uint32_t *gate;      // of an optimizer step: not 0: nothing is updated; null otherwise
};

// The optimizers' gate, read once for all launches and blocks of a step: a status
// word that another stream sets meanwhile skips the next step, never a part of
// this one. A wait that runs out inside the step closes it as well.
__global__ void gate_kernel(const uint32_t *status, uint32_t *gate) {
  start_next();
  *gate = ld_volatile_u32(status);
}
__device__ __forceinline__ void report_timeout(uint32_t *status, uint32_t *gate) {
  atomicCAS(status, 0u, (uint32_t)GS_ERR_DEVICE_TIMEOUT);
  if (gate != nullptr) atomicExch(gate, (uint32_t)GS_ERR_DEVICE_TIMEOUT);
}

__device__ __forceinline__ char *block_at(char *plane, const Matrix &M, int batch, int rb, int cb) {
  return plane + (int64_t)batch * M.batch_bytes + ((int64_t)rb * M.column_blocks + cb) * kBlockBytes;
}

// Byte of the 16-byte chunk that holds columns col..col+7 of row r in a block.
__device__ __forceinline__ int chunk_at(int r, int col) {
  return r * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4);
}

// One plane's rows of an operand: `rows` rows from `row` on, K block kb, into
// shared memory. Above or on the diagonal (of blocks of `tri`) of a symmetric
// matrix, and always for X, as K-major rows; below it as the mirror image,
// MN-major.
__device__ __forceinline__ void fetch_rows(char *plane, const Matrix &M, int batch, int row, int rows,
                                           int kb, bool mirrored, char *dst, uint64_t *bar) {
  if (!mirrored) {
    if (rows < 128) {
      bulk_load(dst, block_at(plane, M, batch, row / 128, kb) + (row % 128) * 128, rows * 128, bar);
    } else {
      for (int u = 0; u < rows / 128; ++u)
        bulk_load(dst + u * kBlockBytes, block_at(plane, M, batch, row / 128 + u, kb), kBlockBytes, bar);
    }
  } else {
    for (int u = 0; u < rows / 64; ++u)
      bulk_load(dst + u * (kBlockBytes / 2),
                block_at(plane, M, batch, kb / 2, row / 64 + u) + (kb & 1) * (kBlockBytes / 2),
                kBlockBytes / 2, bar);
  }
}

// An operand's descriptor, and what 16 elements of K further add to it: 32
// bytes along a row, or 16 rows of 128 bytes (in units of 16 bytes).
template <bool MN>
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  return MN ? tc::descriptor(addr, kBlockBytes / 2, 1024) : tc::descriptor(addr, 16, 1024);
}

// The MMAs of one K block. `main` takes hi hi, `cross` hi lo and lo hi (it may
// be the same accumulator).
template <class S, bool A_MN, bool B_MN, bool FRESH>
__device__ __forceinline__ void issue_block(uint32_t at, uint32_t main, uint32_t cross) {
  constexpr uint32_t kInstr = tc::instruction_f16(128 * S::kCtas, S::kBN, A_MN, B_MN);
  constexpr int kA = A_MN ? 128 : 2, kB = B_MN ? 128 : 2;
  const uint64_t a = operand<A_MN>(at), b = operand<B_MN>(at + S::kPlanesA * S::kPlaneA);
  constexpr int kLoA = S::kPlaneA / 16, kLoB = S::kPlaneB / 16;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (FRESH && k == 0) tc::mma_f16<S::kCtas, false, kInstr>(main, a, b);
    else tc::mma_f16<S::kCtas, true, kInstr>(main, a + k * kA, b + k * kB);
  }
  if (S::kPlanesB == 2) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (FRESH && S::kCross && k == 0) tc::mma_f16<S::kCtas, false, kInstr>(cross, a, b + kLoB);
      else tc::mma_f16<S::kCtas, true, kInstr>(cross, a + k * kA, b + kLoB + k * kB);
    }
  }
  if (S::kPlanesA == 2) {
#pragma unroll
    for (int k = 0; k < 4; ++k) tc::mma_f16<S::kCtas, true, kInstr>(cross, a + kLoA + k * kA, b + k * kB);
  }
}

// Eight values as hi + lo, two at a time (the packed conversions run at several
// times the rate of single ones).
__device__ __forceinline__ void split8(const float *v, uint4 &hi, uint4 &lo) {
  uint32_t *h = &hi.x, *l = &lo.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 a = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    const float2 f = __half22float2(a);
    const __half2 b = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
    h[i] = *reinterpret_cast<const uint32_t *>(&a);
    l[i] = *reinterpret_cast<const uint32_t *>(&b);
  }
}

__device__ __forceinline__ void add8(const uint4 &q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    v[2 * i] += f.x;
    v[2 * i + 1] += f.y;
  }
}

// 32 rows x 64 columns of a block, 4 KB of its image: between global memory,
// where the warp moves 512 adjacent bytes at a time, and registers, where
// thread l holds row l's 16-byte chunks in the order of its columns. `turn` is
// the warp's 4 KB of shared memory; both of its access patterns are free of bank
// conflicts (the swizzle). Accesses by row straight to global memory touch 32
// lines each: they took 9 us of a 256 x 256 tile per direction.
__device__ __forceinline__ void load_image(const char *at, char *turn, uint4 (&q)[8]) {
  const int lane = (int)lane_id();
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = *reinterpret_cast<const uint4 *>(at + e * 512 + lane * 16);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4 *>(turn + e * 512 + lane * 16) = q[e];
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = *reinterpret_cast<const uint4 *>(turn + chunk_at(lane, 8 * e));
}
__device__ __forceinline__ void store_image(char *at, char *turn, const uint4 (&q)[8]) {
  const int lane = (int)lane_id();
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4 *>(turn + chunk_at(lane, 8 * e)) = q[e];
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 8; ++e)
    *reinterpret_cast<uint4 *>(at + e * 512 + lane * 16) = *reinterpret_cast<const uint4 *>(turn + e * 512 + lane * 16);
}

__device__ __forceinline__ void store_as(void *p, int type, int64_t at, float v) {
  if (type == GS_TYPE_F32) reinterpret_cast<float *>(p)[at] = v;
  else if (type == GS_TYPE_BF16) reinterpret_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half *>(p)[at] = __float2half_rn(v);
}

// 32 rows x 32 columns of the result, thread l holding row `row` (+ l) from
// column `col` on. A tall result is X's transpose: the warp's rows are adjacent
// there. Otherwise the warp turns them in shared memory, so that its threads
// write adjacent columns.
__device__ __forceinline__ void store_result(const Out &o, int batch, int row, int col,
                                             const float (&w)[32], float (*turn)[33]) {
  const int lane = (int)lane_id();
  const int64_t base = (int64_t)batch * o.batch_stride;
  if (!o.tall) {
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 32; ++e) turn[lane][e] = w[e];
    __syncwarp();
  }
  // entry e of this thread: (row + lane, col + e), or turned (row + e, col + lane)
  const int limit = o.tall ? o.cols - col : o.rows - row;
  const bool on = o.tall ? row + lane < o.rows : col + lane < o.cols;
  const int64_t first = base + (o.tall ? (int64_t)col * o.rows + row + lane
                                       : (int64_t)row * o.cols + col + lane);
  const int64_t step = o.tall ? o.rows : o.cols;
  if (!on) return;
#pragma unroll
  for (int e0 = 0; e0 < 32; e0 += 8) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = o.tall ? w[e0 + e] : turn[e0 + e][lane];
    if (o.update) {
      float *p = reinterpret_cast<float *>(o.p);
      float old[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) old[e] = e0 + e < limit ? p[first + (e0 + e) * step] : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e0 + e < limit) p[first + (e0 + e) * step] = fmaf(o.decay, old[e], -o.step * v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e0 + e < limit) store_as(o.p, o.type, first + (e0 + e) * step, v[e]);
    }
  }
}

template <int BN, int KIND, bool FULL, int CTAS>
struct Shape {
  static constexpr int kBN = BN, kCtas = CTAS;
  static constexpr int kPlanesA = FULL ? 2 : 1;
  static constexpr int kPlanesB = FULL || KIND == kApply ? 2 : 1;
  static constexpr int kRowsB = BN / CTAS;                 // of B's rows in each block
  static constexpr int kPlaneA = 128 * 128, kPlaneB = kRowsB * 128;  // bytes
  static constexpr int kStage = kPlanesA * kPlaneA + kPlanesB * kPlaneB;
  static constexpr int kTri = BN > 128 * CTAS ? BN : 128 * CTAS;
  static constexpr int kChunk = FULL ? 4 : 128;            // K blocks of an accumulator
  // Where there is room, hi lo + lo hi have an accumulator of their own: far
  // fewer cut-off additions to the large one (128 x 64 in fp32: the result's
  // error 2.3e-6 -> 1.2e-6, as fp32 products have).
  static constexpr bool kCross = FULL && BN <= 128;
  static constexpr int kWidth = kCross ? 2 * BN : BN;      // columns of tensor memory
  static constexpr int kColumns = 2 * kWidth;              // two accumulators take turns
  // A copy warp, an MMA warp and the epilogue, whose warps hold 32 rows x 64
  // (128) columns each. Where the registers of 64 such sums and more would not
  // go round, a whole warpgroup goes to the first two, so that it can hand its
  // own over: 384 threads x 168 = 128 x 40 + 256 x 232.
  static constexpr int kEpilogueWarps = BN == 64 ? 4 : 8;
  static constexpr int kHeld = BN * 4 / kEpilogueWarps;    // columns of an epilogue warp
  static constexpr bool kHandOver = BN >= 128;
  static constexpr int kEpilogue = kHandOver ? 4 : 2;      // its first warp
  static constexpr int kThreads = 32 * (kEpilogue + kEpilogueWarps);
  static constexpr int kTurn = kEpilogueWarps * 32 * 33 * 4;
};

// Tiles of 128 CTAS x BN, one after another in a persistent block (or pair of
// blocks): while the epilogue works on a tile, the next one's products run
// into the other accumulator.
template <int BN, int KIND, bool FULL, int CTAS>
__global__ void __launch_bounds__(Shape<BN, KIND, FULL, CTAS>::kThreads, 1)
    product_kernel(const __grid_constant__ Args A) {
  using S = Shape<BN, KIND, FULL, CTAS>;
  extern __shared__ char raw[];
  char *smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
  __shared__ uint64_t full[kMaxStages], peer[kMaxStages], empty[kMaxStages], ready[2], drained[2];
  __shared__ uint32_t tmem_base, failed;
  const int warp = threadIdx.x / 32;
  const int rank = CTAS == 2 ? (int)cluster_rank() : 0;
  const int k_blocks = KIND == kGram ? A.k_blocks_n : A.k_blocks_m;
  const int chunks = (k_blocks + S::kChunk - 1) / S::kChunk;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS, total = A.tiles * A.batches;
  if (threadIdx.x == 0) {
    for (int s = 0; s < A.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&peer[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ready[s], 1);
      mbar_init(&drained[s], S::kEpilogueWarps * CTAS);
    }
    failed = 0;
    fence_mbar_init();
  }
  if (warp == 1) tc::tmem_alloc<CTAS>(&tmem_base, S::kColumns);
  tc::fence_before();
  __syncthreads();
  if (CTAS == 2) cluster_sync();
  tc::fence_after();
  const uint32_t tmem = tmem_base;
  start_next();
  wait_for_previous();
  asm volatile("fence.proxy.async.global;" ::: "memory");  // the bulk copies read what it wrote
  // Tile t: its matrix, row of tiles and column of tiles.
  struct Spot {
    int batch, i, j;
  };
  const auto spot = [&](int t) {
    Spot p;
    p.batch = t / A.tiles;
    int left = t % A.tiles;
    if (KIND == kApply) {
      p.i = left % A.row_tiles;
      p.j = left / A.row_tiles;
    } else {  // column j of tiles holds the rows down to its diagonal block
      int rows;
      for (p.j = 0;; ++p.j) {
        rows = (p.j * BN / S::kTri + 1) * (S::kTri / (128 * CTAS));
        if (left < rows) break;
        left -= rows;
      }
      p.i = left;
    }
    return p;
  };
  // Whether a K block of a symmetric matrix lies below the diagonal of rows.
  const auto below = [&](int row, int kb) { return KIND != kGram && kb * 64 / S::kTri < row / S::kTri; };

  if (S::kHandOver && warp < S::kEpilogue) tc::registers_down<40>();
  if (warp == 0) {
    if (tc::elect_one()) {
      const Matrix &MA = KIND == kGram ? A.x : KIND == kSquare ? A.sq : A.poly;
      const Matrix &MB = KIND == kSquare ? A.sq : A.x;
      int s = 0, used = 0;
      uint32_t phase = 1;  // of the slot's last reader; the first round has none
      bool good = true;
      for (int t = first; t < total && good; t += step) {
        const Spot p = spot(t);
        const int row_a = (p.i * CTAS + rank) * 128, row_b = p.j * BN + rank * S::kRowsB;
        for (int kb = 0; kb < k_blocks; ++kb) {
          good = used < A.stages || mbar_wait(&empty[s], phase);
          if (!good) break;
          char *a = smem + (size_t)s * S::kStage, *b = a + S::kPlanesA * S::kPlaneA;
          mbar_expect_tx(&full[s], S::kStage);
#pragma unroll
          for (int q = 0; q < S::kPlanesA; ++q)
            fetch_rows(q ? MA.lo : MA.hi, MA, p.batch, row_a, 128, kb, below(row_a, kb),
                       a + q * S::kPlaneA, &full[s]);
#pragma unroll
          for (int q = 0; q < S::kPlanesB; ++q)
            fetch_rows(q ? MB.lo : MB.hi, MB, p.batch, row_b, S::kRowsB, kb,
                       KIND == kApply || (KIND == kSquare && below(p.j * BN, kb)),
                       b + q * S::kPlaneB, &full[s]);
          ++used;
          if (++s == A.stages) s = 0, phase ^= 1;
        }
      }
      if (!good) {  // given up: the copies in flight still land here
        failed = 1;
        for (int q = used > A.stages ? used - A.stages : 0; q < used; ++q)
          mbar_wait(&full[q % A.stages], (q / A.stages) & 1);
      }
    }
  } else if (warp == 1 && rank == 1) {
    if (tc::elect_one()) {  // tells block 0 what has arrived here
      int s = 0;
      uint32_t phase = 0;
      bool good = true;
      for (int t = first; t < total && good; t += step)
        for (int kb = 0; kb < k_blocks && good; ++kb) {
          good = mbar_wait(&full[s], phase);
          if (good) tc::arrive_at(&peer[s], 0);
          if (++s == A.stages) s = 0, phase ^= 1;
        }
      if (!good) failed = 1;
    }
  } else if (warp == 1) {
    if (tc::elect_one()) {
      int s = 0, chunk = 0;
      uint32_t phase = 0;
      bool good = true;
      for (int t = first; t < total && good; t += step) {
        const Spot p = spot(t);
        int left = 0;  // K blocks to go in this accumulator
        for (int kb = 0; kb < k_blocks; ++kb) {
          const int acc = chunk & 1;
          const bool fresh = left == 0;
          if (fresh) left = k_blocks - kb < S::kChunk ? k_blocks - kb : S::kChunk;
          good = (!fresh || chunk < 2 || tc::wait_cluster(&drained[acc], (chunk / 2 - 1) & 1)) &&
                 mbar_wait(&full[s], phase) && (CTAS == 1 || tc::wait_cluster(&peer[s], phase));
          if (!good) break;
          tc::fence_after();
          const uint32_t at = smem_addr(smem) + s * S::kStage;
          const bool a_mn = below(p.i * CTAS * 128, kb);
          const bool b_mn = KIND == kApply || (KIND == kSquare && below(p.j * BN, kb));
          const uint32_t main = tmem + acc * S::kWidth, cross = S::kCross ? main + BN : main;
          const auto issue = [&](auto a_is_mn, auto b_is_mn) {
            if (fresh) issue_block<S, decltype(a_is_mn)::value, decltype(b_is_mn)::value, true>(at, main, cross);
            else issue_block<S, decltype(a_is_mn)::value, decltype(b_is_mn)::value, false>(at, main, cross);
          };
          using Yes = std::true_type;
          using No = std::false_type;
          if (KIND == kGram) issue(No(), No());
          else if (KIND == kApply && a_mn) issue(Yes(), Yes());
          else if (KIND == kApply) issue(No(), Yes());
          else if (a_mn && b_mn) issue(Yes(), Yes());
          else if (a_mn) issue(Yes(), No());
          else if (b_mn) issue(No(), Yes());
          else issue(No(), No());
          tc::commit<CTAS>(&empty[s]);
          if (--left == 0) {
            tc::commit<CTAS>(&ready[acc]);
            ++chunk;
          }
          if (++s == A.stages) s = 0, phase ^= 1;
        }
      }
      if (!good) failed = 1;
    }
  } else if (warp >= S::kEpilogue) {
    if (S::kHandOver) tc::registers_up<232>();
    const int quarter = warp & 3;  // the lanes of tensor memory that the warp may read
    const int c0 = (warp - S::kEpilogue) / 4 * S::kHeld;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + c0;
    char *turn = smem + (size_t)A.stages * S::kStage + (warp - S::kEpilogue) * (32 * 33 * 4);
    const Matrix &dst = KIND == kGram ? A.sq : KIND == kSquare ? A.poly : A.y;
    const Matrix &old = KIND == kSquare ? A.sq : A.x;
    constexpr bool kLo = FULL || KIND == kApply;  // of the old and the new values
    // The old values of one block are on their way before the products are done.
    constexpr bool kAhead = KIND != kGram && S::kHeld == 64;
    int chunk = 0;
    bool good = true;
    for (int t = first; t < total && good; t += step) {
      const Spot p = spot(t);
      const int i = p.i * CTAS + rank;  // the block's rows: 128 i..
      const auto image = [&](char *plane, const Matrix &M, int c) {
        return block_at(plane, M, p.batch, i, (p.j * BN + c0 + c) / 64) + quarter * 4096;
      };
      uint4 hi[8], lo[8];
      if (kAhead) {
        load_image(image(old.hi, old, 0), turn, hi);
        if (kLo) load_image(image(old.lo, old, 0), turn, lo);
      }
      float v[S::kHeld];
#pragma unroll
      for (int e = 0; e < S::kHeld; ++e) v[e] = 0.f;
#pragma unroll 1
      for (int part = 0; part < chunks; ++part, ++chunk) {
        const int acc = chunk & 1;
        good = __all_sync(0xffffffffu, mbar_wait(&ready[acc], (chunk / 2) & 1));
        if (!good) break;
        tc::fence_after();
#pragma unroll
        for (int c = 0; c < S::kHeld; c += 32) {
          float f[32];
          tc::load_columns(lanes + acc * S::kWidth + c, f);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[c + e] += f[e];
          if (S::kCross) {
            tc::load_columns(lanes + acc * S::kWidth + BN + c, f);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[c + e] += f[e];
          }
        }
        tc::fence_before();
        __syncwarp();
        if (lane_id() == 0) {
          if (CTAS == 2) tc::arrive_at(&drained[acc], 0);
          else tc::arrive(&drained[acc]);
        }
      }
      if (!good) break;
      // One lane reads, so that the warp stays together.
      if (A.out.update && __shfl_sync(0xffffffffu, lane_id() == 0 ? ld_volatile_u32(A.gate) : 0u, 0) != 0u) continue;
#pragma unroll
      for (int c = 0; c < S::kHeld; c += 64) {
        if (KIND != kGram && !kAhead) {
          load_image(image(old.hi, old, c), turn, hi);
          if (kLo) load_image(image(old.lo, old, c), turn, lo);
        }
        const float f = KIND == kSquare ? A.b : A.a, h = KIND == kSquare ? A.c * kUnscale : kUnscale;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          float o[8] = {};
          if (KIND != kGram) {
            add8(hi[g], o);
            if (kLo) add8(lo[g], o);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float &x = v[c + 8 * g + e];
            x = KIND == kGram ? x * kUnscale : fmaf(f, o[e], h * x);
          }
        }
        if (KIND == kApply && A.out.p != nullptr) {
#pragma unroll
          for (int g = 0; g < 64; g += 32) {
            float w[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = v[c + g + e] * kUnscale;
            store_result(A.out, p.batch, i * 128 + quarter * 32, p.j * BN + c0 + c + g, w,
                         reinterpret_cast<float(*)[33]>(turn));
          }
        } else {
#pragma unroll
          for (int g = 0; g < 8; ++g) split8(v + c + 8 * g, hi[g], lo[g]);
          store_image(image(dst.hi, dst, c), turn, hi);
          if (kLo) store_image(image(dst.lo, dst, c), turn, lo);
        }
      }
    }
    if (!good) failed = 1;
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  if (CTAS == 2) cluster_sync();  // neither block leaves while the other may reach into it
  if (threadIdx.x == 0 && failed) report_timeout(A.status, A.gate);
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_free<CTAS>(tmem, S::kColumns);
  }
}

// ---- the update: what is orthogonalised -------------------------------------------

struct Source {
  const void *u;          // the update, or the gradient that feeds the momentum
  int type;
  int64_t batch_stride, row_stride, col_stride;  // of X's rows and columns
  float *momentum;        // contiguous like the gradient; null: u is the update
  float beta, fresh;      // fresh = 1 - beta, from 64 bits
  int nesterov;
  int rows, cols;         // of X
};

__device__ __forceinline__ float read_f32(const void *p, int type, int64_t at) {
  return type == GS_TYPE_F32 ? reinterpret_cast<const float *>(p)[at]
         : type == GS_TYPE_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[at])
                                : __half2float(reinterpret_cast<const __half *>(p)[at]);
}

// M = beta M + (1 - beta) G and what of it is orthogonalised, rounded alike in
// both kernels that need it.
__device__ __forceinline__ float next_momentum(const Source &s, float m, float g) {
  return fmaf(s.beta, m, s.fresh * g);
}
__device__ __forceinline__ float update_of(const Source &s, float m_new, float g) {
  return s.nesterov ? fmaf(s.beta, m_new, s.fresh * g) : m_new;
}

// Eight adjacent elements, in 16-byte loads (the caller knows that they fit).
__device__ __forceinline__ void read8(const void *p, int type, int64_t at, float (&v)[8]) {
  if (type == GS_TYPE_F32) {
    const float4 *q = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + at);
    const float4 a = q[0], b = q[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 q = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p) + at);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t h = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
      v[e] = type == GS_TYPE_BF16 ? __bfloat162float(__ushort_as_bfloat16(h)) : __half2float(__ushort_as_half(h));
    }
  }
}
// Whether rows of 8 adjacent elements can be read so everywhere.
__device__ __forceinline__ bool vector_rows(const Source &s, int64_t stride) {
  const int each = s.type == GS_TYPE_F32 ? 4 : 8;
  return (((uintptr_t)s.u | (uintptr_t)s.momentum) & 15) == 0 && stride % each == 0 &&
         s.batch_stride % each == 0 && (s.momentum == nullptr || (stride % 4 == 0 && s.batch_stride % 4 == 0));
}

// The sum of 8 squares: in fp32 where neither the largest nor what matters next
// to it can leave the range, else in 64 bits.
__device__ __forceinline__ double squares(const float (&v)[8]) {
  float most = 0.f, sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    most = fmaxf(most, fabsf(v[e]));
    sum = fmaf(v[e], v[e], sum);
  }
  if (most > 1e-14f && most < 1e14f) return (double)sum;
  double wide = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) wide = fma((double)v[e], (double)v[e], wide);
  return wide;
}

// 2^12 / max(norm, eps), applied in fp32 where it is a normal number.
struct Scale {
  double wide;
  float narrow;
  bool fits;
  __device__ __forceinline__ Scale(double sum_of_squares, double eps) {
    const double norm = sqrt(sum_of_squares);
    wide = (double)kScale / (norm < eps ? eps : norm);
    narrow = (float)wide;
    fits = wide > 1e-30 && wide < 1e30;
  }
  __device__ __forceinline__ float operator()(float v) const {
    return fits ? v * narrow : (float)((double)v * wide);
  }
};

constexpr int kNormThreads = 256, kMaxParts = 296;

// Sums of squares, in 64 bits so that neither tiny nor huge gradients leave
// the range; the momentum is updated on the way. A matrix in one
// piece is read in 16-byte loads, others a line at a time along the smaller
// stride. Parts are added in order by the reader.
__global__ void __launch_bounds__(kNormThreads) norm_kernel(const Source s, double *parts, const uint32_t *gate) {
  start_next();
  wait_for_previous();
  if (gate != nullptr && *gate != 0u) return;
  const int64_t base = (int64_t)blockIdx.y * s.batch_stride;
  const bool cols_fast = s.col_stride <= s.row_stride;
  const int64_t lines = cols_fast ? s.rows : s.cols, len = cols_fast ? s.cols : s.rows;
  const int64_t fs = cols_fast ? s.col_stride : s.row_stride, ss = cols_fast ? s.row_stride : s.col_stride;
  const int64_t size = (int64_t)s.rows * s.cols;
  const int64_t warp = (int64_t)blockIdx.x * (kNormThreads / 32) + threadIdx.x / 32;
  const int64_t warps_all = (int64_t)gridDim.x * (kNormThreads / 32);
  double sum = 0.0;
  const auto take = [&](int64_t at, float v, float m) {
    if (s.momentum != nullptr) {
      m = next_momentum(s, m, v);
      s.momentum[at] = m;
      v = update_of(s, m, v);
    }
    sum = fma((double)v, (double)v, sum);
  };
  if (fs == 1 && ss == len && vector_rows(s, 8)) {  // one piece of memory
    for (int64_t k = warp * 1024; k < size; k += warps_all * 1024) {
      float v[4][8], m[4][8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t at = k + q * 256 + lane_id() * 8;
        if (at + 8 <= size) {
          read8(s.u, s.type, base + at, v[q]);
          if (s.momentum != nullptr) read8(s.momentum, GS_TYPE_F32, base + at, m[q]);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t at = k + q * 256 + lane_id() * 8;
        if (at + 8 <= size) {
          if (s.momentum != nullptr) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              m[q][e] = next_momentum(s, m[q][e], v[q][e]);
              v[q][e] = update_of(s, m[q][e], v[q][e]);
            }
            float4 *to = reinterpret_cast<float4 *>(s.momentum + base + at);
            to[0] = make_float4(m[q][0], m[q][1], m[q][2], m[q][3]);
            to[1] = make_float4(m[q][4], m[q][5], m[q][6], m[q][7]);
          }
          sum += squares(v[q]);
        } else {
          for (int64_t f = at; f < size; ++f)
            take(base + f, read_f32(s.u, s.type, base + f), s.momentum != nullptr ? s.momentum[base + f] : 0.f);
        }
      }
    }
  } else {
    for (int64_t k = warp; k < lines; k += warps_all)
#pragma unroll 4
      for (int64_t f = lane_id(); f < len; f += 32) {
        const int64_t at = base + k * ss + f * fs;
        take(at, read_f32(s.u, s.type, at), s.momentum != nullptr ? s.momentum[at] : 0.f);
      }
  }
  __shared__ double warps[kNormThreads / 32];
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_down_sync(0xffffffffu, sum, d);
  if (lane_id() == 0) warps[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kNormThreads / 32; ++w) sum += warps[w];
    parts[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = sum;
  }
}

// X0, 64 x 64 elements a block, scaled and split into the workspace's layout.
// Rows of adjacent elements go straight into their chunks, others are turned
// in shared memory.
__global__ void __launch_bounds__(256) split_kernel(const Source s, const double *parts, int num_parts,
                                                    double eps, Matrix x) {
  __shared__ float tile[64][65];
  __shared__ double total;  // sum of squares
  start_next();
  wait_for_previous();
  const int batch = blockIdx.y, r0 = blockIdx.x / x.column_blocks * 64, c0 = blockIdx.x % x.column_blocks * 64;
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < num_parts; k += 32) sum += parts[(int64_t)batch * num_parts + k];
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_down_sync(0xffffffffu, sum, d);
    if (threadIdx.x == 0) total = sum;
  }
  __syncthreads();
  const Scale scale(total, eps);
  const int64_t base = (int64_t)batch * s.batch_stride;
  const auto read = [&](int r, int c) {
    if (r0 + r >= s.rows || c0 + c >= s.cols) return 0.f;
    const int64_t at = base + (r0 + r) * s.row_stride + (c0 + c) * s.col_stride;
    float v = read_f32(s.u, s.type, at);
    if (s.momentum != nullptr) v = update_of(s, s.momentum[at], v);
    return scale(v);
  };
  const bool cols_fast = s.col_stride <= s.row_stride;
  const bool wide = s.col_stride == 1 && vector_rows(s, s.row_stride);
  if (!cols_fast) {
#pragma unroll 4
    for (int k = threadIdx.x; k < 64 * 64; k += 256) tile[k % 64][k / 64] = read(k % 64, k / 64);
    __syncthreads();
  }
#pragma unroll
  for (int k = threadIdx.x; k < 64 * 8; k += 256) {
    const int r = k / 8, c = k % 8 * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (!cols_fast) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = tile[r][c + e];
    } else if (wide && r0 + r < s.rows && c0 + c + 8 <= s.cols) {
      const int64_t at = base + (r0 + r) * s.row_stride + c0 + c;
      read8(s.u, s.type, at, v);
      float m[8];
      if (s.momentum != nullptr) read8(s.momentum, GS_TYPE_F32, at, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (s.momentum != nullptr) v[e] = update_of(s, m[e], v[e]);
        v[e] = scale(v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = read(r, c + e);
    }
    uint4 hi, lo;
    split8(v, hi, lo);
    const int at = chunk_at((r0 + r) % 128, c);
    *reinterpret_cast<uint4 *>(block_at(x.hi, x, batch, (r0 + r) / 128, c0 / 64) + at) = hi;
    *reinterpret_cast<uint4 *>(block_at(x.lo, x, batch, (r0 + r) / 128, c0 / 64) + at) = lo;
  }
}

// ---- small matrices -----------------------------------------------------------------
//
// Up to 128 rows, a matrix stays on chip for the whole call: a block (or a
// cluster of C blocks, NC columns each) keeps its columns of X and the whole of
// A in shared memory, in the same block images, and runs norm, steps and result
// in one launch. A launch for each product took 5 to 6 us each, 17 of them.
// In a cluster every block forms the part of A = X X^T that its columns give;
// block k adds the parts of its MC / C rows in the blocks' order, and every block
// fetches all of A. Both go through global memory (L2), between cluster barriers:
// through the blocks' shared memory they took 8 us a step, 5 here. B = b A +
// c A A is cheap enough to be formed by each block.
constexpr int kSmallThreads = 512;  // four warps for each quarter of tensor memory's lanes

struct SmallArgs {
  Source src;
  Out out;
  int cluster, steps;
  float a, b, c;
  double eps;
  char *shared;  // of a matrix's blocks: their parts of A, then A's planes
  uint32_t *status, *gate;
};

// X has up to MC rows. The MMAs' M is 128: what their rows beyond MC hold is
// neither set nor looked at.
template <int MC, int NC>
struct SmallShape {
  static constexpr int kBlocks = NC / 64;
  static constexpr int kX = kBlocks * kBlockBytes;          // a plane of X
  static constexpr int kSq = MC / 64 * kBlockBytes;         // a plane of A or B
  static constexpr int kTurn = kSmallThreads / 32 * 32 * 33 * 4;  // in place of A, and behind
  static constexpr int kRest = 2 * kSq > kTurn ? 2 * kSq : kTurn;
  static constexpr int kBytes = 2 * kX + kRest;
  static constexpr int kTop = NC > MC ? NC : MC;            // columns of an accumulator
};

// What a matrix's blocks share in global memory: their parts of A, A's planes.
__host__ __device__ constexpr int64_t shared_bytes(int mc, int cluster) {
  return cluster == 1 ? 0 : (int64_t)cluster * mc * mc * 4 + 2 * (mc / 64) * kBlockBytes;
}

// All MMAs of D = P Q^T (or P Q, Q's rows along K) over `blocks` K blocks:
// hi hi into main, hi lo + lo hi into cross.
template <int N, bool Q_MN>
__device__ __forceinline__ void small_product(uint32_t main, uint32_t cross, uint32_t p, uint32_t p_lo,
                                              uint32_t q, uint32_t q_lo, int blocks) {
  constexpr uint32_t kInstr = tc::instruction_f16(128, N, false, Q_MN);
  // K-major: a block of 64 K per image, 16 of them 32 bytes further. MN-major:
  // 16 rows of 128 bytes, images 64 columns apart.
  const auto q_at = [&](uint32_t base, int kb, int k) {
    return Q_MN ? tc::descriptor(base + (kb * 4 + k) * 2048, kBlockBytes, 1024)
                : tc::descriptor(base + kb * kBlockBytes + k * 32, 16, 1024);
  };
  for (int kb = 0; kb < blocks; ++kb) {
    const bool fresh = kb == 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t a = tc::descriptor(p + kb * kBlockBytes + k * 32, 16, 1024);
      if (fresh && k == 0) tc::mma_f16<1, false, kInstr>(main, a, q_at(q, kb, k));
      else tc::mma_f16<1, true, kInstr>(main, a, q_at(q, kb, k));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint64_t a = tc::descriptor(p + kb * kBlockBytes + k * 32, 16, 1024);
      if (fresh && k == 0) tc::mma_f16<1, false, kInstr>(cross, a, q_at(q_lo, kb, k));
      else tc::mma_f16<1, true, kInstr>(cross, a, q_at(q_lo, kb, k));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      tc::mma_f16<1, true, kInstr>(cross, tc::descriptor(p_lo + kb * kBlockBytes + k * 32, 16, 1024),
                                   q_at(q, kb, k));
  }
}

template <int MC, int NC>
__global__ void __launch_bounds__(kSmallThreads, 1) small_kernel(const __grid_constant__ SmallArgs A) {
  using S = SmallShape<MC, NC>;
  extern __shared__ char raw[];
  char *x_hi = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023), *x_lo = x_hi + S::kX;
  char *sq_hi = x_lo + S::kX, *sq_lo = sq_hi + S::kSq;
  __shared__ uint64_t done;
  __shared__ uint32_t tmem_base, failed;
  __shared__ double warp_sums[kSmallThreads / 32], block_sum;
  const int warp = threadIdx.x / 32, lane = (int)lane_id();
  const int C = A.cluster, rank = C > 1 ? (int)cluster_rank() : 0, batch = blockIdx.x / C;
  const int col_base = rank * NC;  // of X
  const Source &s = A.src;
  if (threadIdx.x == 0) {
    mbar_init(&done, 1);
    failed = 0;
    fence_mbar_init();
  }
  if (warp == 0) tc::tmem_alloc<1>(&tmem_base, 2 * S::kTop);
  // Skipped optimizer steps run through, so that the blocks of a cluster stay
  // together, and write nothing.
  wait_for_previous();
  bool skip = A.gate != nullptr && *A.gate != 0u;

  // The update, 8 columns of a row at a time, and its sum of squares.
  constexpr int kEach = MC * NC / 8 / kSmallThreads;
  const bool cols_fast = s.col_stride <= s.row_stride;
  const bool wide = s.col_stride == 1 && vector_rows(s, s.row_stride);
  const int64_t base = (int64_t)batch * s.batch_stride;
  float u[kEach][8];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = k * kSmallThreads + threadIdx.x;
    const int r = cols_fast ? at / (NC / 8) : at % MC, c = (cols_fast ? at % (NC / 8) : at / MC) * 8;
    const int col = col_base + c;
    const int64_t from = base + r * s.row_stride + col * s.col_stride;
    if (wide && r < s.rows && col + 8 <= s.cols) {
      read8(s.u, s.type, from, u[k]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        u[k][e] = r < s.rows && col + e < s.cols ? read_f32(s.u, s.type, from + e * s.col_stride) : 0.f;
    }
  }
  if (s.momentum != nullptr) {
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int at = k * kSmallThreads + threadIdx.x;
      const int r = cols_fast ? at / (NC / 8) : at % MC, c = (cols_fast ? at % (NC / 8) : at / MC) * 8;
      const int col = col_base + c;
      const int64_t from = base + r * s.row_stride + col * s.col_stride;
      float m[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        m[e] = r < s.rows && col + e < s.cols ? s.momentum[from + e * s.col_stride] : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = next_momentum(s, m[e], u[k][e]);
        if (!skip && r < s.rows && col + e < s.cols) s.momentum[from + e * s.col_stride] = m[e];
        u[k][e] = update_of(s, m[e], u[k][e]);
      }
    }
  }
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kEach; ++k) sum += squares(u[k]);
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_down_sync(0xffffffffu, sum, d);
  if (lane == 0) warp_sums[warp] = sum;
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSmallThreads / 32; ++w) sum += warp_sums[w];
    block_sum = sum;
  }
  double total = 0.0;
  if (C > 1) {
    cluster_sync();
    for (int k = 0; k < C; ++k) total += cluster_load_f64(cluster_addr(&block_sum, k));
  } else {
    __syncthreads();
    total = block_sum;
  }
  const Scale scale(total, A.eps);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = k * kSmallThreads + threadIdx.x;
    const int r = cols_fast ? at / (NC / 8) : at % MC, c = (cols_fast ? at % (NC / 8) : at / MC) * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = scale(u[k][e]);
    uint4 hi, lo;
    split8(v, hi, lo);
    const int to = c / 64 * kBlockBytes + chunk_at(r, c);
    *reinterpret_cast<uint4 *>(x_hi + to) = hi;
    *reinterpret_cast<uint4 *>(x_lo + to) = lo;
  }
  float *part = reinterpret_cast<float *>(A.shared + (int64_t)batch * shared_bytes(MC, C));
  char *whole = reinterpret_cast<char *>(part + C * MC * MC);
  const uint32_t tmem = tmem_base, cross = tmem + S::kTop;
  const int quarter = warp & 3, group = warp / 4, r = quarter * 32 + lane;
  const bool on = quarter * 32 < MC;  // the warp's rows are X's
  const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
  uint32_t phase = 0;
  bool timed_out = false;
  const auto run = [&](auto issue) {  // what was written is read by the tensor core
    fence_proxy_async_smem();
    tc::fence_before();
    __syncthreads();
    if (warp == 0 && tc::elect_one()) {
      tc::fence_after();
      issue();
      tc::commit<1>(&done);
    }
    __syncwarp();
    if (!mbar_wait(&done, phase)) timed_out = true;
    phase ^= 1;
    __syncwarp();
    tc::fence_after();
  };
  // 32 columns of the product for this thread's row.
  const auto columns = [&](int c, float (&v)[32]) {
    tc::load_sum(tmem + lanes + c, cross + lanes + c, v);
  };
  // w = f old + g w for 8 columns, old from the image that the result replaces.
  const auto blend = [&](char *hi_at, char *lo_at, float f, float g, const float *v, float (&w)[8]) {
    float o[8] = {};
    add8(*reinterpret_cast<const uint4 *>(hi_at), o);
    add8(*reinterpret_cast<const uint4 *>(lo_at), o);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = fmaf(f, o[e], g * v[e]);
  };
  const auto put = [&](char *hi_at, char *lo_at, const float *w) {
    uint4 hi, lo;
    split8(w, hi, lo);
    *reinterpret_cast<uint4 *>(hi_at) = hi;
    *reinterpret_cast<uint4 *>(lo_at) = lo;
  };

  for (int step = 0; step < A.steps; ++step) {
    run([&] {
      small_product<MC, false>(tmem, cross, smem_addr(x_hi), smem_addr(x_lo), smem_addr(x_hi),
                               smem_addr(x_lo), S::kBlocks);
    });
    if (on && group * 32 < MC) {
      const int c = group * 32;
      float v[32];
      columns(c, v);
      if (C == 1) {
#pragma unroll
        for (int g = 0; g < 32; g += 8) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = v[g + e] * kUnscale;
          const int to = (c + g) / 64 * kBlockBytes + chunk_at(r, c + g);
          put(sq_hi + to, sq_lo + to, w);
        }
      } else {  // column by column, so that the warp writes adjacent rows
#pragma unroll
        for (int e = 0; e < 32; ++e) __stcg(part + rank * (MC * MC) + (c + e) * MC + r, v[e]);
      }
    }
    if (C > 1) {
      __threadfence();
      cluster_sync();
      // A is symmetric: its row `row` is what lies in column `row` of the parts.
      const int rows = MC / C;
      for (int k = threadIdx.x; k < rows * (MC / 8); k += kSmallThreads) {
        const int row = rank * rows + k / (MC / 8), c = k % (MC / 8) * 8;
        const float4 *from = reinterpret_cast<const float4 *>(part + row * MC + c);
        float4 f[8], g[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < C) {
            f[q] = __ldcg(from + q * (MC * MC / 4));
            g[q] = __ldcg(from + q * (MC * MC / 4) + 1);
          }
        float w[8] = {};
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < C) {
            w[0] += f[q].x, w[1] += f[q].y, w[2] += f[q].z, w[3] += f[q].w;
            w[4] += g[q].x, w[5] += g[q].y, w[6] += g[q].z, w[7] += g[q].w;
          }
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] *= kUnscale;
        uint4 hi, lo;
        split8(w, hi, lo);
        const int to = c / 64 * kBlockBytes + chunk_at(row, c);
        __stcg(reinterpret_cast<uint4 *>(whole + to), hi);
        __stcg(reinterpret_cast<uint4 *>(whole + S::kSq + to), lo);
      }
      __threadfence();
      __syncwarp();
      cluster_sync();
      // Rows beyond MC of the images are neither written nor read.
      constexpr int kCopies = 2 * MC / 64 * MC * 8 / kSmallThreads;
      uint4 q[kCopies];
      int at[kCopies];
#pragma unroll
      for (int k = 0; k < kCopies; ++k) {
        const int e = k * kSmallThreads + threadIdx.x;  // chunks of MC rows, image after image
        at[k] = e / (MC * 8) * kBlockBytes + e % (MC * 8) * 16;
        q[k] = __ldcg(reinterpret_cast<const uint4 *>(whole + at[k]));
      }
#pragma unroll
      for (int k = 0; k < kCopies; ++k) *reinterpret_cast<uint4 *>(sq_hi + at[k]) = q[k];
    }
    run([&] {
      small_product<MC, false>(tmem, cross, smem_addr(sq_hi), smem_addr(sq_lo), smem_addr(sq_hi),
                               smem_addr(sq_lo), MC / 64);
    });
    if (on && group * 32 < MC) {
      const int c = group * 32;
      float v[32];
      columns(c, v);
#pragma unroll
      for (int g = 0; g < 32; g += 8) {
        const int to = (c + g) / 64 * kBlockBytes + chunk_at(r, c + g);
        float w[8];
        blend(sq_hi + to, sq_lo + to, A.b, A.c * kUnscale, v + g, w);
        put(sq_hi + to, sq_lo + to, w);
      }
    }
    run([&] {
      small_product<NC, true>(tmem, cross, smem_addr(sq_hi), smem_addr(sq_lo), smem_addr(x_hi),
                              smem_addr(x_lo), MC / 64);
    });
    const bool last = step + 1 == A.steps;
    if (last) {  // whether a wait ran out, in any block of the matrix
      const int any = __syncthreads_or(timed_out);
      if (threadIdx.x == 0) failed = any;
      if (any) skip = true;
      if (C > 1 && A.gate != nullptr) {
        cluster_sync();
        if (__syncthreads_or((int)threadIdx.x < C ? (int)cluster_load_u32(cluster_addr(&failed, threadIdx.x)) : 0))
          skip = true;
      }
    }
    if (on) {
#pragma unroll 1
      for (int c = group * 32; c < NC; c += 128) {
        float v[32];
        columns(c, v);
#pragma unroll
        for (int g = 0; g < 32; g += 8) {
          const int to = (c + g) / 64 * kBlockBytes + chunk_at(r, c + g);
          float w[8];
          blend(x_hi + to, x_lo + to, A.a, kUnscale, v + g, w);
          if (!last) put(x_hi + to, x_lo + to, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[g + e] = w[e] * kUnscale;
        }
        if (last && !skip)  // B is done with: its place serves to turn the result
          store_result(A.out, batch, quarter * 32, col_base + c, v,
                       reinterpret_cast<float(*)[33]>(sq_hi + warp * (32 * 33 * 4)));
      }
    }
    __syncwarp();
  }
  tc::fence_before();
  __syncthreads();
  if (C > 1) cluster_sync();  // no block leaves while another may reach into it
  if (threadIdx.x == 0 && failed) report_timeout(A.status, A.gate);
  if (warp == 0) {
    tc::fence_after();
    tc::tmem_free<1>(tmem, 2 * S::kTop);
  }
}

// ---- host -----------------------------------------------------------------------------

constexpr size_t kGateBytes = 256;  // the gate, first in the scratch; what follows keeps its lines

struct Plan {
  int m, n, bn, ctas;       // X is m x n, tiles are 128 ctas x bn
  int row_blocks, column_blocks, sq_column_blocks;
  bool full;
  int parts;
  size_t x_bytes, sq_bytes, total;  // of a plane and of everything, all batches
};

// How a matrix of m <= 128 rows is cut for small_kernel: columns of a block (0:
// too wide for it) and blocks.
struct SmallPlan {
  int columns, cluster;
};
static SmallPlan small_plan(int m, int n) {
  if (m > 128 || n > 2048) return {0, 0};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {128, 1};
  if (n <= 256) return {256, 1};
  return {n <= 1024 ? 128 : 256, n <= 512 ? 4 : 8};
}

// What a step costs in tiles of 128 ctas x bn, in microseconds: each of its three
// products a constant for filling, draining and the launch, and rounds of tiles
// at so much a K block, both fitted to measurements between 256 x 256 and
// 4096 x 4096. Small tiles start and end sooner and fill the device with small
// matrices (512 x 512 fp32: 135 us a call in 128 x 64 tiles, 162 in pairs of
// 128 x 128, 260 in pairs of 128 x 256), large ones read less through the L2
// (4096 x 4096 bf16: 3.36, 2.01 and 1.54 ms). Full products gain nothing from the
// largest (4096 x 4096 fp32: 3.31 ms against 3.20 in pairs of 128 x 128, which
// also have room for the second accumulator).
struct TileShape {
  int bn, ctas;
  double fixed_full, block_full;              // fp32 and fp16 results
  double fixed_half, syrk_half, apply_half;   // bf16 results: A and A A, a X + B X
};
constexpr TileShape kShapes[] = {{64, 1, 5.0, 0.55, 4.1, 0.33, 0.38},
                                 {128, 1, 6.2, 0.75, 4.2, 0.40, 0.47},
                                 {128, 2, 6.4, 0.60, 4.9, 0.39, 0.45},
                                 {256, 2, 0.0, 0.0, 7.1, 0.48, 0.72}};  // half only

static double cost_of(int batch, int m, int n, bool full, const TileShape &t) {
  const int rows = 128 * t.ctas, tri = t.bn > rows ? t.bn : rows;
  const int64_t sq = (m + tri - 1) / tri, per = tri / rows;  // superblocks, rows of tiles in one
  const int64_t half = sq * (sq + 1) / 2 * per * (tri / t.bn);
  const int64_t whole = sq * per * ((n + t.bn - 1) / t.bn);
  const int kn = (n + 63) / 64, km = (m + 63) / 64;
  const auto product = [&](int64_t tiles, int k, double block) {
    const double rounds = (double)((tiles * batch * t.ctas + 147) / 148);
    return (full ? t.fixed_full : t.fixed_half) + rounds * (k * block + 1.0);
  };
  const double syrk = full ? t.block_full : t.syrk_half, apply = full ? t.block_full : t.apply_half;
  return product(half, kn, syrk) + product(half, km, syrk) + product(whole, km, apply);
}

static Plan make_plan(int batch, int rows, int cols, int type) {
  Plan p;
  p.m = rows < cols ? rows : cols;
  p.n = rows < cols ? cols : rows;
  p.full = type != GS_TYPE_BF16;
  double best = 0.0;
  p.bn = 0;
  for (const TileShape &t : kShapes) {
    if (p.full && t.bn == 256) continue;
    const double cost = cost_of(batch, p.m, p.n, p.full, t);
    if (p.bn == 0 || cost < best) best = cost, p.bn = t.bn, p.ctas = t.ctas;
  }
  const int tri = p.bn > 128 * p.ctas ? p.bn : 128 * p.ctas;
  const int mp = (p.m + tri - 1) / tri * tri, np = (p.n + p.bn - 1) / p.bn * p.bn;
  p.row_blocks = mp / 128;
  p.column_blocks = np / 64;
  p.sq_column_blocks = mp / 64;
  const int64_t size = (int64_t)rows * cols;
  const int64_t parts = (size + 8191) / 8192;
  p.parts = (int)(parts < kMaxParts ? parts : kMaxParts);
  p.x_bytes = (size_t)batch * p.row_blocks * p.column_blocks * kBlockBytes;
  p.sq_bytes = (size_t)batch * p.row_blocks * p.sq_column_blocks * kBlockBytes;
  p.total = kGateBytes + 4 * p.x_bytes + (p.full ? 4 : 2) * p.sq_bytes + (size_t)batch * p.parts * 8;
  const SmallPlan small = small_plan(p.m, p.n);
  if (small.columns) p.total = kGateBytes + (size_t)batch * shared_bytes(p.m <= 64 ? 64 : 128, small.cluster);
  return p;
}

template <int BN, int KIND, bool FULL, int CTAS>
static int launch_product(Args A, int tiles, int row_tiles, int batch, cudaStream_t st) {
  using S = Shape<BN, KIND, FULL, CTAS>;
  const auto kernel = product_kernel<BN, KIND, FULL, CTAS>;
  A.stages = (227 * 1024 - 2048 - S::kTurn) / S::kStage;
  if (A.stages > kMaxStages) A.stages = kMaxStages;
  A.tiles = tiles;
  A.row_tiles = row_tiles;
  A.batches = batch;
  const int bytes = A.stages * S::kStage + S::kTurn + 1024;
  // Per context: the kernel's shared memory and how many blocks run at a time.
  thread_local unsigned long long ready = 0;
  thread_local int resident = 0;
  const unsigned long long ctx = current_context_id();
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CTAS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1] = overlapping();
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  if (ctx == 0 || ctx != ready) {
    int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (rc) return rc;
    cfg.gridDim = dim3(CTAS);
    rc = cuda_status(cudaOccupancyMaxActiveClusters(&resident, kernel, &cfg));
    if (rc) return rc;
    if (resident < 1) return GS_ERR_CUDA;
    ready = ctx != 0 ? ctx : current_context_id();
  }
  const int64_t all = (int64_t)tiles * batch;
  cfg.gridDim = dim3((unsigned)(all < resident ? all : resident) * CTAS);
  const int rc = cuda_status(cudaLaunchKernelEx(&cfg, kernel, A));
  if (rc) return rc;
  count_launch();
  return GS_OK;
}

template <int BN, bool FULL, int CTAS>
static int run_steps(Args A, const Plan &p, int batch, int steps, const Out &out, cudaStream_t st) {
  int tri_tiles = 0;
  constexpr int kTri = BN > 128 * CTAS ? BN : 128 * CTAS;
  for (int j = 0; j < p.sq_column_blocks * 64 / BN; ++j)
    tri_tiles += (j * BN / kTri + 1) * (kTri / (128 * CTAS));
  const int row_tiles = p.row_blocks / CTAS;
  for (int k = 0; k < steps; ++k) {
    A.out = out;
    if (k + 1 < steps) A.out.p = nullptr, A.out.update = 0;
    int rc = launch_product<BN, kGram, FULL, CTAS>(A, tri_tiles, row_tiles, batch, st);
    if (!rc) rc = launch_product<BN, kSquare, FULL, CTAS>(A, tri_tiles, row_tiles, batch, st);
    if (!rc)
      rc = launch_product<BN, kApply, FULL, CTAS>(A, row_tiles * (p.column_blocks * 64 / BN), row_tiles, batch, st);
    if (rc) return rc;
    const Matrix x = A.x;
    A.x = A.y;
    A.y = x;
  }
  return GS_OK;
}

template <int MC, int NC>
static int launch_small(const SmallArgs &A, int batch, cudaStream_t st) {
  constexpr int kBytes = SmallShape<MC, NC>::kBytes + 1024;
  thread_local unsigned long long ready = 0;
  const unsigned long long ctx = current_context_id();
  if (ctx == 0 || ctx != ready) {
    const int rc = cuda_status(cudaFuncSetAttribute(small_kernel<MC, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes));
    if (rc) return rc;
    ready = ctx != 0 ? ctx : current_context_id();
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = A.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1] = overlapping();
  cfg.attrs = attr;
  cfg.numAttrs = A.gate != nullptr ? 2 : 1;
  cfg.gridDim = dim3(batch * A.cluster);
  cfg.blockDim = dim3(kSmallThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = st;
  const int rc = cuda_status(cudaLaunchKernelEx(&cfg, small_kernel<MC, NC>, A));
  if (rc) return rc;
  count_launch();
  return GS_OK;
}

// The largest |X|_2, |A|_2 and |b A + c A A|_2 that the steps can reach from
// |X|_2 <= 1, from the extremes of the two polynomials on [0, r]. X and B have
// to stay below 8 for the fp16 range, and A = X X^T, which each step starts
// with, below 15: 6% below the range's end, for the rounding of what led there.
constexpr double kMostA = 15.0;
static bool in_range(int steps, double a, double b, double c) {
  double r = 1.0;
  for (int k = 0; k < steps; ++k) {
    const auto p = [&](double s) { return fabs(s * (a + s * s * (b + s * s * c))); };
    const auto q = [&](double y) { return fabs(y * (b + y * c)); };
    if (!(r * r < kMostA)) return false;
    double most = p(r), poly = q(r * r);
    // p'(s) = a + 3 b s^2 + 5 c s^4
    const double disc = 9 * b * b - 20 * a * c;
    if (c != 0 && disc >= 0)
      for (int sign = -1; sign <= 1; sign += 2) {
        const double y = (-3 * b + sign * sqrt(disc)) / (10 * c);
        if (y > 0 && y < r * r) most = fmax(most, p(sqrt(y)));
      }
    else if (c == 0 && b != 0 && -a / (3 * b) > 0 && -a / (3 * b) < r * r)
      most = fmax(most, p(sqrt(-a / (3 * b))));
    if (c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < r * r) poly = fmax(poly, q(-b / (2 * c)));
    if (!(most < 8.0) || !(poly < 8.0)) return false;
    r = fmax(most, 1.0);
  }
  return true;
}

static int run(int batch, const Plan &p, const Source &src, const Out &out, int steps, float a, float b,
               float c, float eps, void *scratch, size_t scratch_bytes, cudaStream_t st) {
  if (scratch == nullptr || ((uintptr_t)scratch & 15)) return GS_ERR_INVALID_ARGUMENT;
  if (scratch_bytes < p.total) return GS_ERR_CAPACITY;
  if ((int64_t)p.row_blocks * p.column_blocks * batch > INT32_MAX / 2) return GS_ERR_CAPACITY;
  Args A{};
  A.status = device_status_word();
  if (A.status == nullptr) return GS_ERR_CUDA;
  char *at = static_cast<char *>(scratch) + kGateBytes;
  if (out.update) {
    A.gate = static_cast<uint32_t *>(scratch);
    gate_kernel<<<1, 1, 0, st>>>(A.status, A.gate);
    const int rc = launch_status();
    if (rc) return rc;
    count_launch();
  }
  const SmallPlan small = small_plan(p.m, p.n);
  if (small.columns) {
    const SmallArgs B{src, out, small.cluster, steps, a, b, c, (double)eps, at, A.status, A.gate};
    if (p.m <= 64)
      return small.columns == 64    ? launch_small<64, 64>(B, batch, st)
             : small.columns == 128 ? launch_small<64, 128>(B, batch, st)
                                    : launch_small<64, 256>(B, batch, st);
    return small.columns == 128 ? launch_small<128, 128>(B, batch, st) : launch_small<128, 256>(B, batch, st);
  }
  const auto take = [&](size_t n) {
    char *q = at;
    at += n;
    return q;
  };
  const int64_t xb = (int64_t)(p.x_bytes / batch), sb = (int64_t)(p.sq_bytes / batch);
  A.x = {take(p.x_bytes), take(p.x_bytes), xb, p.column_blocks};
  A.y = {take(p.x_bytes), take(p.x_bytes), xb, p.column_blocks};
  A.sq = {take(p.sq_bytes), p.full ? take(p.sq_bytes) : nullptr, sb, p.sq_column_blocks};
  A.poly = {take(p.sq_bytes), p.full ? take(p.sq_bytes) : nullptr, sb, p.sq_column_blocks};
  double *parts = reinterpret_cast<double *>(at);
  A.k_blocks_n = (p.n + 63) / 64;
  A.k_blocks_m = (p.m + 63) / 64;
  A.a = a;
  A.b = b;
  A.c = c;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr = overlapping();
  cfg.attrs = &attr;
  cfg.numAttrs = A.gate != nullptr ? 1 : 0;
  cfg.gridDim = dim3(p.parts, batch);
  cfg.blockDim = dim3(kNormThreads);
  cfg.stream = st;
  int rc = cuda_status(cudaLaunchKernelEx(&cfg, norm_kernel, src, parts, (const uint32_t *)A.gate));
  if (rc) return rc;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(p.row_blocks * 2 * p.column_blocks, batch);
  cfg.blockDim = dim3(256);
  rc = cuda_status(cudaLaunchKernelEx(&cfg, split_kernel, src, (const double *)parts, p.parts, (double)eps, A.x));
  if (rc) return rc;
  count_launch(2);
  if (p.full)
    return p.bn == 128 && p.ctas == 2 ? run_steps<128, true, 2>(A, p, batch, steps, out, st)
           : p.bn == 128 ? run_steps<128, true, 1>(A, p, batch, steps, out, st)
                         : run_steps<64, true, 1>(A, p, batch, steps, out, st);
  return p.bn == 256   ? run_steps<256, false, 2>(A, p, batch, steps, out, st)
         : p.bn == 128 && p.ctas == 2 ? run_steps<128, false, 2>(A, p, batch, steps, out, st)
         : p.bn == 128 ? run_steps<128, false, 1>(A, p, batch, steps, out, st)
                       : run_steps<64, false, 1>(A, p, batch, steps, out, st);
}

static bool known_type(int type) {
  return type == GS_TYPE_F32 || type == GS_TYPE_BF16 || type == GS_TYPE_F16;
}

static int check(int batch, int rows, int cols, int type, int steps, float a, float b, float c, float eps) {
  if (batch < 1 || batch > 65535 || rows < 1 || cols < 1 || rows > (1 << 24) || cols > (1 << 24) ||
      (rows < cols ? rows : cols) > (1 << 15) || !known_type(type) || steps < 1 || steps > 100 ||
      !(eps > 0.f) || !in_range(steps, a, b, c))
    return GS_ERR_INVALID_ARGUMENT;
  return GS_OK;
}

}  // namespace ns
}  // namespace gs

using namespace gs;
using namespace gs::ns;

extern "C" size_t gs_orthogonalize_scratch_bytes(int batch, int rows, int cols, int type) {
  if (check(batch, rows, cols, type, 1, 1.f, 0.f, 0.f, 1.f)) return 0;
  return make_plan(batch, rows, cols, type).total;
}

extern "C" int gs_orthogonalize(int batch, int rows, int cols, int type, const void *update,
                                int64_t batch_stride, int64_t row_stride, int64_t col_stride, void *out,
                                int steps, float a, float b, float c, float eps, void *scratch,
                                size_t scratch_bytes, void *stream) {
  const int rc = check(batch, rows, cols, type, steps, a, b, c, eps);
  if (rc) return rc;
  const int mask = type == GS_TYPE_F32 ? 3 : 1;
  if (update == nullptr || out == nullptr || (((uintptr_t)update | (uintptr_t)out) & mask) ||
      batch_stride < 0 || row_stride < 0 || col_stride < 0)
    return GS_ERR_INVALID_ARGUMENT;
  const Plan p = make_plan(batch, rows, cols, type);
  const bool tall = rows > cols;
  Source s{};
  s.u = update;
  s.type = type;
  s.batch_stride = batch_stride;
  s.row_stride = tall ? col_stride : row_stride;
  s.col_stride = tall ? row_stride : col_stride;
  s.rows = p.m;
  s.cols = p.n;
  Out o{};
  o.p = out;
  o.type = type;
  o.tall = tall;
  o.rows = p.m;
  o.cols = p.n;
  o.batch_stride = (int64_t)rows * cols;
  return run(batch, p, s, o, steps, a, b, c, eps, scratch, scratch_bytes,
             reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int gs_muon_step(int batch, int rows, int cols, int grad_type, float *params, const void *grads,
                            float *momentum, double lr, double beta, int nesterov, double weight_decay,
                            double scale, int steps, float a, float b, float c, float eps, void *scratch,
                            size_t scratch_bytes, void *stream) {
  const int rc = check(batch, rows, cols, grad_type, steps, a, b, c, eps);
  if (rc) return rc;
  const int mask = grad_type == GS_TYPE_F32 ? 3 : 1;
  if (params == nullptr || grads == nullptr || momentum == nullptr ||
      (((uintptr_t)params | (uintptr_t)momentum) & 3) || ((uintptr_t)grads & mask) || !(beta >= 0.0) ||
      !(beta < 1.0))
    return GS_ERR_INVALID_ARGUMENT;
  // fp32 weights: the full products, whatever the gradient's type
  const Plan p = make_plan(batch, rows, cols, GS_TYPE_F32);
  const bool tall = rows > cols;
  Source s{};
  s.u = grads;
  s.type = grad_type;
  s.batch_stride = (int64_t)rows * cols;
  s.row_stride = tall ? 1 : cols;
  s.col_stride = tall ? cols : 1;
  s.momentum = momentum;
  s.beta = (float)beta;
  s.fresh = (float)(1.0 - beta);
  s.nesterov = nesterov != 0;
  s.rows = p.m;
  s.cols = p.n;
  Out o{};
  o.p = params;
  o.type = GS_TYPE_F32;
  o.update = 1;
  o.tall = tall;
  o.rows = p.m;
  o.cols = p.n;
  o.batch_stride = s.batch_stride;
  o.decay = (float)(1.0 - lr * weight_decay);
  o.step = (float)(lr * scale);
  return run(batch, p, s, o, steps, a, b, c, eps, scratch, scratch_bytes,
             reinterpret_cast<cudaStream_t>(stream));
}
