// gfx950 (CDNA4 / MI355X) kernels for the Byzantine-resilient GARs.
//
// Written MI355X-first from the algorithm definitions in the reference
// (semantics of /root/reference/native/op_krum/cpu.cpp,
// op_bulyan/cpu.cpp and aggregators/deprecated_native/native.cpp -- see
// aggregathor_amd/ops/reference.py for the line-by-line mapping), NOT a
// port of its CPU threadpool code:
//
// - The [n, d] gradient matrix (n <= 64 workers, d up to ~100M fp32) lives in
//   HBM3E; every kernel is memory-bound, so the design minimizes passes over
//   the matrix and vectorizes global accesses (up to fvec<8> = 32 B/row per
//   thread, width-dispatched on the row alignment that d admits).
// - Pairwise distances: one pass over the matrix; each block accumulates ALL
//   pair partial sums for its d-chunk in registers (each loaded element is
//   reused n-1 times), then a deterministic fixed-shape tree reduction
//   produces the [n, n] matrix. No atomics -> bit-identical results on every
//   rank, which is what lets the GAR run replicated instead of
//   PS-and-broadcast.
// - Krum / Bulyan selection: a single workgroup stages the n x n distance
//   matrix in LDS and computes scores + top-k by rank counting (total order:
//   non-finite last, then value, then index -- the reference's isfinite
//   comparators refined to a deterministic tie-break). No host round trip:
//   the selection result stays on device, so a whole GAR step is
//   graph-capturable.
// - Bulyan tail is FUSED: selection averages of t rounds + coordinate-wise
//   averaged-median in ONE pass over [n, d] (the reference materialized a
//   t x d intermediate and re-read it, op_bulyan/cpu.cpp:59-60,163-187).
// - Coordinate-wise rules keep each column of n values in registers (rank
//   selection, fully unrolled over a templated NMAX) -- columns are read
//   coalesced since consecutive lanes hold consecutive coordinates.
//
// Numerics: fp32 throughout (the reference kernels are float/double; the
// training path feeds fp32 flattened gradients). Compiled WITHOUT fast-math:
// NaN ordering is load-bearing (NaN == +inf in every sort, NaN-skip in
// means).

#include <float.h>
#include <stdlib.h>
#include <string.h>

#include <hip/hip_runtime.h>

#include "gar_kernels.h"

namespace gar {

constexpr int kBlock = 256;
constexpr int kMaxBlocksD = 2048;  // cap + grid-stride (guideline 11)

static inline int nblocks_d(long d) {
  long d4 = d / 4;
  long want = (d4 + kBlock - 1) / kBlock;
  if (want < 1) want = 1;
  if (want > kMaxBlocksD) want = kMaxBlocksD;
  return (int)want;
}

// Aligned fp32 vector: rows of the [n, d] matrix start at arbitrary
// d-multiples, so the usable vector width is the largest power of two
// dividing d (a float4 access on a row with d % 4 != 0 would be
// misaligned). Launchers dispatch VW in {8, 4, 2, 1} per kernel (wider
// isn't always better: some NMAX variants clamp VW for register balance).
template <int VW>
struct alignas((VW * 4) < 16 ? (VW * 4) : 16) fvec {
  float v[VW];
};

static inline int vec_width(long d) {
  if (d % 8 == 0) return 8;
  if (d % 4 == 0) return 4;
  if (d % 2 == 0) return 2;
  return 1;
}

// Pair enumeration layout of the partials buffer: the templated small-n
// kernels enumerate pairs over NR compile-time rows; the generic tile kernel
// enumerates over n directly. pair_index(i, j, rows) for i < j.
__host__ __device__ static inline int pair_index(int i, int j, int rows) {
  return i * (2 * rows - i - 1) / 2 + (j - i - 1);
}

static inline int pair_layout_rows(int n) {
  if (n <= 8) return 8;
  if (n <= 16) return 16;
  return n;  // tile kernel uses n-enumeration
}

constexpr int kMfmaTC = 512;  // d-tile columns of the MFMA sqdist kernel

static inline int nblocks_mfma(long d) {
  long nt = (d + kMfmaTC - 1) / kMfmaTC;
  if (nt < 1) nt = 1;
  if (nt > kMaxBlocksD) nt = kMaxBlocksD;
  return (int)nt;
}

// Kernel choice for the distance pass: hand-written MFMA formulation or the
// VALU register-tile formulation (both deterministic, same partial layout).
// Env AGGREGATHOR_SQDIST = "mfma" | "valu"; the default is the measured
// winner on MI355X for the flagship n=8 shape.
static bool use_mfma_sqdist() {
  static int v = -1;
  if (v < 0) {
    const char* e = getenv("AGGREGATHOR_SQDIST");
    if (e && strcmp(e, "mfma") == 0) v = 1;
    else if (e && strcmp(e, "valu") == 0) v = 0;
    // Default: VALU. Measured on MI355X (d=25.6M fp32, built without packed
    // fp32): n=8 VALU 0.174 ms (4.7 TB/s algorithmic) vs MFMA 0.640 ms, n=11
    // 0.617 vs 1.95, n=16 0.710 vs 2.12. The f32-input MFMA runs at
    // the f32 VECTOR rate (64 cyc/SIMD issue for 32x32x2, guide section 3)
    // and only the 28-of-1024 diagonal outputs are useful, so the MFMA
    // formulation is ISSUE-bound ~2.5x over HBM at small n, while the VALU
    // kernel at 1.75 flop/B is purely HBM-bound. MFMA pairwise-L2 would pay
    // only for bf16-stored gradients (2075 TF rate); the reference's GAR
    // semantics are fp32.
    else v = 0;
  }
  return v != 0;
}

long sqdist_partials_elems(int n, long d) {
  int rows = pair_layout_rows(n);
  int nb = nblocks_d(d);
  if (n <= 16 && nblocks_mfma(d) > nb) nb = nblocks_mfma(d);
  return (long)nb * (rows * (rows - 1) / 2);
}

// ---------------------------------------------------------------------------
// Total order: non-finite last, then value, then index. This is the
// reference's isfinite comparator (op_krum/cpu.cpp:81-89) refined with a
// deterministic index tie-break (matches the stable argsort of
// ops/reference.py).
__device__ __forceinline__ bool lt_total(float av, int ai, float bv, int bi) {
  bool fa = isfinite(av), fb = isfinite(bv);
  if (fa != fb) return fa;
  if (!fa) return ai < bi;
  if (av != bv) return av < bv;
  return ai < bi;
}

// ---------------------------------------------------------------------------
// Pairwise squared-L2 distances, stage 1: per-block partial sums.
//
// Small-n kernel (n <= NR, NR in {8, 16}): every block walks its grid-stride
// share of the d dimension with float4 loads and keeps ALL NR*(NR-1)/2 pair
// accumulators in VGPRs (NR=8: 28 acc + 8 float4 = ~75 VGPR; NR=16 uses
// float2 loads to stay under the register cliff).

template <int NR, int VW>
__global__ __launch_bounds__(kBlock) void sqdist_small_kernel(
    const float* __restrict__ g, float* __restrict__ partials, long dv,
    long d, int n) {
  constexpr int P = NR * (NR - 1) / 2;
  float acc[P];
#pragma unroll
  for (int p = 0; p < P; ++p) acc[p] = 0.f;

  const long stride = (long)gridDim.x * blockDim.x;
  for (long x = (long)blockIdx.x * blockDim.x + threadIdx.x; x < dv;
       x += stride) {
    fvec<VW> v[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      if (i < n) {
        v[i] = reinterpret_cast<const fvec<VW>*>(g + (long)i * d)[x];
      } else {
#pragma unroll
        for (int c = 0; c < VW; ++c) v[i].v[c] = 0.f;
      }
    }
    int p = 0;
#pragma unroll
    for (int i = 0; i < NR - 1; ++i) {
#pragma unroll
      for (int j = i + 1; j < NR; ++j, ++p) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < VW; ++c) {
          float dd = v[i].v[c] - v[j].v[c];
          s = fmaf(dd, dd, s);
        }
        acc[p] += s;
      }
    }
  }
  // Tail coordinates (d % VW), handled once by block 0.
  long tail0 = dv * VW;
  if (blockIdx.x == 0 && threadIdx.x < (int)(d - tail0)) {
    long x = tail0 + threadIdx.x;
    int p = 0;
#pragma unroll
    for (int i = 0; i < NR - 1; ++i) {
#pragma unroll
      for (int j = i + 1; j < NR; ++j, ++p) {
        if (j < n) {
          float dd = g[(long)i * d + x] - g[(long)j * d + x];
          acc[p] = fmaf(dd, dd, acc[p]);
        }
      }
    }
  }
  // Deterministic per-pair block reduction (fixed tree shape).
  __shared__ float red[kBlock];
  for (int p = 0; p < P; ++p) {
    red[threadIdx.x] = acc[p];
    __syncthreads();
    for (int s = kBlock / 2; s > 0; s >>= 1) {
      if ((int)threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
      __syncthreads();
    }
    if (threadIdx.x == 0) partials[(long)blockIdx.x * P + p] = red[0];
    __syncthreads();
  }
}

// Generic row-tile kernel for n > 16: blockIdx.y selects an 8x8 tile of the
// upper-triangular pair space; each row chunk is re-read ~n/8 times (still
// one HBM pass per tile thanks to L2), accumulators stay at 64 VGPRs.
template <int VW>
__global__ __launch_bounds__(kBlock) void sqdist_tile_kernel(
    const float* __restrict__ g, float* __restrict__ partials, long dv,
    long d, int n, int tiles_per_row) {
  // Decode upper-triangular tile (ti <= tj).
  int tile = blockIdx.y;
  int ti = 0;
  {
    int rem = tile;
    while (rem >= tiles_per_row - ti) {
      rem -= tiles_per_row - ti;
      ++ti;
    }
    tile = rem;
  }
  int tj = ti + tile;
  int i0 = ti * 8, j0 = tj * 8;
  const int P = n * (n - 1) / 2;

  float acc[64];
#pragma unroll
  for (int p = 0; p < 64; ++p) acc[p] = 0.f;

  const long stride = (long)gridDim.x * blockDim.x;
  for (long x = (long)blockIdx.x * blockDim.x + threadIdx.x; x < dv;
       x += stride) {
    fvec<VW> vi[8], vj[8];
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      int gi = i0 + a, gj = j0 + a;
      if (gi < n) {
        vi[a] = reinterpret_cast<const fvec<VW>*>(g + (long)gi * d)[x];
      } else {
#pragma unroll
        for (int c = 0; c < VW; ++c) vi[a].v[c] = 0.f;
      }
      if (gj < n) {
        vj[a] = reinterpret_cast<const fvec<VW>*>(g + (long)gj * d)[x];
      } else {
#pragma unroll
        for (int c = 0; c < VW; ++c) vj[a].v[c] = 0.f;
      }
    }
#pragma unroll
    for (int a = 0; a < 8; ++a) {
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < VW; ++c) {
          float dd = vi[a].v[c] - vj[b].v[c];
          s = fmaf(dd, dd, s);
        }
        acc[a * 8 + b] += s;
      }
    }
  }
  long tail0 = dv * VW;
  if (blockIdx.x == 0 && threadIdx.x < (int)(d - tail0)) {
    long x = tail0 + threadIdx.x;
#pragma unroll
    for (int a = 0; a < 8; ++a) {
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        int gi = i0 + a, gj = j0 + b;
        if (gi < n && gj < n && gi < gj) {
          float dd = g[(long)gi * d + x] - g[(long)gj * d + x];
          acc[a * 8 + b] = fmaf(dd, dd, acc[a * 8 + b]);
        }
      }
    }
  }
  __shared__ float red[kBlock];
  for (int a = 0; a < 8; ++a) {
    for (int b = 0; b < 8; ++b) {
      int gi = i0 + a, gj = j0 + b;
      if (!(gi < n && gj < n && gi < gj)) continue;
      red[threadIdx.x] = acc[a * 8 + b];
      __syncthreads();
      for (int s = kBlock / 2; s > 0; s >>= 1) {
        if ((int)threadIdx.x < s) red[threadIdx.x] += red[threadIdx.x + s];
        __syncthreads();
      }
      if (threadIdx.x == 0)
        partials[(long)blockIdx.x * P + pair_index(gi, gj, n)] = red[0];
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// LDS-staged single-HBM-pass kernel for 16 < n <= 64 (round-2 fix for the
// large-n bandwidth cliff, profiles/gar_scaling_n.txt).
//
// The 8x8 tile kernel above re-reads each row chunk ~n/8 times from HBM
// because its pair tiles land on different XCDs whose L2s cannot share the
// working set (measured: krum algorithmic bandwidth 4.4 TB/s at n=8 but
// 1.75 at n=16 and 0.93 at n=32). This kernel makes the amplification 1:
// each workgroup stages a [n, CHUNK] tile of the matrix in LDS ONCE per
// chunk, then its 4 waves sweep all upper-triangular 8x8 pair tiles from
// LDS, so every gradient byte is fetched from HBM exactly once per block
// stripe. Per chunk, each wave reduces its 64 per-lane pair partials with
// a fixed-shape shfl_xor butterfly (deterministic) and accumulates them
// into an LDS pair table; the table is flushed to the per-block partials
// row at the end (same layout as the other kernels, reduced by
// sqdist_reduce_kernel). No atomics anywhere; every reduction order is
// fixed -> bit-deterministic, replicated-GAR safe.
//
// LDS budget (64 KB default): tile n*CHUNK*4 B + pair table
// n(n-1)/2*4 B. CHUNK is chosen at launch as the largest multiple of 64
// that fits (n=32 -> 448 cols, n=64 -> 192).

constexpr int kLdsBlock = 512;  // 8 waves: latency hiding at 1 block/CU

template <int VW>
__global__ __launch_bounds__(kLdsBlock) void sqdist_lds_kernel(
    const float* __restrict__ g, float* __restrict__ partials, long d,
    int n, int chunk, int tiles_per_row, int ntiles) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int P = n * (n - 1) / 2;
  float* tile = lds;          // [n, chunk] staged rows
  float* accp = lds + (long)n * chunk;  // [P] pair accumulators

  for (int p = threadIdx.x; p < P; p += kLdsBlock) accp[p] = 0.f;

  const int lane = (int)threadIdx.x & 63;
  const int wave = (int)threadIdx.x >> 6;
  const int nwaves = kLdsBlock / 64;
  const long nchunks = (d + chunk - 1) / chunk;

  for (long ci = blockIdx.x; ci < nchunks; ci += gridDim.x) {
    const long c0 = ci * chunk;
    const int cw = (int)((d - c0) < chunk ? (d - c0) : chunk);
    __syncthreads();  // pair-table reads of the previous chunk done
    // Stage [n, cw] into LDS (vectorized when alignment allows: chunk is
    // a multiple of 64, so c0 keeps the row alignment class of d).
    const int cwv = cw / VW;
    for (int idx = threadIdx.x; idx < n * cwv; idx += kLdsBlock) {
      int r = idx / cwv, cc = (idx - r * cwv) * VW;
      fvec<VW> v = *reinterpret_cast<const fvec<VW>*>(g + (long)r * d + c0 + cc);
#pragma unroll
      for (int k = 0; k < VW; ++k) tile[(long)r * chunk + cc + k] = v.v[k];
    }
    for (int idx = threadIdx.x; idx < n * (cw - cwv * VW); idx += kLdsBlock) {
      int rem = cw - cwv * VW;
      int r = idx / rem, cc = cwv * VW + (idx - r * rem);
      tile[(long)r * chunk + cc] = g[(long)r * d + c0 + cc];
    }
    __syncthreads();

    for (int t = wave; t < ntiles; t += nwaves) {
      // Decode upper-triangular tile t -> (ti, tj), ti <= tj.
      int ti = 0, rem = t;
      while (rem >= tiles_per_row - ti) {
        rem -= tiles_per_row - ti;
        ++ti;
      }
      int tj = ti + rem;
      int i0 = ti * 8, j0 = tj * 8;
      float acc[64];
#pragma unroll
      for (int p = 0; p < 64; ++p) acc[p] = 0.f;
      // Main loop: ds_read_b128 (4 coords per LDS access per row); chunk
      // is a multiple of 64 so LDS rows are 16 B aligned.
      const int cw4 = cw & ~3;
      for (int x = lane * 4; x < cw4; x += 64 * 4) {
        fvec<4> vi[8], vj[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          if (i0 + a < n)
            vi[a] = *reinterpret_cast<const fvec<4>*>(
                tile + (long)(i0 + a) * chunk + x);
          else
#pragma unroll
            for (int k = 0; k < 4; ++k) vi[a].v[k] = 0.f;
          if (j0 + a < n)
            vj[a] = *reinterpret_cast<const fvec<4>*>(
                tile + (long)(j0 + a) * chunk + x);
          else
#pragma unroll
            for (int k = 0; k < 4; ++k) vj[a].v[k] = 0.f;
        }
#pragma unroll
        for (int a = 0; a < 8; ++a)
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            float s = acc[a * 8 + b];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float dd = vi[a].v[k] - vj[b].v[k];
              s = fmaf(dd, dd, s);
            }
            acc[a * 8 + b] = s;
          }
      }
      for (int x = cw4 + lane; x < cw; x += 64) {  // scalar tail
        float vi[8], vj[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) {
          vi[a] = (i0 + a < n) ? tile[(long)(i0 + a) * chunk + x] : 0.f;
          vj[a] = (j0 + a < n) ? tile[(long)(j0 + a) * chunk + x] : 0.f;
        }
#pragma unroll
        for (int a = 0; a < 8; ++a)
#pragma unroll
          for (int b = 0; b < 8; ++b) {
            float dd = vi[a] - vj[b];
            acc[a * 8 + b] = fmaf(dd, dd, acc[a * 8 + b]);
          }
      }
      // Butterfly TRANSPOSE-reduce (fixed shape, deterministic): at the
      // step with xor-distance s the register count halves and pair-index
      // bit log2(s) is re-encoded as lane bit log2(s); after 6 steps
      // lane l's acc[0] holds the complete wave sum of pair index l.
#pragma unroll
      for (int s = 32, R = 32; s >= 1; s >>= 1, R >>= 1) {
#pragma unroll
        for (int p = 0; p < 32; ++p) {
          if (p >= R) break;
          bool hi = (lane & s) != 0;
          float mine = hi ? acc[p + R] : acc[p];
          float send = hi ? acc[p] : acc[p + R];
          acc[p] = mine + __shfl_xor(send, s, 64);
        }
      }
      // One parallel LDS add per lane (distinct pairs -> distinct
      // addresses; tile owned by this wave alone -> no race; chunk-
      // sequential order -> deterministic).
      {
        int gi = i0 + (lane >> 3), gj = j0 + (lane & 7);
        if (gi < n && gj < n && gi < gj)
          accp[pair_index(gi, gj, n)] += acc[0];
      }
    }
  }
  __syncthreads();
  for (int p = threadIdx.x; p < P; p += kLdsBlock)
    partials[(long)blockIdx.x * P + p] = accp[p];
}

// ---------------------------------------------------------------------------
// MFMA pairwise-distance kernel (n <= 16): the matrix-core formulation of
// the same computation.
//
// Per d-tile staged in LDS, each wave builds per-lane DIFFERENCE values
// v = g[a_p][k] - g[b_p][k] (pair p = lane%32, k-slot = lane/32) and issues
// `v_mfma_f32_32x32x2_f32` with the SAME register as both A and B operands:
// A[i][k] = v(lane: i=l&31, k=l>>5) and B[k][j] = v(lane: j=l&31, k=l>>5)
// means C = P P^T exactly, and its DIAGONAL is the per-pair squared
// distance. f32-in MFMA is exact fp32 fma-chain math (no xf32 on gfx950),
// so numerics match the VALU kernel's class. The off-diagonal 31/32 of the
// MFMA tile is unused compute -- irrelevant here because the kernel is HBM-
// bound (28 pairs x 2 flop / 32 B/coordinate = 1.75 flop/B << any peak);
// what MFMA buys is freeing the VALU from the 28-accumulator FMA chains.
// Selection between this and the VALU kernel: env AGGREGATHOR_SQDIST
// (mfma | valu); both produce the same partials layout.
//
// C/D layout of 32x32 MFMA (guide §3): col = l&31, row = (reg&3) + 8*(reg>>2)
// + 4*(l>>5). Diagonal element p lives in lane (p&31) + 32*hi with
// hi = (p>>2)&1 and reg = (val&3) | ((val>>3)<<2) where val = p - 4*hi.

using f32x16 = __attribute__((ext_vector_type(16))) float;

template <int NR, int TC>  // NR rows (<=16), TC tile columns (multiple of 8)
__global__ __launch_bounds__(kBlock) void sqdist_mfma_kernel(
    const float* __restrict__ g, float* __restrict__ partials, long d,
    int n, int ntiles) {
  constexpr int P = NR * (NR - 1) / 2;
  constexpr int NPG = (P + 31) / 32;  // pair groups of 32
  constexpr int LDC = TC + 1;         // +1 word: bank-conflict break
  __shared__ float tile[NR * LDC];
  __shared__ float part[4][P];  // per-wave partials, combined in fixed order

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  // Pair tables (compile-time NR enumeration, runtime n guard).
  int pa[NPG], pb[NPG];
#pragma unroll
  for (int gidx = 0; gidx < NPG; ++gidx) {
    int p = gidx * 32 + (lane & 31);
    // decode NR-enumeration pair p -> (i, j)
    int i = 0, rem = p;
    bool valid = p < P;
#pragma unroll
    for (int r = 0; r < NR - 1; ++r) {
      if (valid && rem >= NR - 1 - r && i == r) {
        rem -= NR - 1 - r;
        ++i;
      }
    }
    int j = i + 1 + rem;
    valid = valid && (j < n);
    pa[gidx] = valid ? i : 0;
    pb[gidx] = valid ? j : 0;  // invalid pairs: i==j==0 -> zero difference
  }
  const int khalf = lane >> 5;  // k-slot within the 2-deep MFMA K

  f32x16 acc[NPG];
#pragma unroll
  for (int gidx = 0; gidx < NPG; ++gidx)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[gidx][r] = 0.f;

  for (int t = blockIdx.x; t < ntiles; t += gridDim.x) {
    const long x0 = (long)t * TC;
    // Stage [NR][TC] into LDS, coalesced, zero-fill past d and past n.
    for (int idx = tid; idx < NR * TC; idx += kBlock) {
      int row = idx / TC, col = idx % TC;
      long x = x0 + col;
      tile[row * LDC + col] =
          (row < n && x < d) ? g[(long)row * d + x] : 0.f;
    }
    __syncthreads();
    // Each wave owns a contiguous quarter of the tile's K range.
    const int kper = TC / 4;
    const int kbeg = wave * kper;
#pragma unroll 4
    for (int k = 0; k < kper; k += 2) {
      const int kk = kbeg + k + khalf;
#pragma unroll
      for (int gidx = 0; gidx < NPG; ++gidx) {
        float va = tile[pa[gidx] * LDC + kk];
        float vb = tile[pb[gidx] * LDC + kk];
        float v = va - vb;
        acc[gidx] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, v, acc[gidx],
                                                         0, 0, 0);
      }
    }
    __syncthreads();
  }
  // Diagonal extraction: pair p owned by lane (p&31)+32*((p>>2)&1).
#pragma unroll
  for (int gidx = 0; gidx < NPG; ++gidx) {
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      if (khalf == hi) {
        int p_lane = lane & 31;                       // candidate col
        int val = p_lane - 4 * hi;
        if (val >= 0 && (val & 4) == 0) {
          int reg = (val & 3) | ((val >> 3) << 2);
          int row = (reg & 3) + 8 * (reg >> 2) + 4 * hi;
          if (row == p_lane) {
            int p = gidx * 32 + p_lane;
            if (p < P) part[wave][p] = acc[gidx][reg];
          }
        }
      }
    }
  }
  __syncthreads();
  // Fixed-order cross-wave combine -> deterministic block partial.
  for (int p = tid; p < P; p += kBlock) {
    float s = part[0][p];
    s += part[1][p];
    s += part[2][p];
    s += part[3][p];
    partials[(long)blockIdx.x * P + p] = s;
  }
}

// Stage 2: deterministic cross-block reduction -> [n, n] symmetric matrix
// with +inf diagonal (the diagonal is never a candidate; the reference
// stores T::max there, op_bulyan/cpu.cpp:75).
__global__ void sqdist_reduce_kernel(const float* __restrict__ partials,
                                     float* __restrict__ dist, int nblk,
                                     int n, int layout_rows) {
  int p = blockIdx.x;  // n-enumeration pair index
  // Decode p -> (i, j).
  int i = 0, rem = p;
  while (rem >= n - 1 - i) {
    rem -= n - 1 - i;
    ++i;
  }
  int j = i + 1 + rem;
  int P = layout_rows * (layout_rows - 1) / 2;
  int pl = pair_index(i, j, layout_rows);

  __shared__ float red[kBlock];
  float s = 0.f;
  for (int b = threadIdx.x; b < nblk; b += kBlock)
    s += partials[(long)b * P + pl];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int st = kBlock / 2; st > 0; st >>= 1) {
    if ((int)threadIdx.x < st) red[threadIdx.x] += red[threadIdx.x + st];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    dist[(long)i * n + j] = red[0];
    dist[(long)j * n + i] = red[0];
  }
}

__global__ void fill_diag_inf_kernel(float* dist, int n) {
  int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) dist[(long)i * n + i] = HUGE_VALF;
}

void sqdist(const float* g, int n, long d, float* partials, float* dist,
            hipStream_t stream) {
  int nblk = nblocks_d(d);
  int vw = vec_width(d);
  if (n <= 16 && use_mfma_sqdist()) {
    int ntiles = (int)((d + kMfmaTC - 1) / kMfmaTC);
    nblk = nblocks_mfma(d);
    if (n <= 8)
      sqdist_mfma_kernel<8, kMfmaTC>
          <<<nblk, kBlock, 0, stream>>>(g, partials, d, n, ntiles);
    else
      sqdist_mfma_kernel<16, kMfmaTC>
          <<<nblk, kBlock, 0, stream>>>(g, partials, d, n, ntiles);
  } else if (n <= 8) {
    if (vw == 4)
      sqdist_small_kernel<8, 4>
          <<<nblk, kBlock, 0, stream>>>(g, partials, d / 4, d, n);
    else if (vw == 2)
      sqdist_small_kernel<8, 2>
          <<<nblk, kBlock, 0, stream>>>(g, partials, d / 2, d, n);
    else
      sqdist_small_kernel<8, 1>
          <<<nblk, kBlock, 0, stream>>>(g, partials, d, d, n);
  } else if (n <= 16) {
    if (vw >= 2)
      sqdist_small_kernel<16, 2>
          <<<nblk, kBlock, 0, stream>>>(g, partials, d / 2, d, n);
    else
      sqdist_small_kernel<16, 1>
          <<<nblk, kBlock, 0, stream>>>(g, partials, d, d, n);
  } else {
    int tiles_per_row = (n + 7) / 8;
    int ntiles = tiles_per_row * (tiles_per_row + 1) / 2;
    const char* e = getenv("AGGREGATHOR_SQDIST");
    if (e && strcmp(e, "tile") == 0) {
      // Legacy multi-pass tile kernel (A/B reference; ~n/8 HBM re-reads).
      // Measured: VW=4 (170 VGPR + scratch) loses to VW=2.
      dim3 grid(nblk, ntiles);
      if (vw >= 2)
        sqdist_tile_kernel<2><<<grid, kBlock, 0, stream>>>(
            g, partials, d / 2, d, n, tiles_per_row);
      else
        sqdist_tile_kernel<1><<<grid, kBlock, 0, stream>>>(g, partials, d, d,
                                                           n, tiles_per_row);
    } else {
      // Default: LDS-staged single-HBM-pass kernel. 128 KB dynamic LDS
      // (gfx950 has 160 KB/CU; >64 KB needs the explicit opt-in) doubles
      // the chunk, halving the per-chunk fold overhead; occupancy is one
      // block/CU, which the 8-wave block size covers.
      int P = n * (n - 1) / 2;
      int chunk = ((128 * 1024 / 4 - P) / n) / 64 * 64;
      long nchunks = (d + chunk - 1) / chunk;
      int grid = (int)(nchunks < 512 ? nchunks : 512);
      if (grid > nblk) grid = nblk;
      nblk = grid;
      size_t shmem = ((size_t)n * chunk + P) * 4;
      const void* fn = (vw >= 4) ? (const void*)&sqdist_lds_kernel<4>
                     : (vw >= 2) ? (const void*)&sqdist_lds_kernel<2>
                                 : (const void*)&sqdist_lds_kernel<1>;
      (void)hipFuncSetAttribute(fn,
                                hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)shmem);
      if (vw >= 4)
        sqdist_lds_kernel<4><<<grid, kLdsBlock, shmem, stream>>>(
            g, partials, d, n, chunk, tiles_per_row, ntiles);
      else if (vw >= 2)
        sqdist_lds_kernel<2><<<grid, kLdsBlock, shmem, stream>>>(
            g, partials, d, n, chunk, tiles_per_row, ntiles);
      else
        sqdist_lds_kernel<1><<<grid, kLdsBlock, shmem, stream>>>(
            g, partials, d, n, chunk, tiles_per_row, ntiles);
    }
  }
  int P = n * (n - 1) / 2;
  sqdist_reduce_kernel<<<P, kBlock, 0, stream>>>(partials, dist, nblk, n,
                                                 pair_layout_rows(n));
  fill_diag_inf_kernel<<<1, 64, 0, stream>>>(dist, n);
}

// ---------------------------------------------------------------------------
// Multi-Krum selection (one workgroup, LDS-staged; op_krum/cpu.cpp:74-119
// semantics). Scores and top-m by rank counting under the total order.

__global__ void krum_select_kernel(const float* __restrict__ dist, int n,
                                   int f, int m, int* __restrict__ sel) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* sd = reinterpret_cast<float*>(smem);  // n*n
  float* scores = sd + n * n;                  // n
  for (int i = threadIdx.x; i < n * n; i += blockDim.x) sd[i] = dist[i];
  __syncthreads();
  const int nbin = n - f - 2;
  const int i = threadIdx.x;
  if (i < n) {
    // score_i = sum of i's nbin smallest distances (rank < nbin under the
    // total order == stable-sorted prefix).
    float score = 0.f;
    for (int j = 0; j < n; ++j) {
      if (j == i) continue;
      float vj = sd[i * n + j];
      int rank = 0;
      for (int l = 0; l < n; ++l) {
        if (l == i || l == j) continue;
        if (lt_total(sd[i * n + l], l, vj, j)) ++rank;
      }
      if (rank < nbin) score += vj;
    }
    scores[i] = score;
  }
  __syncthreads();
  if (i < n) {
    float vi = scores[i];
    int rank = 0;
    for (int l = 0; l < n; ++l)
      if (l != i && lt_total(scores[l], l, vi, i)) ++rank;
    if (rank < m) sel[rank] = i;  // ascending-score order by construction
  }
}

void krum_select(const float* dist, int n, int f, int m, int* sel,
                 hipStream_t stream) {
  size_t lds = (size_t)(n * n + n) * sizeof(float);
  krum_select_kernel<<<1, kBlock, lds, stream>>>(dist, n, f, m, sel);
}

// ---------------------------------------------------------------------------
// Selection average: out = mean of the m selected rows (operations.hpp:67-76).

template <int VW>
__global__ __launch_bounds__(kBlock) void selection_average_kernel(
    const float* __restrict__ g, float* __restrict__ out, long dv, long d,
    const int* __restrict__ sel_g, int m) {
  __shared__ int sel[kMaxNSelect];
  if ((int)threadIdx.x < m) sel[threadIdx.x] = sel_g[threadIdx.x];
  __syncthreads();
  const float inv = 1.f / (float)m;
  const long stride = (long)gridDim.x * blockDim.x;
  for (long x = (long)blockIdx.x * blockDim.x + threadIdx.x; x < dv;
       x += stride) {
    fvec<VW> s;
#pragma unroll
    for (int c = 0; c < VW; ++c) s.v[c] = 0.f;
    for (int i = 0; i < m; ++i) {
      fvec<VW> v = reinterpret_cast<const fvec<VW>*>(g + (long)sel[i] * d)[x];
#pragma unroll
      for (int c = 0; c < VW; ++c) s.v[c] += v.v[c];
    }
#pragma unroll
    for (int c = 0; c < VW; ++c) s.v[c] *= inv;
    reinterpret_cast<fvec<VW>*>(out)[x] = s;
  }
  long tail0 = dv * VW;
  if (blockIdx.x == 0 && threadIdx.x < (int)(d - tail0)) {
    long x = tail0 + threadIdx.x;
    float s = 0.f;
    for (int i = 0; i < m; ++i) s += g[(long)sel[i] * d + x];
    out[x] = s * inv;
  }
}

void selection_average(const float* g, int n, long d, const int* sel, int m,
                       float* out, hipStream_t stream) {
  (void)n;
  int nblk = nblocks_d(d);
  int vw = vec_width(d);
  if (vw == 8)
    selection_average_kernel<8>
        <<<nblk, kBlock, 0, stream>>>(g, out, d / 8, d, sel, m);
  else if (vw == 4)
    selection_average_kernel<4>
        <<<nblk, kBlock, 0, stream>>>(g, out, d / 4, d, sel, m);
  else if (vw == 2)
    selection_average_kernel<2>
        <<<nblk, kBlock, 0, stream>>>(g, out, d / 2, d, sel, m);
  else
    selection_average_kernel<1>
        <<<nblk, kBlock, 0, stream>>>(g, out, d, d, sel, m);
}

// ---------------------------------------------------------------------------
// Bulyan selection schedule (one workgroup; op_bulyan/cpu.cpp:88-161
// semantics: initial scores + per-row distance pruning, then t rounds of
// select-average-evict with score decrement by the pruned distance).

__global__ void bulyan_select_kernel(const float* __restrict__ dist, int n,
                                     int f, int m,
                                     unsigned char* __restrict__ flags) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* sd = reinterpret_cast<float*>(smem);  // n*n, pruned in place
  float* scores = sd + n * n;                  // n
  int* evicted = reinterpret_cast<int*>(scores + n);
  unsigned char* alive = reinterpret_cast<unsigned char*>(evicted + 1);
  for (int i = threadIdx.x; i < n * n; i += blockDim.x) sd[i] = dist[i];
  __syncthreads();
  const int nbin = n - f - 2;
  const int t = n - 2 * f - 2;
  const int i = threadIdx.x;
  if (i < n) {
    float score = 0.f;
    unsigned long long keep = 0ull;  // n <= 64
    for (int j = 0; j < n; ++j) {
      if (j == i) continue;
      float vj = sd[i * n + j];
      int rank = 0;
      for (int l = 0; l < n; ++l) {
        if (l == i || l == j) continue;
        if (lt_total(sd[i * n + l], l, vj, j)) ++rank;
      }
      if (rank < nbin) {
        score += vj;
        keep |= 1ull << j;
      }
    }
    // Prune row i: non-kept distances (and the diagonal) become 0
    // (cpu.cpp:116-129), so the eviction decrement reads 0 for them.
    for (int j = 0; j < n; ++j)
      if (j == i || !((keep >> j) & 1ull)) sd[i * n + j] = 0.f;
    scores[i] = score;
    alive[i] = 1;
  }
  __syncthreads();
  for (int k = 0;; ++k) {
    if (i < n) {
      float vi = scores[i];
      int rank = 0;
      for (int l = 0; l < n; ++l)
        if (l != i && lt_total(scores[l], l, vi, i)) ++rank;
      flags[(long)k * n + i] = (rank < m - k) ? 1 : 0;
      if (rank == 0) *evicted = i;
    }
    __syncthreads();
    if (k + 1 >= t) break;
    int ev = *evicted;
    if (i < n) {
      if (i == ev) {
        scores[i] = FLT_MAX;  // reference uses T::max (cpu.cpp:154)
        alive[i] = 0;
      } else if (alive[i]) {
        scores[i] -= sd[i * n + ev];
      }
    }
    __syncthreads();
  }
}

long bulyan_flags_bytes(int n, int f) {
  const int t = n - 2 * f - 2;
  return ((long)(t * n + 15) & ~15L) + (long)t * sizeof(float);
}

void bulyan_select(const float* dist, int n, int f, int m,
                   unsigned char* flags, hipStream_t stream) {
  size_t lds = (size_t)(n * n + n) * sizeof(float) + sizeof(int) + n + 16;
  bulyan_select_kernel<<<1, kBlock, lds, stream>>>(dist, n, f, m, flags);
}

// ---------------------------------------------------------------------------
// Per-coordinate rank-selection helpers (fully unrolled over NMAX so the
// column stays in VGPRs; n is runtime <= NMAX).

// Monotonic integer key for the total order: an ascending unsigned compare
// of keys == lt_total on the values (non-finite -> max key, ties fall to the
// index compare; -0.0 orders just before +0.0 which is observationally
// equivalent since the values compare equal). Computing the key costs O(n)
// per column ONCE, turning every rank comparison into 2 integer ops -- the
// naive per-comparison isfinite chain made median/averaged-median VALU-bound
// (measured 1.76 / 0.89 TB/s before, see profiles/).
__device__ __forceinline__ unsigned sort_key(float v) {
  if (!isfinite(v)) return 0xFFFFFFFFu;
  unsigned u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <int NMAX>
__device__ __forceinline__ float coord_median(const float (&vals)[NMAX],
                                              int n) {
  // Element at rank n/2 under the total order (native.cpp:686-694).
  const int target = n / 2;
  unsigned keys[NMAX];
#pragma unroll
  for (int i = 0; i < NMAX; ++i) {
    if (i >= n) continue;
    keys[i] = sort_key(vals[i]);
  }
  float out = 0.f;
#pragma unroll
  for (int i = 0; i < NMAX; ++i) {
    if (i >= n) continue;
    int rank = 0;
#pragma unroll
    for (int j = 0; j < NMAX; ++j) {
      if (j >= n) continue;
      if (j != i)
        rank += (keys[j] < keys[i]) | ((keys[j] == keys[i]) & (j < i));
    }
    if (rank == target) out = vals[i];
  }
  return out;
}

template <int NMAX>
__device__ __forceinline__ float coord_averaged_median(
    const float (&vals)[NMAX], int n, int beta) {
  // Mean of the beta elements closest to the median (native.cpp:714-739).
  const float zero = coord_median<NMAX>(vals, n);
  unsigned dkeys[NMAX];
#pragma unroll
  for (int i = 0; i < NMAX; ++i) {
    if (i >= n) continue;
    dkeys[i] = sort_key(fabsf(vals[i] - zero));
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NMAX; ++i) {
    if (i >= n) continue;
    int rank = 0;
#pragma unroll
    for (int j = 0; j < NMAX; ++j) {
      if (j >= n) continue;
      if (j != i)
        rank += (dkeys[j] < dkeys[i]) | ((dkeys[j] == dkeys[i]) & (j < i));
    }
    if (rank < beta) sum += vals[i];
  }
  return sum / (float)beta;
}

// Load one float4-column block of the matrix into registers, then run a
// scalar per-coordinate functor on each of the 4 components. OP signature:
// float op(const float (&vals)[NMAX], int n).
template <int NMAX, int VW, class OP>
__global__ __launch_bounds__(kBlock) void coordwise_kernel(
    const float* __restrict__ g, float* __restrict__ out, long dv, long d,
    int n, OP op) {
  const long stride = (long)gridDim.x * blockDim.x;
  for (long x = (long)blockIdx.x * blockDim.x + threadIdx.x; x < dv;
       x += stride) {
    fvec<VW> colv[NMAX];
#pragma unroll
    for (int i = 0; i < NMAX; ++i) {
      if (i >= n) continue;
      colv[i] = reinterpret_cast<const fvec<VW>*>(g + (long)i * d)[x];
    }
    fvec<VW> res;
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      float vals[NMAX];
#pragma unroll
      for (int i = 0; i < NMAX; ++i) {
        if (i >= n) continue;
        vals[i] = colv[i].v[c];
      }
      res.v[c] = op(vals, n);
    }
    reinterpret_cast<fvec<VW>*>(out)[x] = res;
  }
  long tail0 = dv * VW;
  if (blockIdx.x == 0 && threadIdx.x < (int)(d - tail0)) {
    long x = tail0 + threadIdx.x;
    float vals[NMAX];
#pragma unroll
    for (int i = 0; i < NMAX; ++i) {
      if (i >= n) continue;
      vals[i] = g[(long)i * d + x];
    }
    out[x] = op(vals, n);
  }
}

template <int NMAX>
struct MedianOp {
  __device__ float operator()(const float (&vals)[NMAX], int n) const {
    return coord_median<NMAX>(vals, n);
  }
};

template <int NMAX>
struct AveragedMedianOp {
  int beta;
  __device__ float operator()(const float (&vals)[NMAX], int n) const {
    return coord_averaged_median<NMAX>(vals, n, beta);
  }
};

template <int NMAX>
struct AverageNanOp {
  // Mean of the finite values; 0/0 -> NaN (native.cpp:756-775).
  __device__ float operator()(const float (&vals)[NMAX], int n) const {
    float sum = 0.f;
    float count = 0.f;
#pragma unroll
    for (int i = 0; i < NMAX; ++i) {
      if (i >= n) continue;
      if (isfinite(vals[i])) {
        sum += vals[i];
        count += 1.f;
      }
    }
    return sum / count;
  }
};

template <int NMAX, template <int> class OP, class... Args>
static void launch_coordwise_n(const float* g, int n, long d, float* out,
                               hipStream_t stream, Args... args) {
  int nblk = nblocks_d(d);
  int vw = vec_width(d);
  if (vw > 4) vw = 4;  // register balance: 8-wide doubles the column regs
  if (NMAX >= 32 && vw > 2) vw = 2;  // NMAX=32 @ VW=4 spills to scratch
  if (vw == 4)
    coordwise_kernel<NMAX, 4, OP<NMAX>>
        <<<nblk, kBlock, 0, stream>>>(g, out, d / 4, d, n, OP<NMAX>{args...});
  else if (vw == 2)
    coordwise_kernel<NMAX, 2, OP<NMAX>>
        <<<nblk, kBlock, 0, stream>>>(g, out, d / 2, d, n, OP<NMAX>{args...});
  else
    coordwise_kernel<NMAX, 1, OP<NMAX>>
        <<<nblk, kBlock, 0, stream>>>(g, out, d, d, n, OP<NMAX>{args...});
}

template <template <int> class OP, class... Args>
static void launch_coordwise(const float* g, int n, long d, float* out,
                             hipStream_t stream, Args... args) {
  if (n <= 8)
    launch_coordwise_n<8, OP>(g, n, d, out, stream, args...);
  else if (n <= 16)
    launch_coordwise_n<16, OP>(g, n, d, out, stream, args...);
  else
    // NMAX=32 at VW=4 spills the 128-register column to scratch; VW=2
    // keeps it resident (measured in kernel-resource-usage).
    launch_coordwise_n<kMaxNCoord, OP>(g, n, d, out, stream, args...);
}

void median(const float* g, int n, long d, float* out, hipStream_t stream) {
  launch_coordwise<MedianOp>(g, n, d, out, stream);
}

void averaged_median(const float* g, int n, long d, int beta, float* out,
                     hipStream_t stream) {
  launch_coordwise<AveragedMedianOp>(g, n, d, out, stream, beta);
}

void average_nan(const float* g, int n, long d, float* out,
                 hipStream_t stream) {
  launch_coordwise<AverageNanOp>(g, n, d, out, stream);
}

// ---------------------------------------------------------------------------
// Fused Bulyan tail: per coordinate, compute the t selection averages (from
// the flags schedule) and the averaged-median over them, in one pass over
// [n, d] (the reference wrote a t x d intermediate, op_bulyan/cpu.cpp:59-60).

template <int NMAX, int VW>
__global__ __launch_bounds__(kBlock) void bulyan_final_kernel(
    const float* __restrict__ g, float* __restrict__ out, long dv, long d,
    int n, int t, int b, const unsigned char* __restrict__ flags_g,
    const float* __restrict__ inv_mk) {
  __shared__ float inv[NMAX];
  // Selection sets as uint64 bitmasks (n <= 64) in LDS, read back through
  // a VOLATILE pointer inside the hot loop: the per-wave SGPR file (~102
  // words) cannot hold t masks as hoisted uniforms -- a byte-matrix
  // version produced 633 SGPR spills + 272 B/lane scratch (measured 33x
  // over the kernel's traffic bound), and a register-array version 2522
  // spills. The volatile ds_read_b64 lands each mask in VGPRs per
  // iteration (t reads per coordinate, trivially cheap) and the bit
  // tests stay VALU cndmask/add chains with zero scratch.
  __shared__ unsigned long long mk_s[NMAX];
  if ((int)threadIdx.x < t) {
    inv[threadIdx.x] = inv_mk[threadIdx.x];
    unsigned long long m = 0;
    for (int i = 0; i < n; ++i)
      if (flags_g[threadIdx.x * n + i]) m |= 1ull << i;
    mk_s[threadIdx.x] = m;
  }
  __syncthreads();
  // The masks must stay in VGPRs, re-read per iteration: left to itself
  // the compiler hoists the (wave-uniform) loads into SGPRs and spills
  // them (~102 addressable SGPRs/wave; the byte-matrix version measured
  // 633 spills + 272 B/lane scratch, 33x over the traffic bound). The
  // empty volatile asm pins each half in a VGPR and is opaque to LICM.
  const unsigned* mkv32 = reinterpret_cast<const unsigned*>(mk_s);

  const long stride = (long)gridDim.x * blockDim.x;
  for (long x = (long)blockIdx.x * blockDim.x + threadIdx.x; x < dv;
       x += stride) {
    fvec<VW> colv[NMAX];
#pragma unroll
    for (int i = 0; i < NMAX; ++i) {
      if (i >= n) continue;
      colv[i] = reinterpret_cast<const fvec<VW>*>(g + (long)i * d)[x];
    }
    fvec<VW> res;
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      float inters[NMAX];
#pragma unroll
      for (int k = 0; k < NMAX; ++k) {
        if (k >= t) continue;
        unsigned mlo = mkv32[2 * k], mhi = mkv32[2 * k + 1];
        asm volatile("" : "+v"(mlo), "+v"(mhi));
        const unsigned long long m = ((unsigned long long)mhi << 32) | mlo;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) {
          if (i >= n) continue;
          if ((m >> i) & 1) s += colv[i].v[c];
        }
        inters[k] = s * inv[k];
      }
      res.v[c] = coord_averaged_median<NMAX>(inters, t, b);
    }
    reinterpret_cast<fvec<VW>*>(out)[x] = res;
  }
  long tail0 = dv * VW;
  if (blockIdx.x == 0 && threadIdx.x < (int)(d - tail0)) {
    long x = tail0 + threadIdx.x;
    float inters[NMAX];
#pragma unroll
    for (int k = 0; k < NMAX; ++k) {
      if (k >= t) continue;
      unsigned mlo = mkv32[2 * k], mhi = mkv32[2 * k + 1];
      asm volatile("" : "+v"(mlo), "+v"(mhi));
      const unsigned long long m = ((unsigned long long)mhi << 32) | mlo;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NMAX; ++i) {
        if (i >= n) continue;
        if ((m >> i) & 1) s += g[(long)i * d + x];
      }
      inters[k] = s * inv[k];
    }
    out[x] = coord_averaged_median<NMAX>(inters, t, b);
  }
}

__global__ void bulyan_inv_mk_kernel(float* inv_mk, int t, int m) {
  int k = threadIdx.x;
  if (k < t) inv_mk[k] = 1.f / (float)(m - k);
}

void bulyan_final(const float* g, int n, long d, int f, int m,
                  const unsigned char* flags, float* out,
                  hipStream_t stream) {
  const int t = n - 2 * f - 2;
  const int b = t - 2 * f;
  // Small helper buffer for 1/(m-k): lives at the end of the flags buffer?
  // Simpler: compute on the fly in a tiny kernel into a static buffer is not
  // graph-safe; instead reuse the flags allocation convention: the caller
  // allocates flags of t*n bytes PLUS t floats (aligned) right after.
  float* inv_mk = reinterpret_cast<float*>(
      const_cast<unsigned char*>(flags) + ((t * n + 15) & ~15));
  bulyan_inv_mk_kernel<<<1, 64, 0, stream>>>(inv_mk, t, m);
  int nblk = nblocks_d(d);
  int vw = vec_width(d);
  if (vw > 4) vw = 4;  // register balance
  if (n > 16 && vw > 2) vw = 2;  // NMAX=32 @ VW=4 spills to scratch
  long dv = d / vw;
#define GAR_BULYAN_LAUNCH(NMAX, VW)                                   \
  bulyan_final_kernel<NMAX, VW><<<nblk, kBlock, 0, stream>>>(         \
      g, out, dv, d, n, t, b, flags, inv_mk)
  if (n <= 8) {
    if (vw == 4) GAR_BULYAN_LAUNCH(8, 4);
    else if (vw == 2) GAR_BULYAN_LAUNCH(8, 2);
    else GAR_BULYAN_LAUNCH(8, 1);
  } else if (n <= 16) {
    if (vw == 4) GAR_BULYAN_LAUNCH(16, 4);
    else if (vw == 2) GAR_BULYAN_LAUNCH(16, 2);
    else GAR_BULYAN_LAUNCH(16, 1);
  } else {
    if (vw == 4) GAR_BULYAN_LAUNCH(kMaxNCoord, 4);
    else if (vw == 2) GAR_BULYAN_LAUNCH(kMaxNCoord, 2);
    else GAR_BULYAN_LAUNCH(kMaxNCoord, 1);
  }
#undef GAR_BULYAN_LAUNCH
}

}  // namespace gar
