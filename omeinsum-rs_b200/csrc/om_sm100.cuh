// Tensor-core product D[m, n] = sum_k A[m, k] B[n, k] of 16-bit or 8-bit
// operands on sm_100a, with the caller's own epilogue.
//
// Persistent: each CTA (CG = 1) or pair of CTAs (CG = 2) takes tiles of
// 128 CG x BN round robin. 320 threads: warp 0 issues TMA loads of 128-byte
// deep k slabs into a ring of stages, warp 1 issues the MMAs
// (accumulators in tensor memory, two of them, so that one tile's epilogue
// runs under the next tile's products), warps 2..9 read a finished
// accumulator and hand it to the epilogue 32 columns at a time: warp w has the
// rows 32 (w % 4) .. + 31, one per lane, and every second group of columns.
//
// With CG = 2 two SMs share a tile: each holds its own 128 rows of A and half
// of B's rows, so a slab costs each SM 32 KiB of loads instead of 48 for the
// same 256 columns; the even CTA issues the MMAs of both.
//
// An operand is K-major (k contiguous) or MN-major (rows contiguous); both are
// read by TMA where they lie, with a 128-byte swizzle. TMA fills what lies
// outside the matrix with zeros, so no size needs padding.
//
// P3: operands of three bf16 planes each (x = x0 + x1 + x2 to 24 bits), six
// products per slab, the smallest first:
//     A2 B0 + A0 B2 + A1 B1 + A1 B0 + A0 B1 + A0 B0
// for sums as exact as f32's: what is left out is 2^-24 of a term. The tensor
// core does not round its running sum to nearest, so every CHUNK slabs are
// summed from zero and added up in the epilogue warps' registers. The planes
// of a slab are loaded once for all six.
//
// Without P3 an accumulator runs over all of k in f32. The tensor core cuts the
// running sum where it adds to it instead of rounding to nearest: up to 2^-23 of the
// sum for each 16 products (16 bits; sums of 8-bit integers are exact). Measured: lse
// of 24 x 2048 x 32000 in f16 is 4e-7 off 64 bits, 3e-8 by sums rounded to nearest.
//
// Bound by the tensor cores: 4096 x 1024 by 50001 x 1024 bf16 with the cross
// entropy's forward epilogue takes 257 us, 1.63 PFLOP/s with the tensor pipe 93 %
// active (the library product of the same size 293 us); 8192 x 4096 by 12288 x 4096
// in 8 bits 239 us, 3.4 POP/s, 92 %. Launches that follow one another for
// milliseconds run at the card's power limit, 1.36 PFLOP/s.
//
// Every wait is bounded; on expiry the kernel records an error word that
// om_b200_sync reports, and leaves after its other bounded waits.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "om_internal.h"

namespace om {

// cuTensorMapEncodeTiled, looked up once (null: not available)
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace mma {

constexpr int TM = 128;             // rows of a CTA's accumulator
constexpr int THREADS = 320;        // 2 + 8 warps
constexpr int MAX_STAGES = 12;
constexpr int SLAB = 128;           // bytes of k per stage
constexpr int CHUNK = 2;            // slabs of a sum (P3)
constexpr int A_BYTES = TM * SLAB;
constexpr uint32_t WAIT_LIMIT = 1u << 24;
// Shared memory that an epilogue asks for, per warp: for turning 32 rows of 32
// values (a word of padding each), or for two boxes of 32 x 32 16-bit results
// that TMA stores.
constexpr int TURN_BYTES = 32 * 33 * 4, BOX_BYTES = 32 * 32 * 2;

struct Shape {
  int M, N;        // rows of A and of B
  int slabs;       // of 128 bytes along k, all splits together
  int BN;          // columns of a tile: 32 .. 256, a multiple of 32
  int stages;
  int a_rows;      // rows of A's box: 128, or fewer where all of A has fewer
  int lent;        // bytes of shared memory lent to each epilogue warp
  int tiles_m, tiles_n, splits;
  int group;       // row tiles that are walked before the next column tile
  uint32_t idesc;  // instruction descriptor
  uint32_t* err;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}

__device__ __forceinline__ uint32_t in_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void load_box3(uint32_t dst, const CUtensorMap* map, int x, int y,
                                          int z, uint32_t bar, int cg) {
  if (cg == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else  // the barrier may lie in the other CTA of the pair
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// 128-byte swizzled operand at a shared-memory address. K-major: 8-row groups
// 1024 bytes apart, the next MMA's k 32 bytes on. MN-major: 64 rows x 8 k take
// 1024 bytes, the next 8 k follow, the next 64 rows lie 64 k further (8192
// bytes); the next MMA's k is 2048 bytes on. Addresses are below 2^18, so moving
// on is an addition to the low word.
template <bool MN>
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  constexpr uint32_t lead = MN ? 8192 >> 4 : 1, high = (1024 >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)high << 32) | ((lead << 16) + (addr >> 4));
}
template <bool MN>
__device__ __forceinline__ uint64_t next_k(uint64_t op, int j) {
  return op + (uint64_t)(j * (MN ? 2048 >> 4 : 32 >> 4));
}

// One lane of a converged warp. Loads and MMAs are issued by loops that the
// whole warp runs, so that their operands are computed once in the uniform
// registers that the instructions take them from: a loop of one lane's moves
// them there one by one, 190 cycles per MMA of 128.
__device__ __forceinline__ bool elected() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait(bar, parity));
}

template <bool I8, int CG>
__device__ __forceinline__ void issue(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                      uint32_t acc) {
#define OM_MMA(KIND, GROUP)                                        \
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"         \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND      \
               " [%0], %1, %2, %3, p;\n}\n" ::"r"(d),              \
               "l"(a), "l"(b), "r"(idesc), "r"(acc))
  if constexpr (I8) {
    if constexpr (CG == 1) OM_MMA("i8", "1");
    else OM_MMA("i8", "2");
  } else {
    if constexpr (CG == 1) OM_MMA("f16", "1");
    else OM_MMA("f16", "2");
  }
#undef OM_MMA
}

// arrives on the barrier (of both CTAs of a pair) when the MMAs issued so far
// are done
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}

__device__ __forceinline__ void read_columns(uint32_t addr, uint32_t (&x)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]),
        "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]),
        "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]),
        "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]),
        "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// What a warp's epilogue has been lent, and how many boxes it has stored from it
struct Lent {
  float* words;
  int boxes = 0;
};

// A 32 x 32 box of 16-bit results (row by lane, 64 bytes each) to (x, y) of a
// map made by encode_result: written to shared memory with the map's 64-byte
// swizzle, two boxes in turn, and stored by TMA, which leaves out what lies
// outside the matrix. (Lanes storing their own row touch 32 lines with each
// instruction, which took longer than the products of a few slabs.)
__device__ __forceinline__ void store_box(Lent& lent, const CUtensorMap* map, const uint32_t (&u)[16],
                                          int x, int y) {
  const int lane = threadIdx.x & 31;
  char* box = reinterpret_cast<char*>(lent.words) + (lent.boxes & 1) * BOX_BYTES;
  if (lent.boxes >= 2) {  // the box's last store has read it
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     (uint64_t)map),
                 "r"(x), "r"(y), "r"(smem_addr(box))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
  ++lent.boxes;
}

// the k slabs of split s: [first, last)
__device__ __forceinline__ int slab_at(const Shape& g, int s) {
  return (int)((int64_t)g.slabs * s / g.splits);
}

struct Tile {
  int m, n, split;
};
__device__ __forceinline__ Tile tile_at(const Shape& g, int t) {
  const int per = g.tiles_m * g.tiles_n;
  Tile r;
  r.split = t / per;
  t -= r.split * per;
  const int band = g.group * g.tiles_n, b = t / band, first = b * g.group;
  const int rows = min(g.group, g.tiles_m - first);
  t -= b * band;
  r.m = first + t % rows;
  r.n = t / rows;
  return r;
}

// Epi, per lane and tile: Row begin(m, in, split) before the accumulator is
// read; columns(row, m, in, n0, N, values, lent) for each 32 columns from n0 on,
// by whole warps; and end(row, m, in, slot) with slot = 2 * column tile + column
// group. `in`: row m exists; columns from N on do not. `lent`: shared memory of
// the warp's own, as much as lent_bytes() says.
template <bool I8, bool P3, bool AMN, bool BMN, int CG, class Epi>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                   const __grid_constant__ Shape g, const __grid_constant__ Epi epi) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // the same offset in both CTAs of a pair: the dynamic base is the same
  const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;
  __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[2], tempty[2];
  __shared__ uint32_t tmem_base;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  uint32_t rank = 0;
  if constexpr (CG == 2) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  const int tiles = g.tiles_m * g.tiles_n * g.splits;
  const int b_rows = g.BN / CG;  // of B that this CTA loads
  constexpr int PLANES = P3 ? 3 : 1;
  const uint32_t b_bytes = b_rows * SLAB;
  const uint32_t stage_bytes = PLANES * (A_BYTES + b_bytes);
  const uint32_t loaded = PLANES * ((AMN ? TM : g.a_rows) * SLAB + b_bytes);
  const int kstep = I8 ? 128 : 64;  // elements of a slab

  if (warp == 1) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
          smem_addr(&tmem_base)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
          smem_addr(&tmem_base)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  if (tid == 0) {
    for (int s = 0; s < g.stages; ++s) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(&full[s])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(&empty[s])));
    }
    for (int b = 0; b < 2; ++b) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(&tfull[b])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(&tempty[b])),
                   "r"(8 * CG));
    }
    asm volatile("fence.mbarrier_init.release.cluster;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
  bool ok = true;

  if (warp == 0) {  // loads
    int q = 0, s = 0;
    uint32_t phase = 1;  // of empty[s]: passes at once on the first round
    for (int t = first; t < tiles && ok; t += step) {
      const Tile at = tile_at(g, t);
      const int m0 = (at.m * CG + (int)rank) * TM;
      const int n0 = at.n * g.BN + (int)rank * b_rows;
      const int k1 = slab_at(g, at.split + 1);
      for (int k = slab_at(g, at.split); k < k1; ++k, ++q) {
        if (q >= g.stages) ok = wait_all(smem_addr(&empty[s]), phase);
        if (!ok) break;
        uint32_t bar = smem_addr(&full[s]);
        const uint32_t a = ring + s * stage_bytes, b = a + PLANES * A_BYTES;
        if (elected()) {
          if (CG == 1 || rank == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                         "r"(loaded * CG)
                         : "memory");
          if constexpr (CG == 2) bar = in_rank(bar, 0);
          if constexpr (P3) {
            for (int z = 0; z < 3; ++z) {
              if constexpr (AMN) {
                for (int i = 0; i < TM; i += 64)
                  load_box3(a + z * A_BYTES + i * SLAB, &amap, m0 + i, k * kstep, z, bar, CG);
              } else {
                load_box3(a + z * A_BYTES, &amap, k * kstep, m0, z, bar, CG);
              }
              if constexpr (BMN) {
                for (int i = 0; i < b_rows; i += 64)
                  load_box3(b + z * b_bytes + i * SLAB, &bmap, n0 + i, k * kstep, z, bar, CG);
              } else {
                load_box3(b + z * b_bytes, &bmap, k * kstep, n0, z, bar, CG);
              }
            }
          } else {
            if constexpr (AMN) {
              for (int i = 0; i < TM; i += 64) load_box<CG>(a + i * SLAB, &amap, m0 + i, k * kstep, bar);
            } else {
              load_box<CG>(a, &amap, k * kstep, m0, bar);
            }
            if constexpr (BMN) {
              for (int i = 0; i < b_rows; i += 64)
                load_box<CG>(b + i * SLAB, &bmap, n0 + i, k * kstep, bar);
            } else {
              load_box<CG>(b, &bmap, k * kstep, n0, bar);
            }
          }
        }
        __syncwarp();
        if (++s == g.stages) s = 0, phase ^= 1;
      }
    }
    if (!ok && lane == 0) atomicOr(g.err, 1u);
    // nothing of the last round is in flight when the block leaves: the
    // stages' products are done, or (after an expired wait) their copies in
    for (int j = max(0, q - g.stages); j < q; ++j) {
      uint64_t* bar = ok ? empty : full;
      if (ok || rank == 0) wait(smem_addr(&bar[j % g.stages]), (j / g.stages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {  // products
      int s = 0, i = 0;
      uint32_t phase = 0;
      for (int t = first; t < tiles && ok; t += step) {
        const Tile at = tile_at(g, t);
        const int k0 = slab_at(g, at.split), k1 = slab_at(g, at.split + 1);
        for (int k = k0; k < k1; ++k) {
          const bool fresh = P3 ? (k - k0) % CHUNK == 0 : k == k0;  // an accumulator starts here
          if (fresh) {
            if (i >= 2) ok = wait_all(smem_addr(&tempty[i & 1]), ((i >> 1) - 1) & 1);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;");
          }
          ok = wait_all(smem_addr(&full[s]), phase);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;");
          const uint32_t d = tmem + (i & 1) * 256, at_a = ring + s * stage_bytes;
          const bool done = k + 1 == k1 || (P3 && (k + 1 - k0) % CHUNK == 0);
          if (elected()) {
            if constexpr (P3) {
              constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
              for (int p = 0; p < 6; ++p) {
                const uint64_t a = operand<AMN>(at_a + PA[p] * A_BYTES);
                const uint64_t b = operand<BMN>(at_a + 3 * A_BYTES + PB[p] * b_bytes);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  issue<I8, CG>(d, next_k<AMN>(a, j), next_k<BMN>(b, j), g.idesc, !fresh || p > 0 || j > 0);
              }
            } else {
              const uint64_t a = operand<AMN>(at_a), b = operand<BMN>(at_a + A_BYTES);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                issue<I8, CG>(d, next_k<AMN>(a, j), next_k<BMN>(b, j), g.idesc, !fresh || j > 0);
            }
            commit<CG>(smem_addr(&empty[s]));
            if (done) commit<CG>(smem_addr(&tfull[i & 1]));
          }
          __syncwarp();
          if (done) ++i;
          if (++s == g.stages) s = 0, phase ^= 1;
        }
      }
      if (!ok && lane == 0) atomicOr(g.err, 1u);
    }
    __syncwarp();
  } else {  // epilogue
    const int quad = warp & 3, part = (warp - 2) >> 2;
    Lent lent{reinterpret_cast<float*>(smem_raw + (ring - smem_addr(smem_raw)) +
                                       (size_t)g.stages * stage_bytes + (warp - 2) * g.lent)};
    int i = 0;
    auto release = [&](int ab) {  // the accumulator has been read
      asm volatile("tcgen05.fence::before_thread_sync;");
      __syncwarp();
      if (lane == 0) {
        uint32_t bar = smem_addr(&tempty[ab]);
        if constexpr (CG == 2) bar = in_rank(bar, 0);
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                     : "memory");
      }
    };
    for (int t = first; t < tiles && ok; t += step) {
      const Tile at = tile_at(g, t);
      const uint32_t base = tmem + ((uint32_t)(32 * quad) << 16);
      const int m = (at.m * CG + (int)rank) * TM + 32 * quad + lane;
      const bool in = m < g.M;
      typename Epi::Row row = epi.begin(m, in, at.split);
      if constexpr (P3) {  // BN <= 128: at most two groups of columns
        float sum[2][32];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < 32; ++c) sum[j][c] = 0.f;
        const int slabs = slab_at(g, at.split + 1) - slab_at(g, at.split);
        for (int k = 0; k < slabs; k += CHUNK, ++i) {
          ok = wait(smem_addr(&tfull[i & 1]), (i >> 1) & 1);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;");
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int c = part * 32 + j * 64;
            if (c >= g.BN) break;
            uint32_t r[32];
            read_columns(base + (i & 1) * 256 + c, r);
#pragma unroll
            for (int q = 0; q < 32; ++q) sum[j][q] += __uint_as_float(r[q]);
          }
          release(i & 1);
        }
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int c = part * 32 + j * 64;
          if (c >= g.BN) break;
          uint32_t r[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) r[q] = __float_as_uint(sum[j][q]);
          epi.columns(row, m, in, at.n * g.BN + c, g.N, r, lent);
        }
      } else {
        ok = wait(smem_addr(&tfull[i & 1]), (i >> 1) & 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;");
        for (int c = part * 32; c < g.BN; c += 64) {
          uint32_t r[32];
          read_columns(base + (i & 1) * 256 + c, r);
          epi.columns(row, m, in, at.n * g.BN + c, g.N, r, lent);
        }
        release(i & 1);
        ++i;
      }
      epi.end(row, m, in, at.n * 2 + part);
    }
    if (!ok && lane == 0) atomicOr(g.err, 1u);
    if (lent.boxes && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  if (warp == 1) {
    if constexpr (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---- host side ---------------------------------------------------------------

// A matrix operand: `rows` x `k` elements of 1 or 2 bytes; K-major: rows `ld`
// elements apart; MN-major: k steps `ld` apart.
struct Matrix {
  const void* ptr;
  int64_t rows, k, ld;
  int elem;
  int64_t plane = 0;  // elements between the three planes of P3
};

inline bool tma_readable(const void* ptr, int64_t ld, int elem) {
  return ((uintptr_t)ptr & 15) == 0 && ld > 0 && (ld * elem) % 16 == 0 &&
         ld * elem < ((int64_t)1 << 40);
}

inline int encode(CUtensorMap* map, const Matrix& x, bool mn, int box_rows) {
  auto fn = tensor_map_encoder();
  if (!fn) return set_error(OM_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
  const cuuint64_t dims[3] = {(cuuint64_t)(mn ? x.rows : x.k), (cuuint64_t)(mn ? x.k : x.rows), 3};
  const cuuint64_t strides[2] = {(cuuint64_t)(x.ld * x.elem), (cuuint64_t)(x.plane * x.elem)};
  const cuuint32_t box[3] = {(cuuint32_t)(SLAB / x.elem), (cuuint32_t)(mn ? SLAB / x.elem : box_rows), 1};
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = fn(map, x.elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                        x.plane ? 3 : 2, (void*)x.ptr, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(OM_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return OM_OK;
}

// The map that store_box stores 16-bit results through; rows 16-byte aligned
inline int encode_result(CUtensorMap* map, void* ptr, int64_t rows, int64_t cols, int64_t ld) {
  auto fn = tensor_map_encoder();
  if (!fn) return set_error(OM_ERR_CUDA, "cuTensorMapEncodeTiled not available from the driver");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(ld * 2)};
  const cuuint32_t box[2] = {32, 32}, one[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, ptr, dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(OM_ERR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return OM_OK;
}

// Instruction descriptor: accumulator format (f32 / s32), operand formats,
// which operands are MN-major, the tile's columns and rows.
inline uint32_t instruction(bool i8, bool bf16, bool amn, bool bmn, int rows, int cols) {
  const uint32_t d = i8 ? 2 : 1, fmt = i8 ? 1 : (bf16 ? 1 : 0);
  return (d << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)amn << 15) | ((uint32_t)bmn << 16) |
         ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(rows >> 4) << 24);
}

// Tile columns and whether a pair of CTAs shares a tile, from the result's size:
// pairs of 256 x `most` when they fill four fifths of the card, else the widest
// tile of one CTA that gives three quarters of the SMs one. (A pair's tile of
// 512 x 256, its two halves sharing B's slabs, saves a quarter of the loads but
// fills the tensor memory, so that its epilogue is half exposed: 294 us on 4096
// x 1024 by 50001 x 1024 with the loss's forward epilogue, this one 262.)
struct Tiling {
  int bn, pair;
};
// `odd` (B K-major, an epilogue that writes nothing outside the result): one row
// of tiles, which waits for B's bytes alone, gets the width in steps of 32 that
// gives every SM the same share of them (24 x 2048 x 32000 in f16: 143 tiles of
// 224 columns instead of 125 of 256).
inline Tiling tiling(const om_backend* be, int64_t M, int64_t N, int least, int most = 256, bool odd = false) {
  if (odd && M <= TM) {
    const int64_t waves = (N + (int64_t)be->num_sms * most - 1) / ((int64_t)be->num_sms * most);
    const int64_t share = (N + be->num_sms * waves - 1) / (be->num_sms * waves);
    return {(int)std::max<int64_t>(least, (share + 31) / 32 * 32), 0};
  }
  if (M > TM && (M + 255) / 256 * ((N + most - 1) / most) * 5 >= be->num_sms * 2) return {most, 1};
  const int64_t tm = (M + TM - 1) / TM;
  for (int bn = most; bn > least; bn /= 2)
    if (tm * ((N + bn - 1) / bn) * 4 >= be->num_sms * 3) return {bn, 0};
  return {least, 0};
}

// D = A B^T through `epi`. bn: tile columns (a multiple of 32 up to 256; of 64
// for an MN-major B); pair: two CTAs per tile (bn 128 or 256). splits > 1
// cuts k into that many ranges of whole slabs, each handed to the epilogue
// as its own tile. P3: bf16 planes (Matrix::plane), bn at most 128.
template <bool I8, bool P3, bool AMN, bool BMN, int CG, class Epi>
int launch_tiles(om_backend* be, const char* name, const Matrix& a, const Matrix& b, bool bf16,
                   int bn, int splits, const Epi& epi) {
  const int kstep = I8 ? 128 : 64;
  const int64_t tm = (a.rows + TM * CG - 1) / (TM * CG), tn = (b.rows + bn - 1) / bn;
  const int64_t slabs = (a.k + kstep - 1) / kstep;
  if (a.rows > 0x7fffff00 || b.rows > 0x7fffff00 || a.k > 0x7fffff00 || splits < 1 ||
      splits > slabs || tm * tn * splits > 0x7fffffff)
    return set_error(OM_ERR_SHAPE, std::string(name) + ": extents out of range");
  CUtensorMap ma, mb;
  // rows that A does not have need no copies of zeros: what an accumulator's
  // other rows hold is never stored
  const int a_rows = a.rows < TM && CG == 1 ? (int)((a.rows + 7) / 8 * 8) : TM;
  OM_TRY(encode(&ma, a, AMN, a_rows));
  OM_TRY(encode(&mb, b, BMN, bn / CG));
  Shape g{};
  g.M = (int)a.rows, g.N = (int)b.rows, g.slabs = (int)slabs, g.BN = bn;
  g.tiles_m = (int)tm, g.tiles_n = (int)tn, g.splits = splits;
  // a wave's tiles form a square of rows and columns, so that each slab is
  // read by many SMs while it is in L2
  g.group = std::max(1, std::min<int>((int)tm, 2048 / (TM * CG)));
  const int stage = (P3 ? 3 : 1) * (A_BYTES + bn / CG * SLAB);
  g.a_rows = a_rows;
  g.lent = epi.lent_bytes();
  g.stages = std::min(MAX_STAGES, (216 * 1024 - 8 * g.lent) / stage);
  g.idesc = instruction(I8, bf16, AMN, BMN, TM * CG, bn);
  g.err = be->d_flags + 1;
  const size_t smem = (size_t)g.stages * stage + 8 * g.lent + 1024;
  auto kernel = product_kernel<I8, P3, AMN, BMN, CG, Epi>;
  OM_TRY(allow_shared(be, (const void*)kernel, (int)smem, name));
  const int64_t work = tm * tn * splits;
  ProfScope prof(be, name);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(CG * std::min<int64_t>(work, be->num_sms / CG)));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = be->stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CG, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  OM_CUDA(cudaLaunchKernelEx(&cfg, kernel, ma, mb, g, epi), name);
  note_launch();
  return OM_OK;
}

template <bool I8, bool P3, bool AMN, bool BMN, class Epi>
int launch_product(om_backend* be, const char* name, const Matrix& a, const Matrix& b, bool bf16,
                   const Tiling& t, int splits, const Epi& epi) {
  if (t.pair) return launch_tiles<I8, P3, AMN, BMN, 2>(be, name, a, b, bf16, t.bn, splits, epi);
  return launch_tiles<I8, P3, AMN, BMN, 1>(be, name, a, b, bf16, t.bn, splits, epi);
}

}  // namespace mma
}  // namespace om
