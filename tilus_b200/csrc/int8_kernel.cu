// Matrix product in 8-bit integers with a scale per row of A (token) and per row of B (channel):
//
//   C[m, n] = round16( sum_k A[m, k] B[n, k] * a_sf[m] * b_sf[n] + bias[n] )              A [M, K], B [N, K] int8
//   gated:    with g, u = the products with rows n and N + n of B[2N, K], both scaled,
//   C[m, n] = round16( g / (1 + exp(-g)) * u )                                            (g, u clamped if asked for)
//
// The sums are exact: int32 in tensor memory, |sum| <= 128 * 128 * K < 2^31 for K <= 131056.  So neither the order of the
// sums nor a split of K changes a result; what is rounded is the sum's conversion to fp32 (past 2^24), its two or three
// fp32 products and the output.
//
// Both operands are K-major as they come (rows of 128 bytes, 128-byte swizzle); TMA fills what lies behind the last row
// or the end of K with zeros, so ragged sizes cost no code in the main loops.
//
// Two kernels:
//   pair    two CTAs per 256 x 256 tile (gated: 256 x 128, the gate columns in one CTA's half of B and their partners in
//           the other's), tcgen05.mma with cta_group::2, accumulators double-buffered in tensor memory so that a tile's
//           epilogue runs under the next one's products.  For many rows: bound by the tensor cores.
//   stream  up to 256 rows: 128 rows of B are the tensor core's M side and all rows of A its N side, so that B is
//           read once; the CTAs of a cluster share K and add their exact int32 sums in distributed shared memory.  For few
//           rows: bound by reading B.
//
// Both are launched with programmatic stream serialization: they set up under the end of the kernel before them, and read nothing
// of the caller's before that kernel has ended (either operand may be its output).
#include "int8.cuh"
#include "umma_common.cuh"

namespace b200q {

// instruction descriptor of kind::i8: D int32 (bits 4-5: 2), A and B signed (bits 7-9, 10-12: 1), both K-major
__host__ __device__ constexpr uint32_t int8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {  // a shared-memory address in another CTA of the cluster
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// one output: a 32-bit sum with its scales
__device__ __forceinline__ float scaled(uint32_t sum, float sa, float sb) { return __int2float_rn((int)sum) * sa * sb; }
__device__ __forceinline__ float gated_product(float g, float u, int use_clamp, float clamp) {
  if (use_clamp) {  // (comparisons, so that NaN stays NaN)
    g = g > clamp ? clamp : g;
    u = u > clamp ? clamp : u;
    u = u < -clamp ? -clamp : u;
  }
  return __fdividef(g, 1.0f + __expf(-g)) * u;
}
__device__ __forceinline__ uint32_t pack_act(int act, float lo, float hi) { return act == 0 ? pack2<0>(lo, hi) : pack2<1>(lo, hi); }
__device__ __forceinline__ float act_value(int act, unsigned short bits) {
  return act == 0 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
}

// ---- pair kernel ------------------------------------------------------------------------------------------
constexpr int P_STAGES = 6;            // 128 rows of A and 128 of B per CTA and stage
constexpr int P_STAGE = 32768;
constexpr int P_STORE = 16384;         // 128 rows x 64 columns on their way out, two of them
constexpr int P_THREADS = 256;         // copies, products, tensor memory, spare; four warps that write the outputs
struct PairBars {
  uint64_t full[P_STAGES], empty[P_STAGES], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
};
constexpr int P_SCALES = 256 * 4 + 256 * 2;  // a tile's column scales and biases
int int8_pair_smem_bytes() { return 1024 + P_STAGES * P_STAGE + 2 * P_STORE + P_SCALES + (int)sizeof(PairBars); }

// Output tile `t`: raster groups of m_group row tiles, row tile fastest, so that the clusters that run together share columns of B
// while a group's rows of A stay in L2.
__device__ __forceinline__ void pair_tile(const Int8Params& p, int t, int* m_tile, int* n_tile) {
  const int per = p.m_group * p.n_tiles, grp = t / per, in = t - grp * per;
  const int size = min(p.m_group, p.m_tiles - grp * p.m_group);
  *n_tile = in / size;
  *m_tile = grp * p.m_group + in - *n_tile * size;
}

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P_THREADS, 1)
    int8_pair_kernel(const Int8Params p, const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                     const __grid_constant__ CUtensorMap tc) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  unsigned char* base = smem_raw + (ring - raw);
  const uint32_t store_s = ring + P_STAGES * P_STAGE;
  float* col_sf = reinterpret_cast<float*>(base + P_STAGES * P_STAGE + 2 * P_STORE);
  unsigned short* col_bias = reinterpret_cast<unsigned short*>(col_sf + 256);
  const uint32_t bars_off = P_STAGES * P_STAGE + 2 * P_STORE + P_SCALES;
  PairBars* bars = reinterpret_cast<PairBars*>(base + bars_off);
  const uint32_t bars_s = ring + bars_off;
#define BAR(field, i) (bars_s + (uint32_t)offsetof(PairBars, field) + (uint32_t)(i) * 8u)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  volatile int* abort_flag = &bars->abort_flag;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < P_STAGES; ++i) { mbar_init(BAR(full, i), 1); mbar_init(BAR(empty, i), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(BAR(acc_full, i), 1); mbar_init(BAR(acc_empty, i), 8); }
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     bars_s + (uint32_t)offsetof(PairBars, tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == 0) {
    // ---- copies: this CTA's half of both operands; both halves report to the first CTA's barrier ----
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool good = true;
      for (int t = first; t < p.tiles && good; t += step) {
        int m_tile, n_tile;
        pair_tile(p, t, &m_tile, &n_tile);
        const int row = m_tile * 256 + (int)rank * 128;
        const int col = GATED ? n_tile * 128 + (int)rank * p.N : n_tile * 256 + (int)rank * 128;
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait_abortable(BAR(empty, s), phase ^ 1u, abort_flag)) { good = false; break; }
          if (rank == 0) expect_bytes(BAR(full, s), 2u * P_STAGE);
          const uint32_t bar = map_to(BAR(full, s), 0), dst = ring + (uint32_t)s * P_STAGE;
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
              ::"r"(dst), "l"(&ta), "r"(bar), "r"(kb * 128), "r"(row) : "memory");
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
              ::"r"(dst + 16384u), "l"(&tb), "r"(bar), "r"(kb * 128), "r"(col) : "memory");
          ++issued;
          if (++s == P_STAGES) { s = 0; phase ^= 1u; }
        }
      }
      // Having given up: the copies in flight land before the CTA ends (both CTAs' count on the first one's barriers, and the
      // second CTA waits for the first at the end).
      if (*abort_flag && rank == 0) ring_drain(BAR(full, 0), P_STAGES, issued);
    }
  } else if (warp == 1) {
    // ---- products, issued by the first CTA for both ----
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = int8_idesc(256, 256);
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool good = true;
      for (int t = first; t < p.tiles && good; t += step, ++it) {
        const int acc = it & 1;
        if (!mbar_wait_abortable(BAR(acc_empty, acc), ((uint32_t)(it >> 1) & 1u) ^ 1u, abort_flag)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait_abortable(BAR(full, s), phase, abort_flag)) { good = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t ad = umma_smem_desc(ring + (uint32_t)s * P_STAGE), bd = umma_smem_desc(ring + (uint32_t)s * P_STAGE + 16384u);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                ::"r"(tmem + (uint32_t)(acc * 256)), "l"(ad + (uint64_t)(ks * 2)), "l"(bd + (uint64_t)(ks * 2)), "r"(idesc),
                "r"((kb > 0 || ks > 0) ? 1u : 0u)
                : "memory");
          asm volatile(
              "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                  BAR(empty, s)), "h"((unsigned short)3)
              : "memory");
          if (++s == P_STAGES) { s = 0; phase ^= 1u; }
        }
        if (good)
          asm volatile(
              "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                  BAR(acc_full, acc)), "h"((unsigned short)3)
              : "memory");
      }
    }
  } else if (warp >= 4) {
    // ---- outputs: thread = row of the CTA's 128, 64 columns at a time through shared memory ----
    const int ew = warp & 3, r = ew * 32 + lane, et = tid - 128;
    const uint32_t lane_addr = tmem + ((uint32_t)(ew * 32) << 16);
    const uint32_t empty0 = map_to(BAR(acc_empty, 0), 0);
    int it = 0, buf = 0;
    for (int t = first; t < p.tiles; t += step, ++it) {
      int m_tile, n_tile;
      pair_tile(p, t, &m_tile, &n_tile);
      const int row0 = m_tile * 256 + (int)rank * 128, row = row0 + r;
      const int n0 = n_tile * (GATED ? 128 : 256);
      // 256 columns of the product: gated, 128 gates and their 128 partners
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = et + 128 * h, n = GATED ? n0 + et : n0 + i;
        col_sf[i] = n < p.N ? p.b_sf[GATED ? n + h * p.N : n] : 0.f;
        if (!GATED && p.bias) col_bias[i] = n < p.N ? p.bias[n] : (unsigned short)0;
      }
      const float sa = row < p.M ? p.a_sf[row] : 0.f;
      const int acc = it & 1;
      const bool ok = mbar_wait_abortable(BAR(acc_full, acc), (uint32_t)(it >> 1) & 1u, abort_flag);
      // (one thread's patience may end where another's did not: the four warps give up together)
      int bad;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(bad) : "r"(ok ? 0 : 1) : "memory");
      if (bad) break;
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      constexpr int CHUNKS = GATED ? 2 : 4;
#pragma unroll 1
      for (int j = 0; j < CHUNKS; ++j, buf ^= 1) {
        // the copy that read this buffer two chunks ago has done so
        if (et == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const uint32_t row_s = store_s + (uint32_t)buf * P_STORE + (uint32_t)r * 128u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c0 = j * 64 + h * 32;
          uint32_t v[32], o[16];
          tmem_ld_32(lane_addr + (uint32_t)(acc * 256 + c0), v);
          if constexpr (GATED) {
            uint32_t u[32];
            tmem_ld_32(lane_addr + (uint32_t)(acc * 256 + 128 + c0), u);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 sg = *reinterpret_cast<const float2*>(col_sf + c0 + 2 * i);
              const float2 su = *reinterpret_cast<const float2*>(col_sf + 128 + c0 + 2 * i);
              o[i] = pack_act(p.act, gated_product(scaled(v[2 * i], sa, sg.x), scaled(u[2 * i], sa, su.x), p.use_clamp, p.clamp),
                              gated_product(scaled(v[2 * i + 1], sa, sg.y), scaled(u[2 * i + 1], sa, su.y), p.use_clamp, p.clamp));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 sb = *reinterpret_cast<const float2*>(col_sf + c0 + 2 * i);
              float lo = scaled(v[2 * i], sa, sb.x), hi = scaled(v[2 * i + 1], sa, sb.y);
              if (p.bias) {
                lo += act_value(p.act, col_bias[c0 + 2 * i]);
                hi += act_value(p.act, col_bias[c0 + 2 * i + 1]);
              }
              o[i] = pack_act(p.act, lo, hi);
            }
          }
          if (j == CHUNKS - 1 && h == 1) {  // the accumulators are in registers: the next but one tile may have them
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
              asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(empty0 + (uint32_t)acc * 8u) : "memory");
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)  // 16-byte pieces, swizzled as the tensor map says
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_s + (uint32_t)(((h * 4 + q) ^ (r & 7)) * 16)),
                         "r"(o[4 * q]), "r"(o[4 * q + 1]), "r"(o[4 * q + 2]), "r"(o[4 * q + 3]) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (et == 0) {
          const int n = n0 + j * 64;
          if (n < p.N && row0 < p.M)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&tc),
                         "r"(store_s + (uint32_t)buf * P_STORE), "r"(n), "r"(row0) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // (an empty group where nothing was stored: the count stays)
        }
      }
    }
    if (et == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag && tid == 0) {
    atomicExch(p.status, ST_DEVICE_TIMEOUT);
    p.status[1] = 12;  // where: pair kernel
    p.status[2] = blockIdx.x;
    p.status[3] = 0;
  }
  cluster_sync();  // neither CTA's shared memory or tensor memory goes while the other still uses it
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
#undef BAR
}

// ---- stream kernel ----------------------------------------------------------------------------------------
constexpr int S_THREADS = 128;
constexpr int S_STAGES_MAX = 12;
struct StreamBars {
  uint64_t full[S_STAGES_MAX], empty[S_STAGES_MAX], done;
  uint32_t tmem_base;
  int abort_flag;
};
static __host__ __device__ int stream_ring_bytes(int rows, int stages) {
  // (the ring's memory takes the int32 sums afterwards: rows x 128)
  const int ring = stages * (16384 + rows * 128), sums = rows * 512;
  return ring > sums ? ring : sums;
}
int int8_stream_smem_bytes(int rows, int stages) { return 1024 + stream_ring_bytes(rows, stages) + (int)sizeof(StreamBars); }

template <bool GATED>
__global__ void __launch_bounds__(S_THREADS)
    int8_stream_kernel(const Int8Params p, const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  unsigned char* base = smem_raw + (ring - raw);
  const uint32_t bars_off = (uint32_t)stream_ring_bytes(p.rows, p.stages);
  StreamBars* bars = reinterpret_cast<StreamBars*>(base + bars_off);
  const uint32_t bars_s = ring + bars_off;
#define BAR(field, i) (bars_s + (uint32_t)offsetof(StreamBars, field) + (uint32_t)(i) * 8u)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile int* abort_flag = &bars->abort_flag;
  const int S = p.cluster;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int tile = S > 1 ? blockIdx.x / S : blockIdx.x;
  const int kb0 = (int)((long long)p.kblocks * rank / S), kb1 = (int)((long long)p.kblocks * (rank + 1) / S);
  const uint32_t a_bytes = (uint32_t)p.rows * 128u, stage_bytes = 16384u + a_bytes;
  const uint32_t cols = p.rows <= 32 ? 32u : p.rows <= 64 ? 64u : p.rows <= 128 ? 128u : 256u;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) { mbar_init(BAR(full, i), 1); mbar_init(BAR(empty, i), 1); }
    mbar_init(BAR(done, 0), 1);
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     bars_s + (uint32_t)offsetof(StreamBars, tmem_base)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == 0) {
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_abortable(BAR(empty, s), phase ^ 1u, abort_flag)) break;
        const uint32_t bar = BAR(full, s), dst = ring + (uint32_t)s * stage_bytes;
        expect_bytes(bar, stage_bytes);
        if constexpr (GATED) {  // 64 gates, then their 64 partners
          for (int h = 0; h < 2; ++h)
            asm volatile(
                "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                ::"r"(dst + (uint32_t)h * 8192u), "l"(&tb), "r"(bar), "r"(kb * 128), "r"(tile * 64 + h * p.N) : "memory");
        } else {
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
              ::"r"(dst), "l"(&tb), "r"(bar), "r"(kb * 128), "r"(tile * 128) : "memory");
        }
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst + 16384u), "l"(&ta), "r"(bar), "r"(kb * 128), "r"(0) : "memory");
        ++issued;
        if (++s == p.stages) { s = 0; phase ^= 1u; }
      }
      if (*abort_flag) ring_drain(BAR(full, 0), p.stages, issued);  // the copies in flight land before the CTA ends
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = int8_idesc(128, p.rows);
      int s = 0;
      uint32_t phase = 0;
      bool good = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_abortable(BAR(full, s), phase, abort_flag)) { good = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t wd = umma_smem_desc(ring + (uint32_t)s * stage_bytes), xd = umma_smem_desc(ring + (uint32_t)s * stage_bytes + 16384u);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          asm volatile(
              "{\n\t.reg .pred p;\n\t"
              "setp.ne.b32 p, %4, 0;\n\t"
              "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
              ::"r"(tmem), "l"(wd + (uint64_t)(ks * 2)), "l"(xd + (uint64_t)(ks * 2)), "r"(idesc), "r"((kb > kb0 || ks > 0) ? 1u : 0u)
              : "memory");
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(BAR(empty, s)) : "memory");
        if (++s == p.stages) { s = 0; phase ^= 1u; }
      }
      if (good)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(BAR(done, 0)) : "memory");
    }
    __syncwarp();
  }
  // Every product has read its operands: the ring's memory takes the sums, [row of A][128 rows of B].
  const bool ok = mbar_wait_abortable(BAR(done, 0), 0, abort_flag);
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  __syncwarp();
  if (__all_sync(0xffffffffu, ok)) {
    const uint32_t mine = ring + (uint32_t)(warp * 32 + lane) * 4u;
    for (int c0 = 0; c0 < p.rows; c0 += 16) {
      uint32_t v[16];
      tmem_ld_16(tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)c0, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) asm volatile("st.shared.b32 [%0], %1;" ::"r"(mine + (uint32_t)(c0 + i) * 512u), "r"(v[i]) : "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if (S > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  }
  // The cluster's CTAs share the outputs: four columns of a row each time.
  constexpr int QUADS = GATED ? 16 : 32;
  const int n0 = tile * (4 * QUADS);
  for (int i = rank * S_THREADS + tid; i < p.M * QUADS; i += S * S_THREADS) {
    const int m = i / QUADS, q = i % QUADS, n = n0 + 4 * q;
    if (n >= p.N) continue;
    int4 x = make_int4(0, 0, 0, 0), y = make_int4(0, 0, 0, 0);
    const uint32_t at = ring + (uint32_t)m * 512u + (uint32_t)q * 16u;
    for (int c = 0; c < S; ++c) {
      const uint32_t from = S > 1 ? map_to(at, (uint32_t)c) : at;
      int4 w;
      asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(from));
      x.x += w.x; x.y += w.y; x.z += w.z; x.w += w.w;
      if constexpr (GATED) {
        asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(from + 256u));
        y.x += w.x; y.y += w.y; y.z += w.z; y.w += w.w;
      }
    }
    const float sa = p.a_sf[m];
    const float4 sb = *reinterpret_cast<const float4*>(p.b_sf + n);
    float o[4] = {scaled((uint32_t)x.x, sa, sb.x), scaled((uint32_t)x.y, sa, sb.y), scaled((uint32_t)x.z, sa, sb.z),
                  scaled((uint32_t)x.w, sa, sb.w)};
    if constexpr (GATED) {
      const float4 su = *reinterpret_cast<const float4*>(p.b_sf + p.N + n);
      o[0] = gated_product(o[0], scaled((uint32_t)y.x, sa, su.x), p.use_clamp, p.clamp);
      o[1] = gated_product(o[1], scaled((uint32_t)y.y, sa, su.y), p.use_clamp, p.clamp);
      o[2] = gated_product(o[2], scaled((uint32_t)y.z, sa, su.z), p.use_clamp, p.clamp);
      o[3] = gated_product(o[3], scaled((uint32_t)y.w, sa, su.w), p.use_clamp, p.clamp);
    } else if (p.bias) {
      const ushort4 b = *reinterpret_cast<const ushort4*>(p.bias + n);
      o[0] += act_value(p.act, b.x); o[1] += act_value(p.act, b.y); o[2] += act_value(p.act, b.z); o[3] += act_value(p.act, b.w);
    }
    if (*abort_flag == 0)
      *reinterpret_cast<uint2*>(p.c + (size_t)m * p.ldc + n) = make_uint2(pack_act(p.act, o[0], o[1]), pack_act(p.act, o[2], o[3]));
  }
  if (*abort_flag && tid == 0) {
    atomicExch(p.status, ST_DEVICE_TIMEOUT);
    p.status[1] = 13;  // where: stream kernel
    p.status[2] = blockIdx.x;
    p.status[3] = 0;
  }
  if (S > 1) cluster_sync();  // nobody's sums go while another CTA reads them
#undef BAR
}

// ---- launches -----------------------------------------------------------------------------------------------
template <class Kernel, class... Args>
static cudaError_t launch_behind(Kernel kern, int grid, int threads, int cluster, int smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <bool GATED>
static cudaError_t pair_launch(const Int8Params& p, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, int grid,
                               cudaStream_t stream) {
  static std::atomic<bool> allowed[16];
  const cudaError_t e = allow_smem(int8_pair_kernel<GATED>, allowed);
  if (e != cudaSuccess) return e;
  return launch_behind(int8_pair_kernel<GATED>, grid, P_THREADS, 1, int8_pair_smem_bytes(), stream, p, ta, tb, tc);
}
template <bool GATED>
static cudaError_t stream_launch(const Int8Params& p, const CUtensorMap& ta, const CUtensorMap& tb, cudaStream_t stream) {
  static std::atomic<bool> allowed[16];
  const cudaError_t e = allow_smem(int8_stream_kernel<GATED>, allowed);
  if (e != cudaSuccess) return e;
  return launch_behind(int8_stream_kernel<GATED>, p.tiles * p.cluster, S_THREADS, p.cluster, int8_stream_smem_bytes(p.rows, p.stages),
                       stream, p, ta, tb);
}

cudaError_t int8_pair_launch(const Int8Params& p, bool gated, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc,
                             int grid, cudaStream_t stream) {
  return gated ? pair_launch<true>(p, ta, tb, tc, grid, stream) : pair_launch<false>(p, ta, tb, tc, grid, stream);
}
cudaError_t int8_stream_launch(const Int8Params& p, bool gated, const CUtensorMap& ta, const CUtensorMap& tb, cudaStream_t stream) {
  return gated ? stream_launch<true>(p, ta, tb, stream) : stream_launch<false>(p, ta, tb, stream);
}

}  // namespace b200q
