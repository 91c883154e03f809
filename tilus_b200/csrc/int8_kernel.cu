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
// Three kernels:
//   pair    two CTAs per tile of 256 rows x 256 or 128 columns of the product (gated: the gate columns in one CTA's half of B and
//           their partners in the other's), tcgen05.mma with cta_group::2, accumulators double-buffered in tensor memory so that a tile's
//           epilogue runs under the next one's products.  For many rows: bound by the tensor cores.
//   stream  up to 256 rows, all of them against an equal share of the columns in each CTA, so that B is read once: bound by that.
//   row     up to 16 rows where the product is small: no pipeline to fill, mma.sync from registers.  Bound by the latency of its loads.
// On a B200, in a graph of such calls: pair, 4096 x 8192 x 8192, 162 us (3.40 POP/s, the tensor pipe busy 88 % of the time); 4096 x 28672
// x 8192 gated 541 to 642 us as the power limit has it (3.0 to 3.5 POP/s); stream, 8 x 28672 x 4096 gated 20.5 us (5.7 TB/s; 23.4 on
// GPUs that read slower), 64 x 28672 x 4096 gated 21.6 us; row, 1 x 4096 x 4096 5.0 us, 3.9 with B read early.
//
// All are launched with programmatic stream serialization: they set up under the end of the kernel before them.  All they read
// before that kernel has ended is, in the stream and row kernels and where the caller says that it may (`early`), rows of B; the
// stream kernel asks for them in L2 otherwise, which reads no value.  Like the
// row-wise kernels they let the kernel behind them start only after their own wait, so that whatever runs then, the kernel
// before the last has ended; and only once they have their tensor memory, which a CTA behind them, waiting for their end, could
// otherwise hold.
#include <mutex>

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
__device__ __forceinline__ void store_peer(uint32_t addr, int v) {  // to an address of map_to
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
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
// N outputs rounded to the activations' type.  (The type is asked for once, not at each value: a branch between them would keep the
// conversions from overlapping.  In the pair kernel's writers that made 4096 x 4096 x 1024 7 us slower.)
template <int N>
__device__ __forceinline__ void pack_all(int act, const float (&f)[N], uint32_t (&o)[N / 2]) {
  if (act == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) o[i] = pack2<0>(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) o[i] = pack2<1>(f[2 * i], f[2 * i + 1]);
  }
}
template <int N>
__device__ __forceinline__ void add_bias(int act, float (&f)[N], const unsigned short* bias) {
  if (act == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] += __half2float(__ushort_as_half(bias[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] += __uint_as_float((uint32_t)bias[i] << 16);
  }
}
template <int N>
__device__ __forceinline__ void gate_all(float (&f)[N], const float (&u)[N], int use_clamp, float clamp) {
  if (use_clamp) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = gated_product(f[i], u[i], 1, clamp);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = gated_product(f[i], u[i], 0, clamp);
  }
}
__device__ __forceinline__ uint32_t pack_act(int act, float lo, float hi) { return act == 0 ? pack2<0>(lo, hi) : pack2<1>(lo, hi); }
__device__ __forceinline__ float act_value(int act, unsigned short bits) {
  return act == 0 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
}

// ---- pair kernel ------------------------------------------------------------------------------------------
// 256 or 128 product columns a tile: 128 rows of A and 128 or 64 of B per CTA and stage
constexpr int pair_stages(int cols) { return cols == 256 ? 6 : 8; }
constexpr int pair_stage_bytes(int cols) { return 16384 + cols * 64; }
constexpr int P_STORE = 4096;  // 32 rows x 64 columns on their way out, for each of the eight warps that write the outputs
constexpr int P_WRITERS = 256;
constexpr int P_THREADS = 128 + P_WRITERS;  // copies of A, products, tensor memory, copies of B; the writers
struct PairBars {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag, peer_abort;
  int issued[4];  // pieces that the copying warps have asked for: of A and of B, and in the first CTA the second one's
};
constexpr int P_SCALES = 256 * 4 + 256 * 2;  // a tile's column scales and biases
int int8_pair_smem_bytes(int cols) {
  return 1024 + pair_stages(cols) * pair_stage_bytes(cols) + (P_WRITERS / 32) * P_STORE + P_SCALES + (int)sizeof(PairBars);
}

// Output tile `t`: raster groups of m_group row tiles, row tile fastest, so that the clusters that run together share columns of B
// while a group's rows of A stay in L2.
__device__ __forceinline__ void pair_tile(const Int8Params& p, int t, int* m_tile, int* n_tile) {
  const int per = p.m_group * p.n_tiles, grp = t / per, in = t - grp * per;
  const int size = min(p.m_group, p.m_tiles - grp * p.m_group);
  *n_tile = in / size;
  *m_tile = grp * p.m_group + in - *n_tile * size;
}

template <bool GATED, int COLS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P_THREADS, 1)
    int8_pair_kernel(const Int8Params p, const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                     const __grid_constant__ CUtensorMap tc) {
  constexpr int STAGES = pair_stages(COLS), STAGE = pair_stage_bytes(COLS);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  unsigned char* base = smem_raw + (ring - raw);
  const uint32_t store_s = ring + STAGES * STAGE;
  float* col_sf = reinterpret_cast<float*>(base + STAGES * STAGE + (P_WRITERS / 32) * P_STORE);
  unsigned short* col_bias = reinterpret_cast<unsigned short*>(col_sf + 256);
  const uint32_t bars_off = STAGES * STAGE + (P_WRITERS / 32) * P_STORE + P_SCALES;
  PairBars* bars = reinterpret_cast<PairBars*>(base + bars_off);
  const uint32_t bars_s = ring + bars_off;
#define BAR(field, i) (bars_s + (uint32_t)offsetof(PairBars, field) + (uint32_t)(i) * 8u)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  volatile int* abort_flag = &bars->abort_flag;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(BAR(full, i), 1); mbar_init(BAR(empty, i), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(BAR(acc_full, i), 1); mbar_init(BAR(acc_empty, i), 2 * (P_WRITERS / 32)); }
    bars->abort_flag = bars->peer_abort = 0;
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
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0 || warp == 3) {
    // ---- copies: this CTA's half of A (warp 0) and of B (warp 3); both CTAs' report to the first one's barrier ----
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t phase = 0;
      bool good = true;
      const CUtensorMap* map = warp == 0 ? &ta : &tb;
      const uint32_t to = ring + (warp == 0 ? 0u : 16384u);
      for (int t = first; t < p.tiles && good; t += step) {
        int m_tile, n_tile;
        pair_tile(p, t, &m_tile, &n_tile);
        const int row = warp == 0 ? m_tile * 256 + (int)rank * 128
                        : GATED   ? n_tile * (COLS / 2) + (int)rank * p.N
                                  : n_tile * COLS + (int)rank * (COLS / 2);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          if (!mbar_wait_abortable(BAR(empty, s), phase ^ 1u, abort_flag)) { good = false; break; }
          if (rank == 0 && warp == 0) expect_bytes(BAR(full, s), 2u * STAGE);
          asm volatile(
              "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
              ::"r"(to + (uint32_t)s * STAGE), "l"(map), "r"(map_to(BAR(full, s), 0)), "r"(kb * 128), "r"(row) : "memory");
          ++issued;
          if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
      }
      bars->issued[warp == 0 ? 0 : 1] = issued;
    }
  } else if (warp == 1) {
    // ---- products, issued by the first CTA for both ----
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc = int8_idesc(256, COLS);
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
          const uint64_t ad = umma_smem_desc(ring + (uint32_t)s * STAGE), bd = umma_smem_desc(ring + (uint32_t)s * STAGE + 16384u);
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                ::"r"(tmem + (uint32_t)(acc * COLS)), "l"(ad + (uint64_t)(ks * 2)), "l"(bd + (uint64_t)(ks * 2)), "r"(idesc),
                "r"((kb > 0 || ks > 0) ? 1u : 0u)
                : "memory");
          asm volatile(
              "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                  BAR(empty, s)), "h"((unsigned short)3)
              : "memory");
          if (++s == STAGES) { s = 0; phase ^= 1u; }
        }
        if (good)
          asm volatile(
              "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                  BAR(acc_full, acc)), "h"((unsigned short)3)
              : "memory");
      }
    }
  } else if (warp >= 4) {
    // ---- outputs: thread = row; the two warps that share a quarter of the lanes take turns with 64 columns, and a warp's outputs go
    // through shared memory of its own, so that the warps need not wait for one another ----
    const int ew = warp & 3, turn = (warp >> 2) - 1, wt = tid - 128;
    const uint32_t lane_addr = tmem + ((uint32_t)(ew * 32) << 16);
    const uint32_t empty0 = map_to(BAR(acc_empty, 0), 0);
    const uint32_t store = store_s + (uint32_t)((warp - 4) * P_STORE), row_s = store + (uint32_t)lane * 128u;
    constexpr int CHUNKS = COLS / (GATED ? 128 : 64);
    // a tile's scales, asked for a tile ahead: of the thread's row, and of one of the product's columns (gated, the gates and then
    // their partners)
    float sa = 0.f, next_sa = 0.f, next_sf = 0.f;
    unsigned short next_bias = 0;
    auto ask = [&](int t) {
      if (t >= p.tiles) return;
      int m_tile, n_tile;
      pair_tile(p, t, &m_tile, &n_tile);
      const int row = m_tile * 256 + (int)rank * 128 + ew * 32 + lane;
      next_sa = row < p.M ? p.a_sf[row] : 0.f;
      const int n = n_tile * (GATED ? COLS / 2 : COLS) + (GATED ? wt % (COLS / 2) : wt);
      const bool is = wt < COLS && n < p.N;
      next_sf = is ? p.b_sf[GATED && wt >= COLS / 2 ? n + p.N : n] : 0.f;
      if (!GATED && p.bias) next_bias = is ? p.bias[n] : (unsigned short)0;
    };
    // The next but one tile may have the accumulators.  (What the arrival orders are the loads from tensor memory, by the fence in front
    // of it.  As a release at cluster scope it also waited for the warp's stores on their way out: 8192 x 6160 x 528 53 us, not 41.)
    auto free_accumulators = [&](int acc) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(empty0 + (uint32_t)acc * 8u) : "memory");
    };
    ask(first);
    int it = 0;
    for (int t = first; t < p.tiles; t += step, ++it) {
      int m_tile, n_tile;
      pair_tile(p, t, &m_tile, &n_tile);
      const int row0 = m_tile * 256 + (int)rank * 128 + ew * 32, n0 = n_tile * (GATED ? COLS / 2 : COLS);
      const int acc = it & 1;
      const bool ok = mbar_wait_abortable(BAR(acc_full, acc), (uint32_t)(it >> 1) & 1u, abort_flag);
      // The writers have used the last tile's scales; and one thread's patience may end where another's did not: they give up together.
      int bad;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(bad) : "r"(ok ? 0 : 1), "n"(P_WRITERS) : "memory");
      if (bad) break;
      sa = next_sa;
      if (wt < COLS) {
        col_sf[wt] = next_sf;
        if (!GATED && p.bias) col_bias[wt] = next_bias;
      }
      ask(t + step);
      asm volatile("bar.sync 1, %0;" ::"n"(P_WRITERS) : "memory");
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
      for (int j = turn; j < CHUNKS; j += 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c0 = j * 64 + h * 32;
          uint32_t v[32], u[GATED ? 32 : 1], o[16];
          tmem_ld_32(lane_addr + (uint32_t)(acc * COLS + c0), v);
          if constexpr (GATED) tmem_ld_32(lane_addr + (uint32_t)(acc * COLS + COLS / 2 + c0), u);
          if (h == 1 && j + 2 >= CHUNKS) free_accumulators(acc);  // this warp's part is in registers
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = scaled(v[i], sa, col_sf[c0 + i]);
          if constexpr (GATED) {
            float g[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) g[i] = scaled(u[i], sa, col_sf[COLS / 2 + c0 + i]);
            gate_all(f, g, p.use_clamp, p.clamp);
          } else if (p.bias) {
            add_bias(p.act, f, col_bias + c0);
          }
          pack_all(p.act, f, o);
          if (h == 0) {  // the last copy has read the buffer
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)  // 16-byte pieces, swizzled as the tensor map says
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_s + (uint32_t)(((h * 4 + q) ^ (lane & 7)) * 16)),
                         "r"(o[4 * q]), "r"(o[4 * q + 1]), "r"(o[4 * q + 2]), "r"(o[4 * q + 3]) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          const int n = n0 + j * 64;
          if (n < p.N && row0 < p.M)
            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&tc),
                         "r"(store), "r"(n), "r"(row0) : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        __syncwarp();
      }
      if (turn >= CHUNKS) free_accumulators(acc);  // (a narrow gated tile is one warp's)
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag && tid == 0) {
    atomicExch(p.status, ST_DEVICE_TIMEOUT);
    p.status[1] = 12;  // where: pair kernel
    p.status[2] = blockIdx.x;
    p.status[3] = 0;
    store_peer(map_to(bars_s + (uint32_t)offsetof(PairBars, peer_abort), rank ^ 1u), 1);
  }
  cluster_sync();  // neither CTA's shared memory or tensor memory goes while the other still uses it
  if (*abort_flag || *static_cast<volatile int*>(&bars->peer_abort)) {
    // One of the two has given up (both see it): the copies in flight, which all report to the first CTA, land before the CTAs end.
    if (rank == 1 && tid < 2) store_peer(map_to(bars_s + (uint32_t)offsetof(PairBars, issued) + (uint32_t)(2 + tid) * 4u, 0), bars->issued[tid]);
    __syncwarp();
    cluster_sync();
    if (rank == 0 && tid < STAGES) {
      const int issued[4] = {bars->issued[0], bars->issued[1], bars->issued[2], bars->issued[3]};
      const uint32_t bytes[4] = {16384u, STAGE - 16384u, 16384u, STAGE - 16384u};
      const RingRest rest = ring_rest(tid, STAGES, issued, bytes);
      if (rest.announce) expect_bytes(BAR(full, tid), rest.announce);
      if (rest.strike)
        asm volatile("mbarrier.complete_tx.relaxed.cluster.shared::cta.b64 [%0], %1;" ::"r"(BAR(full, tid)), "r"(rest.strike) : "memory");
      if (rest.item >= 0) mbar_wait_bounded(BAR(full, tid), (uint32_t)(rest.item / STAGES) & 1u);
    }
    __syncwarp();
    cluster_sync();
  }
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
#undef BAR
}

// ---- stream kernel ----------------------------------------------------------------------------------------
// A CTA: all rows of A (lanes of tensor memory; 128, or two accumulators of 128) against a share of the output columns, which are as many
// rows of B, or gated twice as many (gates, then partners), over its part of K.  Shares differ by eight columns at most, which is what
// spreads B evenly over the SMs, so K is split only where reading A again in each CTA would take longer than B.  Then the CTAs of a
// cluster own a part of the columns each: the others store their sums of these into its shared memory, and it adds them to its own.
constexpr int S_THREADS = 256;
// Warps that take turns with a stage's copies: what a thread does for one (a wait, a count, two or three copies) takes it about as long
// as the tensor core takes for the stage.  100 x 11008 x 4224, us with one / four: 11.9 / 11.5.
constexpr int S_COPIERS = 4;
constexpr int S_STAGES_MAX = 16;
struct StreamBars {
  uint64_t full[S_STAGES_MAX], empty[S_STAGES_MAX], done;
  uint32_t tmem_base;
  int abort_flag;
  float b_sf[264];           // the share's columns: gated, the gates' scales and then their partners' (read 16 at a time)
  unsigned short bias[264];
};
static __host__ __device__ int stream_ring_bytes(int rows, int b_rows, int stages) {
  // (the tensor core reads whole accumulators' rows of A: behind the last stage too there is memory)
  return stages * (b_rows + rows) * 128 + ((rows + 127) / 128 * 128 - rows) * 128;
}
// Sums that a CTA gets from its cluster: [sender][row][own columns], rows 16 bytes further apart than they are long (threads are rows:
// their 16-byte stores then meet different banks).  They lie behind the ring where they are small, so that nobody has to wait
// until the receiver's products have read the ring; else in it.
constexpr int S_INBOX_APART = 16384;
// (of shares of `width` columns: the widest part that a CTA owns)
static __host__ __device__ int stream_inbox_pitch(bool gated, int width, int cluster) {
  return (width / 8 + cluster - 1) / cluster * 8 * (gated ? 2 : 1) * 4 + 16;
}
static __host__ __device__ int stream_inbox_bytes(int M, bool gated, int width, int cluster) {
  return cluster > 1 ? (cluster - 1) * M * stream_inbox_pitch(gated, width, cluster) + 64 : 0;  // (sums are read 16 at a time)
}
int int8_stream_smem_bytes(int M, bool gated, int width, int cluster, int stages) {
  const int inbox = stream_inbox_bytes(M, gated, width, cluster);
  const int ring = stream_ring_bytes((M + 15) / 16 * 16, (gated ? 2 : 1) * width, stages);
  const int data = inbox <= S_INBOX_APART ? ring + inbox : ring > inbox ? ring : inbox;
  return 1024 + data + (int)sizeof(StreamBars);
}

__device__ __forceinline__ void stream_load_b(const Int8Params& p, const CUtensorMap* tb, bool gated, uint32_t dst, uint32_t bar, int kb,
                                              int n0, int width) {
  for (int h = 0; h < (gated ? 2 : 1); ++h)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst + (uint32_t)(h * width) * 128u), "l"(tb), "r"(bar), "r"(kb * 128), "r"(n0 + h * p.N) : "memory");
}

// The same rows into L2 only.
__device__ __forceinline__ void stream_prefetch_b(const Int8Params& p, const CUtensorMap* tb, bool gated, int kb, int n0) {
  for (int h = 0; h < (gated ? 2 : 1); ++h)
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(tb), "r"(kb * 128), "r"(n0 + h * p.N) : "memory");
}

template <bool GATED>
__global__ void __launch_bounds__(S_THREADS)
    int8_stream_kernel(const Int8Params p, const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                       const __grid_constant__ CUtensorMap tb_less) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw);
  const uint32_t bars_s = raw;
  StreamBars* bars = reinterpret_cast<StreamBars*>(smem_raw);
  const uint32_t ring = (raw + (uint32_t)sizeof(StreamBars) + 1023u) & ~1023u;
#define BAR(field, i) (bars_s + (uint32_t)offsetof(StreamBars, field) + (uint32_t)(i) * 8u)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile int* abort_flag = &bars->abort_flag;
  const int S = p.cluster;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  // the first `wide` shares are of p.width columns, the others of eight less
  const int share = S > 1 ? blockIdx.x / S : blockIdx.x, width = share < p.wide ? p.width : p.width - 8;
  const int n0 = share * (p.width - 8) + 8 * min(share, p.wide);
  const CUtensorMap* map_b = share < p.wide ? &tb : &tb_less;
  const int kb0 = (int)((long long)p.kblocks * rank / S), kb1 = (int)((long long)p.kblocks * (rank + 1) / S);
  const int b_rows = GATED ? 2 * width : width;
  const int mma_n = (b_rows + 15) / 16 * 16;  // (what is past B's rows of a stage is rows of A: columns that nobody reads)
  const uint32_t b_bytes = (uint32_t)b_rows * 128u, stage_bytes = b_bytes + (uint32_t)p.rows * 128u;
  const int accs = p.rows > 128 ? 2 : 1;
  uint32_t cols = 32;  // of tensor memory: a power of two
  while (cols < (uint32_t)(accs * mma_n)) cols *= 2;
  const int pitch = stream_inbox_pitch(GATED, p.width, S);
  const bool apart = stream_inbox_bytes(p.M, GATED, p.width, S) <= S_INBOX_APART;
  const uint32_t inbox = apart ? ring + (uint32_t)stream_ring_bytes(p.rows, b_rows, p.stages) : ring;

  if (tid <= p.stages) {
    if (tid < p.stages) {
      mbar_init(BAR(full, tid), 1);
      mbar_init(BAR(empty, tid), 1);
    } else {
      mbar_init(BAR(done, 0), 1);
      bars->abort_flag = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  // every CTA of the cluster runs before its shared memory is written (waited for at the first store)
  if (S > 1 && apart) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  bool copies = false;   // this thread's, and how far they are: the next slot, and how often the ring has been gone round
  int slot = warp, lap = 0;
  if (warp < S_COPIERS) {
    if (elect_one()) {
      // The first rows of B come under the end of the kernel before this one: into shared memory where the caller says that B has been
      // complete since before that kernel, else as far as L2, where what that kernel still writes meets them.  (us, read early / into
      // L2 / neither: 8 x 57344 x 4096 gated 37.5 / 37.9 / 39.1, 64 x 28672 x 4096 gated 21.2 / 21.5 / 22.1.)
      if (p.early)
        for (int i = warp; i < p.stages && kb0 + i < kb1; i += S_COPIERS) {
          expect_bytes(BAR(full, i), stage_bytes);
          stream_load_b(p, map_b, GATED, ring + (uint32_t)i * stage_bytes, BAR(full, i), kb0 + i, n0, width);
        }
      else
        for (int i = warp; i < p.stages && kb0 + i < kb1; i += S_COPIERS) stream_prefetch_b(p, map_b, GATED, kb0 + i, n0);
      asm volatile("prefetch.tensormap [%0];" ::"l"(&ta) : "memory");
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (elect_one()) {
      // Block kb0 + lap * stages + slot goes to slot `slot`, and a slot is one warp's: a wait for its barrier's parity is then never more
      // than a phase behind.
      copies = true;
      for (int kb = kb0 + warp; slot < p.stages && kb < kb1; kb = kb0 + lap * p.stages + slot) {
        if (!mbar_wait_abortable(BAR(empty, slot), ((uint32_t)lap & 1u) ^ 1u, abort_flag)) break;
        const uint32_t bar = BAR(full, slot), dst = ring + (uint32_t)slot * stage_bytes;
        if (!p.early || lap > 0) {
          expect_bytes(bar, stage_bytes);
          stream_load_b(p, map_b, GATED, dst, bar, kb, n0, width);
        }
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst + b_bytes), "l"(&ta), "r"(bar), "r"(kb * 128), "r"(0) : "memory");
        slot += S_COPIERS;
        if (slot >= p.stages) { slot = warp; ++lap; }
      }
    }
    __syncwarp();
  } else if (warp == S_COPIERS) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     bars_s + (uint32_t)offsetof(StreamBars, tmem_base)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    __syncwarp();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base), 0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (elect_one()) {
      const uint32_t idesc = int8_idesc(128, mma_n);
      int s = 0;
      uint32_t phase = 0;
      bool good = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_abortable(BAR(full, s), phase, abort_flag)) { good = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t bd = umma_smem_desc(ring + (uint32_t)s * stage_bytes), ad = umma_smem_desc(ring + (uint32_t)s * stage_bytes + b_bytes);
        for (int m = 0; m < accs; ++m)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                ::"r"(tmem + (uint32_t)(m * mma_n)), "l"(ad + (uint64_t)(m * 1024 + ks * 2)), "l"(bd + (uint64_t)(ks * 2)), "r"(idesc),
                "r"((kb > kb0 || ks > 0) ? 1u : 0u)
                : "memory");
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(BAR(empty, s)) : "memory");
        if (++s == p.stages) { s = 0; phase ^= 1u; }
      }
      if (good)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(BAR(done, 0)) : "memory");
    }
    __syncwarp();
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = tid - 32 * (S_COPIERS + 1); i < b_rows; i += S_THREADS - 32 * (S_COPIERS + 1)) {
      bars->b_sf[i] = p.b_sf[GATED && i >= width ? n0 + p.N + i - width : n0 + i];
      if (!GATED && p.bias) bars->bias[i] = p.bias[n0 + i];
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);
  // ---- outputs: thread = row of A (one or two); the two warps that share a quarter of the lanes take turns with the columns ----
  (void)mbar_wait_abortable(BAR(done, 0), 0, abort_flag);
  __syncwarp();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const int row = (warp & 3) * 32 + lane, turn = warp >> 2;
  const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  // columns that a CTA of the cluster writes, in units of eight
  const int units = width / 8, own0 = units * rank / S * 8, own = units * (rank + 1) / S * 8 - own0;
  if (S > 1) {
    if (!apart) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA's ring may be written
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int m = 0; m < accs; ++m) {
      if (m * 128 + (warp & 3) * 32 >= p.M) break;
      const int t = m * 128 + row;
      for (int j = 8 * turn; j < b_rows; j += 16) {
        uint32_t v[8];
        tmem_ld_8_async(lane_addr + (uint32_t)(m * mma_n + j), v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "+r"(v[i]));  // no use of v moves above the wait
        const int seg = GATED && j >= width ? 1 : 0, unit = j / 8 - seg * units, c = ((unit + 1) * S - 1) / units;
        const int first = units * c / S, at = 8 * (seg * (units * (c + 1) / S - first) + unit - first);
        if (c != rank && t < p.M) {
          const int slot = rank < c ? rank : rank - 1;  // among the senders to c
          const uint32_t to = map_to(inbox + (uint32_t)((slot * p.M + t) * pitch + at * 4), (uint32_t)c);
#pragma unroll
          for (int q = 0; q < 2; ++q)
            asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (uint32_t)(q * 16)), "r"(v[4 * q]),
                         "r"(v[4 * q + 1]), "r"(v[4 * q + 2]), "r"(v[4 * q + 3]) : "memory");
        }
        __syncwarp();
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  for (int m = 0; m < accs; ++m) {
    if (m * 128 + (warp & 3) * 32 >= p.M) break;
    const int t = m * 128 + row;
    const float sa = t < p.M ? p.a_sf[t] : 0.f;
    for (int j = 16 * turn; j < own; j += 32) {
      const int i0 = own0 + j, n = n0 + i0;  // 16 columns, or the last 8 of the CTA's
      const bool full = j + 8 < own;
      uint32_t v[16] = {}, u[16] = {};
      tmem_ld_8_async(lane_addr + (uint32_t)(m * mma_n + i0), v);
      if (full) tmem_ld_8_async(lane_addr + (uint32_t)(m * mma_n + i0 + 8), v + 8);
      if constexpr (GATED) {
        tmem_ld_8_async(lane_addr + (uint32_t)(m * mma_n + width + i0), u);
        if (full) tmem_ld_8_async(lane_addr + (uint32_t)(m * mma_n + width + i0 + 8), u + 8);
      }
      tmem_ld_wait(v);
      if (GATED)
#pragma unroll
        for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(u[i]));
      for (int c = 0; c < S - 1 && t < p.M; ++c) {
        const uint32_t from = inbox + (uint32_t)((c * p.M + t) * pitch + j * 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint4 w = lds_u4(from + (uint32_t)(q * 16));
          v[4 * q] += w.x; v[4 * q + 1] += w.y; v[4 * q + 2] += w.z; v[4 * q + 3] += w.w;
          if constexpr (GATED) {
            const uint4 x = lds_u4(from + (uint32_t)(own * 4 + q * 16));
            u[4 * q] += x.x; u[4 * q + 1] += x.y; u[4 * q + 2] += x.z; u[4 * q + 3] += x.w;
          }
        }
      }
      float f[16];
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = scaled(v[i], sa, bars->b_sf[i0 + i]);
      if constexpr (GATED) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = scaled(u[i], sa, bars->b_sf[width + i0 + i]);
        gate_all(f, x, p.use_clamp, p.clamp);
      } else if (p.bias) {
        add_bias(p.act, f, bars->bias + i0);
      }
      pack_all(p.act, f, o);
      if (t < p.M && *abort_flag == 0) {
        uint4* to = reinterpret_cast<uint4*>(p.c + (size_t)t * p.ldc + n);
        to[0] = make_uint4(o[0], o[1], o[2], o[3]);
        if (full) to[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
      __syncwarp();
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abort_flag && tid == 0) {
    atomicExch(p.status, ST_DEVICE_TIMEOUT);
    p.status[1] = 13;  // where: stream kernel
    p.status[2] = blockIdx.x;
    p.status[3] = 0;
  }
  if (*abort_flag && copies)  // the copies in flight land before the CTA ends: the last of each slot
    for (int q = warp; q < p.stages; q += S_COPIERS) {
      const int last = q < slot ? lap : lap - 1;
      if (last >= 0 && kb0 + last * p.stages + q < kb1) mbar_wait_bounded(BAR(full, q), (uint32_t)last & 1u);
    }
  __syncwarp();
  if (warp == S_COPIERS) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  }
#undef BAR
}

// ---- row kernel -------------------------------------------------------------------------------------------
// Up to 16 rows of A: a CTA takes 16 rows of B at a time (gated: 8 gates and their 8 partners), its warps share K, and each thread
// reads its part of B straight from memory into the registers that mma.sync takes it from: 16 consecutive bytes of a row are the
// four words of two steps, since the order of K inside a sum is free as long as A's words go by the same order.  Nothing passes
// through shared memory but the warps' sums, and there is no pipeline to fill: what a small product takes is little more than the
// latency of its loads.  (us, the stream kernel / this one: 1 x 4096 x 4096 8.1 / 5.1, 4 x 1024 x 4096 5.6 / 3.5; with 12 rows, whose
// loads are as many as B's, 1504 x 11008 8.2 / 10.2.  B read early takes 0.3 to 1.1 us off this one: its loads are what it consists of.
// Rows on their way to L2 instead gave nothing that held over sizes: 1 x 4096 x 4096 4.5 for 5.1, 8 x 14336 x 4096 15.9 for 15.2.)
constexpr int R_WARPS = 16;
constexpr int R_BATCH = 4;  // 64-byte pieces of two rows that a thread has in flight
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool GATED, int NT>  // NT: groups of eight rows of A
__global__ void __launch_bounds__(R_WARPS * 32, 2) int8_row_kernel(const Int8Params p) {
  __shared__ int sums[2][R_WARPS][NT * 8][17];  // [warp][row of A][row of B], twice: the next item's while this one's are read
  constexpr int OUTS = GATED ? 8 : 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
  const int items = p.N / OUTS, k_lane = warp * 64 + tig * 16;
  const signed char* a_rows[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) a_rows[j] = p.a + (size_t)(g + 8 * j) * p.lda;
  uint4 w[R_BATCH][2];
  auto load_b = [&](int item, int k0) {
    const signed char* lo = p.b + (size_t)(item * OUTS + g) * p.ldb;
    const signed char* hi = p.b + (GATED ? (size_t)p.N + item * OUTS + g : (size_t)item * OUTS + g + 8) * p.ldb;
#pragma unroll
    for (int i = 0; i < R_BATCH; ++i) {
      const int k = k0 + i * (R_WARPS * 64);
      const uint4 none = make_uint4(0, 0, 0, 0);
      w[i][0] = k < p.K ? ld_stream_u4(reinterpret_cast<const uint4*>(lo + k)) : none;
      w[i][1] = k < p.K ? ld_stream_u4(reinterpret_cast<const uint4*>(hi + k)) : none;
    }
  };
  int item = blockIdx.x, buf = 0;
  if (p.early && item < items) load_b(item, k_lane);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!p.early && item < items) load_b(item, k_lane);
  for (; item < items; item += gridDim.x, buf ^= 1) {
    int d[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[j][i] = 0;
    for (int k0 = k_lane;; ) {
#pragma unroll
      for (int i = 0; i < R_BATCH; ++i) {
        const int k = k0 + i * (R_WARPS * 64);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint4 x = make_uint4(0, 0, 0, 0);
          if (k < p.K && g + 8 * j < p.M) x = *reinterpret_cast<const uint4*>(a_rows[j] + k);
          mma_s8(d[j], w[i][0].x, w[i][1].x, w[i][0].y, w[i][1].y, x.x, x.y);
          mma_s8(d[j], w[i][0].z, w[i][1].z, w[i][0].w, w[i][1].w, x.z, x.w);
        }
      }
      k0 += R_BATCH * R_WARPS * 64;
      // (the test is the warp's, so that all its lanes multiply)
      if (k0 - tig * 16 >= p.K) break;
      load_b(item, k0);
    }
    const int next = item + gridDim.x;
    if (next < items) load_b(next, k_lane);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      sums[buf][warp][8 * j + 2 * tig][g] = d[j][0];
      sums[buf][warp][8 * j + 2 * tig + 1][g] = d[j][1];
      sums[buf][warp][8 * j + 2 * tig][g + 8] = d[j][2];
      sums[buf][warp][8 * j + 2 * tig + 1][g + 8] = d[j][3];
    }
    __syncthreads();
    const int t = tid / OUTS, f = tid % OUTS, n = item * OUTS + f;
    if (t < p.M) {
      int x = 0, y = 0;
#pragma unroll
      for (int i = 0; i < R_WARPS; ++i) {
        x += sums[buf][i][t][f];
        if (GATED) y += sums[buf][i][t][f + 8];
      }
      const float sa = p.a_sf[t];
      float o = scaled((uint32_t)x, sa, p.b_sf[n]);
      if constexpr (GATED) o = gated_product(o, scaled((uint32_t)y, sa, p.b_sf[p.N + n]), p.use_clamp, p.clamp);
      else if (p.bias) o += act_value(p.act, p.bias[n]);
      p.c[(size_t)t * p.ldc + n] = (unsigned short)(pack_act(p.act, o, 0.f) & 0xffffu);
    }
  }
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

template <bool GATED, int COLS>
static cudaError_t pair_launch(const Int8Params& p, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, int grid,
                               cudaStream_t stream) {
  static std::atomic<bool> allowed[16];
  const cudaError_t e = allow_smem(int8_pair_kernel<GATED, COLS>, allowed);
  if (e != cudaSuccess) return e;
  return launch_behind(int8_pair_kernel<GATED, COLS>, grid, P_THREADS, 1, int8_pair_smem_bytes(COLS), stream, p, ta, tb, tc);
}
template <bool GATED>
static cudaError_t stream_launch(const Int8Params& p, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb_less,
                                 cudaStream_t stream) {
  static std::atomic<bool> allowed[16];
  const cudaError_t e = allow_smem(int8_stream_kernel<GATED>, allowed);
  if (e != cudaSuccess) return e;
  return launch_behind(int8_stream_kernel<GATED>, p.tiles * p.cluster, S_THREADS, p.cluster, p.smem, stream, p, ta, tb, tb_less);
}

cudaError_t int8_pair_launch(const Int8Params& p, bool gated, int cols, const CUtensorMap& ta, const CUtensorMap& tb,
                             const CUtensorMap& tc, int grid, cudaStream_t stream) {
  if (cols == 256) return gated ? pair_launch<true, 256>(p, ta, tb, tc, grid, stream) : pair_launch<false, 256>(p, ta, tb, tc, grid, stream);
  return gated ? pair_launch<true, 128>(p, ta, tb, tc, grid, stream) : pair_launch<false, 128>(p, ta, tb, tc, grid, stream);
}
cudaError_t int8_stream_launch(const Int8Params& p, bool gated, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb_less,
                               cudaStream_t stream) {
  return gated ? stream_launch<true>(p, ta, tb, tb_less, stream) : stream_launch<false>(p, ta, tb, tb_less, stream);
}

// Clusters of 1 << i CTAs with an SM each that run at once: fewer than the SMs make, since a cluster stays in a group of SMs.  (Without
// a GPU estimates, for plans.)
const int* int8_stream_clusters(const DeviceInfo& di) {
  static std::atomic<bool> known[16], allowed[16];
  static int counts[17][4];
  static std::mutex mutex;
  int dev = -1;
  const bool gpu = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 16;
  const int at = gpu ? dev : 16;
  if (gpu && known[dev].load(std::memory_order_acquire)) return counts[dev];
  std::lock_guard<std::mutex> lock(mutex);
  for (int i = 0, s = 1; i < 4; ++i, s *= 2) {
    int n = 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(di.sm_count / s * s), 1, 1);
    cfg.blockDim = dim3(S_THREADS, 1, 1);
    cfg.dynamicSmemBytes = (size_t)di.max_smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (s > 1 && (!gpu || allow_smem(int8_stream_kernel<false>, allowed) != cudaSuccess ||
                  cudaOccupancyMaxActiveClusters(&n, int8_stream_kernel<false>, &cfg) != cudaSuccess || n < 1)) {
      (void)cudaGetLastError();
      n = s == 2 ? di.sm_count / 2 : di.sm_count * 7 / 8 / s;
    }
    counts[at][i] = s > 1 ? n : di.sm_count;
  }
  if (gpu) known[dev].store(true, std::memory_order_release);
  return counts[at];
}

cudaError_t int8_row_launch(const Int8Params& p, bool gated, int grid, cudaStream_t stream) {
  if (p.M <= 8)
    return gated ? launch_behind(int8_row_kernel<true, 1>, grid, R_WARPS * 32, 1, 0, stream, p)
                 : launch_behind(int8_row_kernel<false, 1>, grid, R_WARPS * 32, 1, 0, stream, p);
  return gated ? launch_behind(int8_row_kernel<true, 2>, grid, R_WARPS * 32, 1, 0, stream, p)
               : launch_behind(int8_row_kernel<false, 2>, grid, R_WARPS * 32, 1, 0, stream, p);
}

}  // namespace b200q
