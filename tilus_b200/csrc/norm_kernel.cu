// Row-wise kernels between the products of a decoder block: the per-token int8 cast, and the norms before and after a
// block with its gate and residual scale (norm.cuh has the formulas), forward and backward.
//
// All are bound by memory: each input is read once and each output written once, with a row held on the SM between the
// statistics and their use.  What keeps them from that bound is the number of instructions, so that threads own several vectors
// of eight neighbouring channels (16 bytes of a 16-bit type), which share a reduction's steps, and multiply pairs of channels at
// a time (f32x2).  Sums and statistics are fp32; the only roundings to fewer bits are those of the outputs.
#include "norm.cuh"

namespace b200q {

// The kernel before this one in the stream has ended; the one behind it may set up now, and no earlier: what it reads before this
// one has ended (weights) is then at least one kernel old.
__device__ __forceinline__ void start_behind() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- pairs of fp32 ------------------------------------------------------------------------------------------
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 pair(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 both(float x) { return pair(x, x); }
__device__ __forceinline__ void split(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum(F2 a) {
  float lo, hi;
  split(a, lo, hi);
  return lo + hi;
}

// eight values of a 16-bit type
template <int ACT>
__device__ __forceinline__ void unpack8(const uint4& v, F2 (&f)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (ACT == 0) {
      const float2 t = __half22float2(h2_from_bits(w[i]));
      f[i] = pair(t.x, t.y);
    } else {
      f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
}
template <int ACT>
__device__ __forceinline__ uint4 pack8(const F2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    split(f[i], lo, hi);
    w[i] = pack2<ACT>(lo, hi);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// eight values of the residual stream, of the activation type or fp32, in one or two 16-byte units
template <int ACT, bool F32>
struct Wide {
  static constexpr int UNITS = F32 ? 2 : 1;
  uint4 v[UNITS];
  __device__ __forceinline__ void load(const void* base, long long at) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(base) + at * (F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < UNITS; ++i) v[i] = p[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < UNITS; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(F2 (&f)[4]) const {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[2 * i] = pair(__uint_as_float(v[i].x), __uint_as_float(v[i].y));
        f[2 * i + 1] = pair(__uint_as_float(v[i].z), __uint_as_float(v[i].w));
      }
    } else {
      unpack8<ACT>(v[0], f);
    }
  }
  static __device__ __forceinline__ void store(void* base, long long at, const F2 (&f)[4]) {
    uint4* p = reinterpret_cast<uint4*>(static_cast<char*>(base) + at * (F32 ? 4 : 2));
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x[4];
        split(f[2 * i], x[0], x[1]);
        split(f[2 * i + 1], x[2], x[3]);
        p[i] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      }
    } else {
      p[0] = pack8<ACT>(f);
    }
  }
};

// ---- reductions over the threads of a row: a warp, or all warps of the CTA -----------------------------------------
// `slots`: 32 words that no other reduction uses until the next barrier but one; words of warps that the CTA has not are zero.
// Every thread gets the same result, summed in the same order.
__device__ __forceinline__ float row_sum(float x, float* slots, bool warp_row) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (warp_row) return x;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0.f;
  for (int i = 0; i < (int)blockDim.x / 32; i += 4) {
    const float4 s = *reinterpret_cast<const float4*>(slots + i);
    x += (s.x + s.y) + (s.z + s.w);
  }
  return x;
}
// two sums over a CTA of up to 16 warps: a warp's shuffles after the first serve both
__device__ __forceinline__ void row_sum2(float (&x)[2], float* slots) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float give = lane & 16 ? x[0] : x[1], mine = lane & 16 ? x[1] : x[0];
  float y = mine + __shfl_xor_sync(0xffffffffu, give, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if ((lane & 15) == 0) slots[(lane & 16) + warp] = y;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    x[j] = 0.f;
    for (int i = 0; i < (int)blockDim.x / 32; i += 4) {
      const float4 s = *reinterpret_cast<const float4*>(slots + 16 * j + i);
      x[j] += (s.x + s.y) + (s.z + s.w);
    }
  }
}
__device__ __forceinline__ uint32_t row_max(uint32_t x, uint32_t* slots, bool warp_row) {
  x = __reduce_max_sync(0xffffffffu, x);
  if (warp_row) return x;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0;
  for (int i = 0; i < (int)blockDim.x / 32; i += 4) {
    const uint4 s = *reinterpret_cast<const uint4*>(slots + i);
    x = max(max(x, max(s.x, s.y)), max(s.z, s.w));
  }
  return x;
}
// Words of warps that are not there, before the first reduction's barrier.
template <int N>
__device__ __forceinline__ void clear_slots(float (&slots)[N][32]) {
  if (threadIdx.x < 32 && threadIdx.x >= blockDim.x / 32)
#pragma unroll
    for (int i = 0; i < N; ++i) slots[i][threadIdx.x] = 0.f;
}

// ---- rows copied ahead ----------------------------------------------------------------------------------
// (16 bytes by the thread that will read them, so that nobody waits for anybody's copies)
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// a row or part of one, by the copy engine; the barrier counts its bytes
__device__ __forceinline__ void copy_row(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes),
               "r"(bar) : "memory");
}
template <int PENDING>
__device__ __forceinline__ void copies_wait() {  // all but the latest groups of this thread's have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// ---- per-token int8 cast --------------------------------------------------------------------------------
// m = max |x| of the row (as bits, so that a NaN is the largest);  out_sf = m / 127,  out = rint(x * (127 / m)), quotients and
// product rounded to fp32.  Rows of m < 2^-100 count as zero (127 / m would leave the range of fp32): codes 0, scale 1.  A row
// with a NaN or an infinity gets it as its scale, and codes 0: products with it are NaN, as they would be.
__device__ __forceinline__ void int8_scale(float top, float* sf, float* inv) {
  const bool zero = top < 0x1p-100f;
  *sf = zero ? 1.0f : __fdiv_rn(top, 127.0f);
  *inv = zero ? 0.0f : __fdiv_rn(127.0f, top);
  if (!(top < __int_as_float(0x7f800000))) *inv = 0.0f;
}
// Codes of eight values: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves its low byte in the sum's.  (The
// product is rounded before: a fused one would see its exact value.)
__device__ __forceinline__ uint2 int8_codes(const F2 (&f)[4], float inv) {
  uint32_t w[2];
  const F2 inv2 = both(inv), one = both(1.0f), magic = both(12582912.0f);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float b[4];
    split(fma2(f[2 * h] * inv2, one, magic), b[0], b[1]);
    split(fma2(f[2 * h + 1] * inv2, one, magic), b[2], b[3]);
    w[h] = __byte_perm(__byte_perm(__float_as_uint(b[0]), __float_as_uint(b[1]), 0x0040),
                       __byte_perm(__float_as_uint(b[2]), __float_as_uint(b[3]), 0x0040), 0x5410);
  }
  return inv != 0.0f ? make_uint2(w[0], w[1]) : make_uint2(0, 0);
}
// The largest magnitudes of each half of words of two 16-bit values, as bits (NaN wins), and of both as fp32 bits.
template <int ACT>
__device__ __forceinline__ uint32_t top2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (ACT == 0) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b & 0x7fff7fffu));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b & 0x7fff7fffu));
  return r;
}
template <int ACT>
__device__ __forceinline__ uint32_t top_bits(uint32_t top, const uint4& v) {
  return top2<ACT>(top2<ACT>(top2<ACT>(top2<ACT>(top, v.x), v.y), v.z), v.w);
}
template <int ACT>
__device__ __forceinline__ uint32_t top_value(uint32_t top) {
  const uint32_t one = max(top & 0x7fffu, top >> 16 & 0x7fffu);
  return ACT == 0 ? __float_as_uint(__half2float(__ushort_as_half((unsigned short)one))) & 0x7fffffffu : one << 16;
}

template <int ACT, int V>
__global__ void __launch_bounds__(1024) cast_int_kernel(const CastIntParams p, const int warp_rows) {
  __shared__ __align__(16) float slots[1][32];
  start_behind();
  const bool warp_row = warp_rows != 0;
  const int tpr = warp_row ? 32 : blockDim.x, me = warp_row ? threadIdx.x & 31 : threadIdx.x;
  const int t = warp_row ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (t >= p.T) return;  // (whole warps, and only where a warp has its own row)
  const int nvec = p.D / 8;
  const uint4* row = reinterpret_cast<const uint4*>(p.x + (size_t)t * p.ldx) + me;
  uint4 keep[V];
#pragma unroll
  for (int i = 0; i < V; ++i) keep[i] = me + i * tpr < nvec ? row[i * tpr] : make_uint4(0, 0, 0, 0);
  clear_slots(slots);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) bits = top_bits<ACT>(bits, keep[i]);
  for (int i = V; me + i * tpr < nvec; ++i) bits = top_bits<ACT>(bits, row[i * tpr]);  // (what does not stay in registers is read again)
  float sf, inv;
  int8_scale(__uint_as_float(row_max(top_value<ACT>(bits), reinterpret_cast<uint32_t*>(slots[0]), warp_row)), &sf, &inv);
  if (me == 0) p.out_sf[t] = sf;
  uint2* out = reinterpret_cast<uint2*>(p.out + (size_t)t * p.ldo) + me;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    F2 f[4];
    unpack8<ACT>(keep[i], f);
    if (me + i * tpr < nvec) out[i * tpr] = int8_codes(f, inv);
  }
  for (int i = V; me + i * tpr < nvec; ++i) {
    F2 f[4];
    unpack8<ACT>(row[i * tpr], f);
    out[i * tpr] = int8_codes(f, inv);
  }
}

// ---- block norm -------------------------------------------------------------------------------------------
template <int ACT, bool F32, int V>
__global__ void __launch_bounds__(V <= 2 ? 1024 : 512, V == 4 && !F32 ? 2 : 1) norm_kernel(const NormParams p, const int warp_rows) {
  __shared__ __align__(16) float slots[3][32];
  start_behind();
  const bool warp_row = warp_rows != 0;
  const int tpr = warp_row ? 32 : blockDim.x, me = warp_row ? threadIdx.x & 31 : threadIdx.x;
  const int t = warp_row ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (t >= p.T) return;
  const int nvec = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  const uint4 none = make_uint4(0, 0, 0, 0);
  F2 r[V][4];  // block, then the new residual, then x
  Wide<ACT, F32> res[V];
  uint4 raw[V], ahead[V][2];  // one vector or two: the weights of what comes first are asked for with the row
  const unsigned short* gate = p.gate ? p.gate + (t / p.tokens_per_gate) * p.ldg : nullptr;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    raw[i] = none;
    res[i].zero();
    if (v < nvec) {
      raw[i] = *reinterpret_cast<const uint4*>(p.block + t * p.ldb + v * 8);
      if (p.residual) res[i].load(p.residual, t * p.ldr + v * 8);
    }
  }
  auto weights = [&](const unsigned short* from, int v) { return v < nvec ? *reinterpret_cast<const uint4*>(from + v * 8) : none; };
  if constexpr (V <= 2) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (p.post) ahead[i][0] = weights(p.post, me + i * tpr);
      if (gate) ahead[i][1] = weights(gate, me + i * tpr);
    }
  }
  clear_slots(slots);
#pragma unroll
  for (int i = 0; i < V; ++i) unpack8<ACT>(raw[i], r[i]);
  const F2 zero = both(0.f);
  if (p.post) {
    F2 s = zero;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) s = fma2(r[i][k], r[i][k], s);
    const F2 inv = both(rsqrtf(row_sum(sum(s), slots[0], warp_row) * inv_d + p.eps));
#pragma unroll
    for (int i = 0; i < V; ++i) {
      F2 w[4];
      unpack8<ACT>(V <= 2 ? ahead[i][0] : weights(p.post, me + i * tpr), w);
#pragma unroll
      for (int k = 0; k < 4; ++k) r[i][k] = r[i][k] * (inv * w[k]);
    }
  }
  if (gate) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      F2 w[4];
      unpack8<ACT>(V <= 2 ? ahead[i][1] : weights(gate, me + i * tpr), w);
#pragma unroll
      for (int k = 0; k < 4; ++k) r[i][k] = r[i][k] * w[k];
    }
  }
  F2 s = zero;
  const F2 scale = both(p.scale);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    F2 q[4];
    res[i].get(q);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      r[i][k] = fma2(scale, q[k], r[i][k]);
      s = fma2(r[i][k], r[i][k], s);
    }
    if (v < nvec) Wide<ACT, F32>::store(p.new_residual, t * p.ldn + v * 8, r[i]);
  }
  if constexpr (V <= 2)
#pragma unroll
    for (int i = 0; i < V; ++i) ahead[i][0] = weights(p.weight, me + i * tpr);
  const F2 inv = both(rsqrtf(row_sum(sum(s), slots[1], warp_row) * inv_d + p.eps));
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    F2 w[4];
    unpack8<ACT>(V <= 2 ? ahead[i][0] : weights(p.weight, v), w);
#pragma unroll
    for (int k = 0; k < 4; ++k) r[i][k] = r[i][k] * (inv * w[k]);
    const uint4 x = pack8<ACT>(r[i]);
    if (p.x) {
      if (v < nvec) *reinterpret_cast<uint4*>(p.x + t * p.ldx + v * 8) = x;
    } else {
      unpack8<ACT>(x, r[i]);  // what is cast is the rounded x: the codes are those of a cast of it
      if (v < nvec) bits = top_bits<ACT>(bits, x);
    }
  }
  if (!p.x) {
    float sf, qinv;
    int8_scale(__uint_as_float(row_max(top_value<ACT>(bits), reinterpret_cast<uint32_t*>(slots[2]), warp_row)), &sf, &qinv);
    if (me == 0) p.x_sf[t] = sf;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
      if (v < nvec) *reinterpret_cast<uint2*>(p.x_int + t * p.ldx + v * 8) = int8_codes(r[i], qinv);
    }
  }
}

// The same for many rows of 2056 to 4096 channels with a 16-bit residual: each CTA takes every gridDim.x-th row, keeps the weights of its
// threads' channels in registers and has the next rows copied to shared memory ahead of their turn; a row's reduction takes the next
// row's sum of block block along.  4096 x 4096, us, a CTA to each row / this: with both norms 28.3 / 25.2, with one 24.4 / 22.7, of
// a floor of 20.8.  (Wider rows and 32-bit residuals leave too few rows on an SM for that: 4097 x 8192 with a 32-bit one 69 / 84.)
template <int ACT>
__global__ void __launch_bounds__(256, 2) norm_rows_kernel(const NormParams p) {
  extern __shared__ __align__(16) unsigned char rows_smem[];
  __shared__ __align__(16) float slots[2][32], slots_block[32], slots_top[2][32];
  constexpr int V = 2;
  start_behind();
  if (threadIdx.x < 32) {  // (words of warps that are not there stay zero)
#pragma unroll
    for (int i = 0; i < 2; ++i) slots[i][threadIdx.x] = slots_top[i][threadIdx.x] = 0.f;
    slots_block[threadIdx.x] = 0.f;
  }
  __syncthreads();
  const int me = threadIdx.x, tpr = blockDim.x, nvec = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  const F2 zero = both(0.f), scale = both(p.scale);
  // [stage][block, residual][vector][thread], 16 bytes each
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(rows_smem) + (uint32_t)me * 16u;
  const uint32_t unit = (uint32_t)tpr * 16u, stage = unit * (2 * V), ring_end = ring + stage * NORM_ROWS_STAGES;
  auto at = [&](uint32_t s, int u, int i) { return s + unit * (uint32_t)(u * V + i); };
  auto load = [&](const unsigned short* from, int i) {
    const int v = me + i * tpr;
    return v < nvec ? *reinterpret_cast<const uint4*>(from + v * 8) : make_uint4(0, 0, 0, 0);
  };
  uint4 w_post[V], w_gate[V], w_norm[V];
  const bool one_gate = p.tokens_per_gate >= p.T;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (p.post) w_post[i] = load(p.post, i);
    if (p.gate && one_gate) w_gate[i] = load(p.gate, i);
    w_norm[i] = load(p.weight, i);
  }
  int ask = blockIdx.x;
  uint32_t ask_at = ring;
  auto fetch = [&]() {
    if (ask < p.T) {
      const char* b = reinterpret_cast<const char*>(p.block + ask * p.ldb) + me * 16;
      const char* r = static_cast<const char*>(p.residual) + (ask * p.ldr + me * 8) * 2;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (me + i * tpr < nvec) {
          copy16(at(ask_at, 0, i), b + i * unit);
          if (p.residual) copy16(at(ask_at, 1, i), r + i * unit);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ask += gridDim.x;
    ask_at = ask_at + stage == ring_end ? ring : ask_at + stage;
  };
  auto block_square = [&](uint32_t s) {
    F2 x = zero;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (me + i * tpr < nvec) {
        F2 b[4];
        unpack8<ACT>(lds_u4(at(s, 0, i)), b);
#pragma unroll
        for (int k = 0; k < 4; ++k) x = fma2(b[k], b[k], x);
      }
    return sum(x);
  };
  for (int n = 0; n < NORM_ROWS_STAGES - 1; ++n) fetch();
  float s1 = 1.f;
  if (p.post) {
    copies_wait<NORM_ROWS_STAGES - 2>();
    s1 = rsqrtf(row_sum(block_square(ring), slots_block, false) * inv_d + p.eps);
  }
  uint32_t s = ring;
  int turn = 0;
  for (int t = blockIdx.x; t < p.T; t += gridDim.x, turn ^= 1) {
    const uint32_t next = s + stage == ring_end ? ring : s + stage;
    fetch();
    copies_wait<NORM_ROWS_STAGES - 2>();
    const unsigned short* gate = p.gate ? p.gate + (t / p.tokens_per_gate) * p.ldg : nullptr;
    F2 r[V][4], rr = zero;
    const F2 s1_2 = both(s1);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
#pragma unroll
      for (int k = 0; k < 4; ++k) r[i][k] = zero;
      if (v < nvec) {
        F2 q[4];
        unpack8<ACT>(lds_u4(at(s, 0, i)), r[i]);
        if (p.post) {
          unpack8<ACT>(w_post[i], q);
#pragma unroll
          for (int k = 0; k < 4; ++k) r[i][k] = r[i][k] * (s1_2 * q[k]);
        }
        if (gate) {
          unpack8<ACT>(one_gate ? w_gate[i] : load(gate, i), q);
#pragma unroll
          for (int k = 0; k < 4; ++k) r[i][k] = r[i][k] * q[k];
        }
        if (p.residual) {
          unpack8<ACT>(lds_u4(at(s, 1, i)), q);
#pragma unroll
          for (int k = 0; k < 4; ++k) r[i][k] = fma2(scale, q[k], r[i][k]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) rr = fma2(r[i][k], r[i][k], rr);
        Wide<ACT, false>::store(p.new_residual, t * p.ldn + v * 8, r[i]);
      }
    }
    float x[2] = {sum(rr), p.post && t + (int)gridDim.x < p.T ? block_square(next) : 0.f};
    row_sum2(x, slots[turn]);
    const F2 inv = both(rsqrtf(x[0] * inv_d + p.eps));
    if (p.post) s1 = rsqrtf(x[1] * inv_d + p.eps);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
      F2 w[4];
      unpack8<ACT>(w_norm[i], w);
#pragma unroll
      for (int k = 0; k < 4; ++k) r[i][k] = r[i][k] * (inv * w[k]);
      const uint4 out = pack8<ACT>(r[i]);
      if (p.x) {
        if (v < nvec) *reinterpret_cast<uint4*>(p.x + t * p.ldx + v * 8) = out;
      } else {
        unpack8<ACT>(out, r[i]);
        if (v < nvec) bits = top_bits<ACT>(bits, out);
      }
    }
    if (!p.x) {
      float sf, qinv;
      int8_scale(__uint_as_float(row_max(top_value<ACT>(bits), reinterpret_cast<uint32_t*>(slots_top[turn]), false)), &sf, &qinv);
      if (me == 0) p.x_sf[t] = sf;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        if (v < nvec) *reinterpret_cast<uint2*>(p.x_int + t * p.ldx + v * 8) = int8_codes(r[i], qinv);
      }
    }
    s = next;
  }
  copies_wait<0>();
}

// ---- its gradient ---------------------------------------------------------------------------------------
// With s1, s2 the inverse deviations of the two norms, recomputed from the inputs (which have to be read anyway):
//   bh = block s1, q = bh post gate (= gate n);  r = scale residual + q;  xh = r s2;  e = grad_x weight
//   dr = grad_new + s2 (e - xh mean(e xh));   grad_residual = scale dr
//   grad_block = s1 (dr post gate - bh mean(dr q))      (dr gate without a norm after the block)
//   grad_weight = sum grad_x xh;   with S = sum dr bh over the rows of a gate: grad_gate = post S, grad_post = sum of gate S
// dr is linear in e and r, so that mean(dr q) follows from the row's sums of q grad_new, q e and q r, which can be taken together with
// those of r r and e r, and with the next row's sum of block block: one reduction over the CTA for each row.
//
// A CTA takes a run of rows of one gate and keeps its share of the sums over rows in registers; a second kernel adds the CTAs' shares
// in a fixed order, so that a call gives the same bits each time.  Rows are copied to shared memory ahead of their turn
// by the copy engine.  8192 x 5120 with a 32-bit residual and 8 gates takes 148 us (5.1 TB/s; with a row at a time in registers and three
// reductions 386), 511 x 4096 with a gate 13.9: what bounds it is the latency of a row's reduction between its copies and its outputs, at
// as many rows on an SM as registers allow.
// The sums of eight values over the CTA's threads, in every thread.  Halving exchanges: after the steps over 16, 8 and 4 lanes a lane
// holds one value, lane >> 2; so a warp's part takes 9 shuffles instead of 40.  `slots`: 8 words a warp, of two sets in turn.
__device__ __forceinline__ void sums8(float (&v)[8], float* slots) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float give = lane & 16 ? v[i] : v[i + 4], mine = lane & 16 ? v[i + 4] : v[i];
    v[i] = mine + __shfl_xor_sync(0xffffffffu, give, 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float give = lane & 8 ? v[i] : v[i + 2], mine = lane & 8 ? v[i + 2] : v[i];
    v[i] = mine + __shfl_xor_sync(0xffffffffu, give, 8);
  }
  const float give = lane & 4 ? v[0] : v[1], mine = lane & 4 ? v[1] : v[0];
  float x = mine + __shfl_xor_sync(0xffffffffu, give, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 2);
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  if ((lane & 3) == 0) slots[warp * 8 + (lane >> 2)] = x;
  __syncthreads();
  x = 0.f;
  for (int w = lane >> 3; w < warps; w += 4) x += slots[w * 8 + (lane & 7)];
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  x += __shfl_xor_sync(0xffffffffu, x, 16);
#pragma unroll
  for (int i = 0; i < 6; ++i) v[i] = __shfl_sync(0xffffffffu, x, i);
}

// V: vectors of eight channels to a thread.  Up to two, the weights of a thread's channels stay in registers too.
template <int ACT, bool F32, int V>
__global__ void __launch_bounds__(NORM_BACK_THREADS) norm_backward_kernel(const NormBackwardParams p) {
  extern __shared__ __align__(16) unsigned char rows_smem[];  // [stage]: a row of block, grad_x, residual, grad_new
  __shared__ __align__(16) float slots[2][8 * (NORM_BACK_THREADS / 32)], slots_block[1][32];
  __shared__ uint64_t landed[NORM_BACK_STAGES];
  __shared__ int gave_up, run_start, run_asked;  // (the rows of the runs before thread 0's latest, and those of it that it has asked for)
  constexpr int RB = F32 ? 4 : 2;
  constexpr bool KEEP = V <= 2;
  start_behind();
  clear_slots(slots_block);
  const int me = threadIdx.x, tpr = blockDim.x, nvec = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  const F2 zero = both(0.f), scale = both(p.scale);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(rows_smem), landed_s = (uint32_t)__cvta_generic_to_shared(landed);
  const uint32_t row16 = (uint32_t)p.D * 2u, row_wide = (uint32_t)p.D * RB, stage = 2u * row16 + 2u * row_wide;
  if (me == 0) {
    for (int i = 0; i < p.stages; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(landed_s + (uint32_t)i * 8u) : "memory");
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  auto load = [&](const unsigned short* from, int i, F2 (&w)[4]) {
    const int v = me + i * tpr;
    unpack8<ACT>(v < nvec ? *reinterpret_cast<const uint4*>(from + v * 8) : make_uint4(0, 0, 0, 0), w);
  };
  // what stands in front of a row's block in the new residual: post and gate together
  auto load_pg = [&](int g, int i, F2 (&pg)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) pg[k] = both(1.f);
    if (p.post) load(p.post, i, pg);
    if (p.gate) {
      F2 x[4];
      load(p.gate + g * p.ldg, i, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) pg[k] = pg[k] * x[k];
    }
  };
  auto block_square = [&](uint32_t s) {
    F2 x = zero;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (me + i * tpr < nvec) {
        F2 b[4];
        unpack8<ACT>(lds_u4(s + (uint32_t)(me + i * tpr) * 16u), b);
#pragma unroll
        for (int k = 0; k < 4; ++k) x = fma2(b[k], b[k], x);
      }
    return sum(x);
  };
  auto wide = [&](const void* there, uint32_t from, int v, F2 (&f)[4]) {
    Wide<ACT, F32> w;
    w.zero();
    if (there)
#pragma unroll
      for (int h = 0; h < Wide<ACT, F32>::UNITS; ++h) w.v[h] = lds_u4(from + (uint32_t)v * (8u * RB) + (uint32_t)h * 16u);
    w.get(f);
  };
  F2 kept_w[KEEP ? V : 1][4], kept_pg[KEEP ? V : 1][4], gw[V][4], S[V][4];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (KEEP) load(p.weight, i, kept_w[i]);
#pragma unroll
    for (int k = 0; k < 4; ++k) gw[i][k] = zero;
  }
  // Three stages and more: a row's reduction takes the next row's sum of block block along, whose copies have landed by then.
  const bool ahead = p.stages >= 3;
  const int part = (int)(blockIdx.x % p.ctas_per_gate), stride = (int)(gridDim.x / p.ctas_per_gate);
  bool first_gate = true, good = true;
  int lap = 0, at = 0;  // of the next row to be read: how often its stage has been used, and which
  for (int g = blockIdx.x / p.ctas_per_gate; g < p.gates; g += stride, first_gate = false) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (KEEP) load_pg(g, i, kept_pg[i]);
#pragma unroll
      for (int k = 0; k < 4; ++k) S[i][k] = zero;
    }
    const int r0 = (int)((long long)p.tokens_per_gate * part / p.ctas_per_gate);
    const int rows = (int)((long long)p.tokens_per_gate * (part + 1) / p.ctas_per_gate) - r0;
    const long long t0 = (long long)g * p.tokens_per_gate + r0;
    long long to_b = t0 * p.lddb + me * 8, to_r = t0 * p.lddr + me * 8;
    // Thread 0 asks for rows, in order, the stages in turn from this run's first.
    int asked = 0, ask_stage = at;
    auto fetch = [&]() {
      if (asked >= rows || !good) return;  // (once thread 0 has given up, no stage is asked for again)
      const long long t = t0 + asked;
      const uint32_t bar = landed_s + (uint32_t)ask_stage * 8u, to = ring + (uint32_t)ask_stage * stage;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                   "r"(2u * row16 + (p.residual ? row_wide : 0u) + (p.grad_new ? row_wide : 0u)) : "memory");
      copy_row(to, p.block + t * p.ldb, row16, bar);
      copy_row(to + row16, p.grad_x + t * p.lddx, row16, bar);
      if (p.residual) copy_row(to + 2u * row16, static_cast<const char*>(p.residual) + t * p.ldr * RB, row_wide, bar);
      if (p.grad_new) copy_row(to + 2u * row16 + row_wide, static_cast<const char*>(p.grad_new) + t * p.lddn * RB, row_wide, bar);
      run_asked = ++asked;
      if (++ask_stage == p.stages) ask_stage = 0;
    };
    // A thread that has given up waits no more, but keeps in step with the others; its part of this row's and all later rows'
    // reductions is no number, and so is what they give: the rows' gradients and the CTA's shares of all sums.
    auto await = [&](int stage_i, int lap_i) {
      if (good && !mbar_wait_bounded(landed_s + (uint32_t)stage_i * 8u, (uint32_t)lap_i & 1u)) {
        good = false;
        gave_up = 1;
      }
    };
    if (me == 0 && good) {
      run_start = lap * p.stages + at;
      run_asked = 0;
      for (int n = 0; n < p.stages; ++n) fetch();
    }
    float s1 = 1.f;
    if (ahead && p.post && rows > 0) {
      await(at, lap);
      s1 = rsqrtf(row_sum(block_square(ring + (uint32_t)at * stage), slots_block[0], false) * inv_d + p.eps);
    }
    for (int n = 0; n < rows; ++n) {
      const uint32_t s = ring + (uint32_t)at * stage;
      const int next = at + 1 == p.stages ? 0 : at + 1, next_lap = at + 1 == p.stages ? lap + 1 : lap;
      if (!(ahead && p.post)) await(at, lap);  // (else the last row's turn has waited for it)
      if (!ahead && p.post) s1 = rsqrtf(row_sum(block_square(s), slots_block[0], false) * inv_d + p.eps);
      F2 rr = zero, er = zero, qn = zero, qe = zero, qr = zero;
      const F2 s1_2 = both(s1);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        if (v < nvec) {
          F2 b[4], d[4], res[4], dn[4], w[4], pg[4];
          unpack8<ACT>(lds_u4(s + (uint32_t)v * 16u), b);
          unpack8<ACT>(lds_u4(s + row16 + (uint32_t)v * 16u), d);
          wide(p.residual, s + 2u * row16, v, res);
          wide(p.grad_new, s + 2u * row16 + row_wide, v, dn);
          if constexpr (!KEEP) { load(p.weight, i, w); load_pg(g, i, pg); }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const F2 q = (b[k] * s1_2) * (KEEP ? kept_pg[KEEP ? i : 0][k] : pg[k]), e = d[k] * (KEEP ? kept_w[KEEP ? i : 0][k] : w[k]);
            const F2 r = fma2(scale, res[k], q);
            rr = fma2(r, r, rr);
            er = fma2(e, r, er);
            qn = fma2(q, dn[k], qn);
            qe = fma2(q, e, qe);
            qr = fma2(q, r, qr);
          }
        }
      }
      float x[8] = {good ? sum(rr) : __int_as_float(0x7fc00000), sum(er), sum(qn), sum(qe), sum(qr), 0.f, 0.f, 0.f};
      if (ahead && p.post && n + 1 < rows) {
        await(next, next_lap);
        x[5] = block_square(ring + (uint32_t)next * stage);
      }
      sums8(x, slots[n & 1]);
      if (me == 0 && n > 0 && p.stages > 1) fetch();  // every thread is done with the row before this one
      const float s2 = rsqrtf(x[0] * inv_d + p.eps), mean = x[1] * s2 * inv_d;                       // of e xh
      const float mean_q = p.post ? (x[2] + s2 * (x[3] - s2 * mean * x[4])) * inv_d : 0.f;           // of dr q
      const F2 s2_2 = both(s2), mean_2 = both(-mean), mean_q2 = both(-mean_q);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        if (v < nvec) {
          F2 b[4], d[4], res[4], dn[4], w[4], pg[4], out[4];
          unpack8<ACT>(lds_u4(s + (uint32_t)v * 16u), b);
          unpack8<ACT>(lds_u4(s + row16 + (uint32_t)v * 16u), d);
          wide(p.residual, s + 2u * row16, v, res);
          wide(p.grad_new, s + 2u * row16 + row_wide, v, dn);
          if constexpr (!KEEP) { load(p.weight, i, w); load_pg(g, i, pg); }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const F2 m = KEEP ? kept_pg[KEEP ? i : 0][k] : pg[k];
            const F2 bh = b[k] * s1_2, xh = fma2(scale, res[k], bh * m) * s2_2;
            gw[i][k] = fma2(d[k], xh, gw[i][k]);
            const F2 dr = fma2(s2_2, fma2(mean_2, xh, d[k] * (KEEP ? kept_w[KEEP ? i : 0][k] : w[k])), dn[k]);
            S[i][k] = fma2(dr, bh, S[i][k]);
            res[k] = scale * dr;
            out[k] = s1_2 * fma2(mean_q2, bh, dr * m);
          }
          if (p.grad_residual) Wide<ACT, F32>::store(p.grad_residual, to_r + i * tpr * 8, res);
          *reinterpret_cast<uint4*>(p.grad_block + to_b + i * tpr * 8) = pack8<ACT>(out);
        }
      }
      to_b += p.lddb; to_r += p.lddr;
      if (ahead && p.post) s1 = rsqrtf(x[5] * inv_d + p.eps);
      at = next;
      lap = next_lap;
      if (p.stages == 1) {  // the next row goes where this one was
        __syncthreads();
        if (me == 0) fetch();
      }
    }
    // S: as it is where CTAs share the gate, whose sums the second kernel takes apart; else the gate's own gradient, and what its rows
    // give post.
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
      if (v >= nvec) continue;
      const long long to = ((long long)p.grid + blockIdx.x) * p.D + v * 8;
      if (p.ctas_per_gate > 1) {
        if (p.post || p.grad_gate) Wide<ACT, true>::store(p.partial, to, S[i]);
        continue;
      }
      F2 x[4];
      if (p.grad_gate) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = both(1.f);
        if (p.post) load(p.post, i, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = x[k] * S[i][k];
        Wide<ACT, true>::store(p.grad_gate + (long long)g * p.D, v * 8, x);
      }
      if (p.post) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = both(1.f);
        if (p.gate) load(p.gate + g * p.ldg, i, x);
        Wide<ACT, true> sofar;
        F2 y[4];
        sofar.zero();
        if (!first_gate) sofar.load(p.partial, to);
        sofar.get(y);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = fma2(x[k], S[i][k], y[k]);
        Wide<ACT, true>::store(p.partial, to, x);
      }
    }
    __syncthreads();  // the stages and slots of this run's last row have been read
  }
  if (gave_up) {
    // The copies in flight get their chance to land before the CTA ends.
    if (me == 0) {
      ring_drain(landed_s, p.stages, run_start + run_asked);
      atomicExch(p.status, ST_DEVICE_TIMEOUT);
      p.status[1] = 14;  // where: gradient of the block norm
      p.status[2] = blockIdx.x;
      p.status[3] = 0;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    if (v < nvec) Wide<ACT, true>::store(p.partial, (long long)blockIdx.x * p.D + v * 8, gw[i]);
  }
}

// The sums of the CTAs' shares: 32 columns a CTA (pairs of columns from 4104 on, so that all
// CTAs run at once: 148 x 8192 with a 32-bit residual 13.5 / 12.9 us), 24 runs of shares side by
// side, joined in order.  A thread's loads, which come from L2, are under way together: seven are a CTA to each SM.  (511 x 4096, us for
// the whole gradient: 8 runs and a loop unrolled ten times, whose rest went one by one, 15.7; 8 runs in tens 14.4, 16 in tens 13.3,
// 24 in sevens 12.7.)  blockIdx.y: grad_weight, grad_post and up to 24 gates, whose runs are the fewer the more they are; more
// gates after that.  (Quotients by products: several divisions of a thread's cost 0.3 us.)
constexpr int SUMS_RUNS = 24, SUMS_BATCH = 7;
template <int C>
struct Cols {  // a thread's columns
  float v[C];
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (C == 2) {
      const float2 t = *reinterpret_cast<const float2*>(p);
      v[0] = t.x; v[1] = t.y;
    } else {
      v[0] = *p;
    }
  }
  template <int ACT>
  __device__ __forceinline__ void load16(const unsigned short* p) {
    if constexpr (C == 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
      if constexpr (ACT == 0) {
        const float2 t = __half22float2(h2_from_bits(w));
        v[0] = t.x; v[1] = t.y;
      } else {
        v[0] = __uint_as_float(w << 16); v[1] = __uint_as_float(w & 0xffff0000u);
      }
    } else {
      v[0] = ACT == 0 ? __half2float(__ushort_as_half(*p)) : __uint_as_float((uint32_t)*p << 16);
    }
  }
  __device__ __forceinline__ void store(float* p) const {
    if constexpr (C == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    else *p = v[0];
  }
  __device__ __forceinline__ void set(float x) {
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = x;
  }
  __device__ __forceinline__ Cols operator*(const Cols& o) const {
    Cols r;
#pragma unroll
    for (int c = 0; c < C; ++c) r.v[c] = v[c] * o.v[c];
    return r;
  }
  __device__ __forceinline__ void operator+=(const Cols& o) {
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] += o.v[c];
  }
};
// Run `part` of n shares at `from`, `weigh(share, values)` in between.  The runs meet at n * part / (runs), taken as a product with `per` =
// 65536 / runs + 1 (up to a few thousand shares the last one ends at n: the product is too large by less than one).
template <int C, class Weigh>
__device__ __forceinline__ Cols<C> sum_run(const float* from, int n, int part, int per, long long D, Weigh weigh) {
  Cols<C> s;
  s.set(0.f);
  const int i1 = (int)((unsigned)(n * (part + 1)) * (unsigned)per >> 16);
  for (int i = (int)((unsigned)(n * part) * (unsigned)per >> 16); i < i1; i += SUMS_BATCH) {
    Cols<C> x[SUMS_BATCH];
#pragma unroll
    for (int j = 0; j < SUMS_BATCH; ++j) {
      x[j].set(0.f);
      if (i + j < i1) {
        x[j].load(from + (i + j) * D);
        weigh(i + j, x[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < SUMS_BATCH; ++j) s += x[j];
  }
  return s;
}
// GATES: 0 one gate, none or CTAs that leave nothing for several to be done; else CTAs share several gates, 1 up to 24, 2 more.
template <int ACT, int GATES, int C>
__global__ void __launch_bounds__(SUMS_RUNS * 32, 2) norm_sums_kernel(const NormBackwardParams p) {
  __shared__ Cols<C> sums[SUMS_RUNS][33];
  start_behind();
  const int which = (int)blockIdx.y, lane = threadIdx.x & 31, col = ((int)blockIdx.x * 32 + lane) * C, run = threadIdx.x >> 5;
  const bool there = col < p.D;
  auto value = [&](const unsigned short* from) {
    Cols<C> x;
    x.template load16<ACT>(from + col);
    return x;
  };
  const auto as_is = [](int, Cols<C>&) {};
  constexpr int PER = 65536 / SUMS_RUNS + 1;
  const float* from = p.partial + (which == 0 ? 0ll : (long long)p.grid * p.D) + col;
  if (GATES == 0 || which == 0 || (GATES == 2 && which == 1)) {
    Cols<C> s;
    s.set(0.f);
    if (GATES == 2 && which == 1) {
      if (there)
        s = sum_run<C>(from, p.grid, run, PER, p.D, [&](int i, Cols<C>& x) { x = x * value(p.gate + (i * p.gate_per >> 16) * p.ldg); });
    } else {
      if (there) s = sum_run<C>(from, p.grid, run, PER, p.D, as_is);
    }
    sums[run][lane] = s;
    __syncthreads();
    if (run > 0 || !there) return;
#pragma unroll 12
    for (int i = 1; i < SUMS_RUNS; ++i) s += sums[i][lane];
    if (which == 0) {
      s.store(p.grad_weight + col);
    } else {
      const bool one_gate = GATES == 0 && p.gate && p.ctas_per_gate > 1;
      if (p.post) (one_gate ? s * value(p.gate) : s).store(p.grad_post + col);
      if (one_gate) (p.post ? s * value(p.post) : s).store(p.grad_gate + col);
    }
    return;
  }
  if constexpr (GATES > 0) {
    const int runs = p.sums_runs, at = run * p.sums_per >> 16, part = run - at * runs;
    const int g = (GATES == 2 ? (which - 2) * SUMS_RUNS : 0) + at, n = p.ctas_per_gate;
    const bool mine = there && g < p.gates;
    Cols<C> s;
    s.set(0.f);
    if (mine) s = sum_run<C>(from + (long long)g * n * p.D, n, part, p.sums_per, p.D, as_is);
    sums[run][lane] = s;
    __syncthreads();
    const bool first = part == 0 && mine;
    if (first) {
#pragma unroll 12
      for (int i = 1; i < SUMS_RUNS; ++i)
        if (i < runs) s += sums[run + i < SUMS_RUNS ? run + i : 0][lane];
      (p.post ? s * value(p.post) : s).store(p.grad_gate + (long long)g * p.D + col);
    }
    if (GATES == 2 || !p.post) return;
    if (first) s = s * value(p.gate + g * p.ldg);
    __syncthreads();
    if (first) sums[at][lane] = s;
    __syncthreads();
    if (run > 0 || !there) return;
    for (int i = 1; i < p.gates; ++i) s += sums[i][lane];
    s.store(p.grad_post + col);
  }
}

// ---- launches ---------------------------------------------------------------------------------------------
template <class Kernel, class... Args>
static cudaError_t launch_behind(Kernel kern, dim3 grid, int threads, int smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Threads of a row and vectors of a thread: a warp for up to 512 channels (2048 where rows are many), else a CTA.  Where rows are many,
// 256 threads with up to eight vectors, so that the steps of a reduction are shared by many channels; where they are few, as many as the row has.
struct RowShape { int warp_rows, threads, vectors, ctas; };
static RowShape row_shape(int T, int D) {
  const int nvec = D / 8;
  RowShape s;
  s.warp_rows = nvec <= (T > 1024 ? 256 : 64) ? 1 : 0;
  if (s.warp_rows) {
    s.vectors = nvec <= 32 ? 1 : nvec <= 64 ? 2 : nvec <= 128 ? 4 : 8;
    s.threads = 128;
    s.ctas = T / 4 + (T % 4 != 0);
    return s;
  }
  // (us for 4096 rows, 256 threads / 512.  32-bit residual: 5120 channels 42.3 / 39.1, 6144 54.1 / 48.4, 7168 59.3 / 54.3, 8192 65.4 / 61.0,
  // 8200 82.0 / 92.0.  16-bit: 33.5 / 38.3 for 6144, 38.8 / 42.0 for 7168, 43.5 / 45.6 for 8192, 51.0 / 46.0 for 8200.  So the band is right
  // for 32-bit residuals, could begin lower there, and costs 16-bit ones up to a tenth.)
  const int threads = T <= 296 || (nvec > 768 && nvec <= 1024) ? 512 : 256;
  s.vectors = 1;
  while (s.vectors < 8 && s.vectors * threads < nvec) s.vectors *= 2;
  const int per = (nvec + s.vectors - 1) / s.vectors;
  s.threads = (per + 31) / 32 * 32;
  if (s.threads > 512) s.threads = 512;
  s.ctas = T;
  return s;
}

template <int ACT>
static cudaError_t cast_int_act(const CastIntParams& p, cudaStream_t stream) {
  const RowShape s = row_shape(p.T, p.D);
  const dim3 grid((unsigned)s.ctas, 1, 1);
  switch (s.vectors) {
    case 1: return launch_behind(cast_int_kernel<ACT, 1>, grid, s.threads, 0, stream, p, s.warp_rows);
    case 2: return launch_behind(cast_int_kernel<ACT, 2>, grid, s.threads, 0, stream, p, s.warp_rows);
    case 4: return launch_behind(cast_int_kernel<ACT, 4>, grid, s.threads, 0, stream, p, s.warp_rows);
    default: return launch_behind(cast_int_kernel<ACT, 8>, grid, s.threads, 0, stream, p, s.warp_rows);
  }
}
cudaError_t cast_int_launch(const CastIntParams& p, int act, cudaStream_t stream) {
  return act == 0 ? cast_int_act<0>(p, stream) : cast_int_act<1>(p, stream);
}

template <int ACT>
static cudaError_t norm_rows(NormParams p, int threads, cudaStream_t stream) {
  static std::atomic<bool> allowed[16];
  const cudaError_t e = allow_smem(norm_rows_kernel<ACT>, allowed);
  if (e != cudaSuccess) return e;
  const int most = 2 * p.sms;  // two CTAs to an SM, by registers and shared memory
  return launch_behind(norm_rows_kernel<ACT>, dim3((unsigned)(p.T < most ? p.T : most), 1, 1), threads,
                       NORM_ROWS_STAGES * 2 * 2 * threads * 16, stream, p);
}
template <int ACT, bool F32>
static cudaError_t norm_type(const NormParams& p, cudaStream_t stream) {
  const int nvec = p.D / 8;
  if constexpr (!F32)
    if (nvec > 256 && nvec <= 512 && p.T >= NORM_ROWS_FROM) return norm_rows<ACT>(p, (nvec + 63) / 64 * 32, stream);
  const RowShape s = row_shape(p.T, p.D);
  const dim3 grid((unsigned)s.ctas, 1, 1);
  switch (s.vectors) {
    case 1: return launch_behind(norm_kernel<ACT, F32, 1>, grid, s.threads, 0, stream, p, s.warp_rows);
    case 2: return launch_behind(norm_kernel<ACT, F32, 2>, grid, s.threads, 0, stream, p, s.warp_rows);
    case 4: return launch_behind(norm_kernel<ACT, F32, 4>, grid, s.threads, 0, stream, p, s.warp_rows);
    default: return launch_behind(norm_kernel<ACT, F32, 8>, grid, s.threads, 0, stream, p, s.warp_rows);
  }
}
cudaError_t norm_launch(const NormParams& p, int act, bool residual_f32, cudaStream_t stream) {
  if (act == 0) return residual_f32 ? norm_type<0, true>(p, stream) : norm_type<0, false>(p, stream);
  return residual_f32 ? norm_type<1, true>(p, stream) : norm_type<1, false>(p, stream);
}

template <int ACT, bool F32, int V>
static cudaError_t backward_rows(const NormBackwardParams& p, cudaStream_t stream) {
  static std::atomic<bool> allowed[16];
  const cudaError_t e = allow_smem(norm_backward_kernel<ACT, F32, V>, allowed);
  if (e != cudaSuccess) return e;
  return launch_behind(norm_backward_kernel<ACT, F32, V>, dim3((unsigned)p.grid, 1, 1), p.threads, p.smem, stream, p);
}
template <int ACT, int C>
static cudaError_t sums_launch(const NormBackwardParams& p, int rows, int kind, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.D + 32 * C - 1) / (32 * C)), (unsigned)rows, 1);
  if (kind == 0) return launch_behind(norm_sums_kernel<ACT, 0, C>, grid, SUMS_RUNS * 32, 0, stream, p);
  if (kind == 1) return launch_behind(norm_sums_kernel<ACT, 1, C>, grid, SUMS_RUNS * 32, 0, stream, p);
  return launch_behind(norm_sums_kernel<ACT, 2, C>, grid, SUMS_RUNS * 32, 0, stream, p);
}
template <int ACT, bool F32>
static cudaError_t backward_type(NormBackwardParams p, cudaStream_t stream) {
  p.sums_runs = p.gates < SUMS_RUNS ? SUMS_RUNS / p.gates : 1;
  p.sums_per = 65536 / p.sums_runs + 1;
  p.gate_per = 65536 / p.ctas_per_gate + 1;
  cudaError_t e;
  switch (p.vectors) {
    case 1: e = backward_rows<ACT, F32, 1>(p, stream); break;
    case 2: e = backward_rows<ACT, F32, 2>(p, stream); break;
    default: e = backward_rows<ACT, F32, 4>(p, stream); break;
  }
  if (e != cudaSuccess) return e;
  const bool shared = p.ctas_per_gate > 1;
  const int post = p.post || (shared && p.grad_gate) ? 2 : 1, more = (p.gates + SUMS_RUNS - 1) / SUMS_RUNS;
  const int rows = shared && p.gates > SUMS_RUNS ? 2 + more : post, kind = !shared || p.gates == 1 ? 0 : p.gates <= SUMS_RUNS ? 1 : 2;
  return p.D > 4096 ? sums_launch<ACT, 2>(p, rows, kind, stream) : sums_launch<ACT, 1>(p, rows, kind, stream);
}
// The shape of the gradient's launch: threads and vectors of a row, CTAs (512 threads to an SM), and stages for the rows ahead.
void norm_backward_shape(int D, bool residual_f32, int gates, int tokens_per_gate, int sms, int max_smem, NormBackwardParams* p) {
  const int nvec = D / 8;
  const bool few = (long long)gates * tokens_per_gate <= 12ll * sms;
  p->vectors = nvec <= (few ? 512 : 256) ? 1 : nvec <= 1024 ? 2 : 4;
  p->threads = ((nvec + p->vectors - 1) / p->vectors + 31) / 32 * 32;
  const int per_sm = NORM_BACK_THREADS / p->threads < 8 ? NORM_BACK_THREADS / p->threads : 8, most = sms * per_sm;
  // Runs that a gate's rows are enough for: a row each where the SMs are as many, else two, since a CTA's sums over rows are as many bytes
  // as six rows.  (us, two rows each / one: 8 x 4096 9.3 / 7.9, 148 x 4096 10.3 / 8.9, 296 x 1024 7.4 / 7.7.)
  const int single = sms / gates < tokens_per_gate ? sms / gates : tokens_per_gate, twos = tokens_per_gate / 2 + tokens_per_gate % 2;
  const int runs = single > twos ? single : twos;
  if (gates >= most) {
    p->ctas_per_gate = 1;
    p->grid = most;
  } else {
    p->ctas_per_gate = most / gates < runs ? most / gates : runs;
    p->grid = gates * p->ctas_per_gate;
  }
  const int stage = D * (residual_f32 ? 12 : 8), room = (max_smem + 1024) / per_sm - 1024 - 2048;
  p->stages = room / stage > NORM_BACK_STAGES ? NORM_BACK_STAGES : room / stage;
  p->smem = p->stages * stage;
}
cudaError_t norm_backward_launch(const NormBackwardParams& p, int act, bool residual_f32, cudaStream_t stream) {
  if (act == 0) return residual_f32 ? backward_type<0, true>(p, stream) : backward_type<0, false>(p, stream);
  return residual_f32 ? backward_type<1, true>(p, stream) : backward_type<1, false>(p, stream);
}

}  // namespace b200q
