// Row-wise kernels between the products of a decoder block: the per-token int8 cast, and the norms before and after a
// block with its gate and residual scale (norm.cuh has the formulas), forward and backward.
//
// All are bound by memory: each input is read once and each output written once, with a row held in registers between the
// statistics and their use.  Threads own vectors of eight neighbouring channels (16 bytes of a 16-bit type).  Sums and statistics
// are fp32; the only roundings to fewer bits are those of the outputs.
#include "norm.cuh"

namespace b200q {

// The kernel before this one in the stream has ended; the one behind it may set up now, and no earlier: what it reads before this
// one has ended (weights) is then at least one kernel old.
__device__ __forceinline__ void start_behind() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <int ACT>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (ACT == 0) {
      const float2 t = __half22float2(h2_from_bits(w[i]));
      f[2 * i] = t.x; f[2 * i + 1] = t.y;
    } else {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int ACT>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<ACT>(f[0], f[1]), pack2<ACT>(f[2], f[3]), pack2<ACT>(f[4], f[5]), pack2<ACT>(f[6], f[7]));
}

// eight values of the residual stream, of the activation type or fp32
template <int ACT, bool F32>
struct Wide {
  uint4 v[F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* base, long long at) {
    if constexpr (F32) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + at);
      v[0] = p[0]; v[1] = p[1];
    } else {
      v[0] = *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(base) + at);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (F32 ? 2 : 1); ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (F32) {
      const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    } else {
      unpack8<ACT>(v[0], f);
    }
  }
  static __device__ __forceinline__ void store(void* base, long long at, const float (&f)[8]) {
    if constexpr (F32) {
      float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
      p[0] = make_float4(f[0], f[1], f[2], f[3]);
      p[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<unsigned short*>(base) + at) = pack8<ACT>(f);
    }
  }
};

// Sum (or, with MAX, unsigned maximum) of N values over the threads of a row: a warp, or all warps of the CTA.  `slots`: 32 * N words
// that no other reduction uses until the next barrier but one; every thread gets the same result in the same order.
template <int N, bool MAX>
__device__ __forceinline__ void row_reduce(float (&v)[N], float* slots, bool warp_row) {
  auto join = [](float a, float b) {
    return MAX ? __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))) : a + b;
  };
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] = join(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
  if (warp_row) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) slots[warp * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lane < warps ? slots[lane * N + i] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] = join(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
  }
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
// Codes of eight values: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves its low byte in the sum's.
__device__ __forceinline__ uint2 int8_codes(const float (&f)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[4 * h + i], inv), 12582912.0f));
    w[h] = inv != 0.0f ? __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) : 0u;
  }
  return make_uint2(w[0], w[1]);
}
// The largest magnitude among 16-bit values, as bits (either type's order like integers, NaN above infinity), two at a time.
__device__ __forceinline__ uint32_t top_bits(uint32_t top, const uint4& v) {
  top = __vmaxu2(__vmaxu2(top, v.x & 0x7fff7fffu), v.y & 0x7fff7fffu);
  return __vmaxu2(__vmaxu2(top, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu);
}
template <int ACT>
__device__ __forceinline__ float top_value(uint32_t top) {
  const uint32_t one = max(top & 0xffffu, top >> 16);
  return ACT == 0 ? __half2float(__ushort_as_half((unsigned short)one)) : __uint_as_float(one << 16);
}

template <int ACT, int V>
__global__ void __launch_bounds__(1024) cast_int_kernel(const CastIntParams p, const int warp_rows) {
  __shared__ float slots[32];
  start_behind();
  const bool warp_row = warp_rows != 0;
  const int tpr = warp_row ? 32 : blockDim.x, me = warp_row ? threadIdx.x & 31 : threadIdx.x;
  const int t = warp_row ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (t >= p.T) return;  // (whole warps, and only where a warp has its own row)
  const int nvec = p.D / 8;
  const uint4* row = reinterpret_cast<const uint4*>(p.x + (size_t)t * p.ldx);
  uint4 keep[V];
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    keep[i] = v < nvec ? row[v] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) bits = top_bits(bits, keep[i]);
  for (int v = me + V * tpr; v < nvec; v += tpr) bits = top_bits(bits, row[v]);  // (what does not stay in registers is read again)
  float top[1] = {top_value<ACT>(bits)};
  row_reduce<1, true>(top, slots, warp_row);
  float sf, inv;
  int8_scale(top[0], &sf, &inv);
  if (me == 0) p.out_sf[t] = sf;
  uint2* out = reinterpret_cast<uint2*>(p.out + (size_t)t * p.ldo);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    float f[8];
    unpack8<ACT>(keep[i], f);
    if (v < nvec) out[v] = int8_codes(f, inv);
  }
  for (int v = me + V * tpr; v < nvec; v += tpr) {
    float f[8];
    unpack8<ACT>(row[v], f);
    out[v] = int8_codes(f, inv);
  }
}

// ---- block norm -------------------------------------------------------------------------------------------
template <int ACT, bool F32, int V>
__global__ void __launch_bounds__(1024) norm_kernel(const NormParams p, const int warp_rows) {
  __shared__ float slots[3][32];
  start_behind();
  const bool warp_row = warp_rows != 0;
  const int tpr = warp_row ? 32 : blockDim.x, me = warp_row ? threadIdx.x & 31 : threadIdx.x;
  const int t = warp_row ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (t >= p.T) return;
  const int nvec = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  float r[V][8];  // block, then the new residual, then x
  Wide<ACT, F32> res[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    uint4 b = make_uint4(0, 0, 0, 0);
    res[i].zero();
    if (v < nvec) {
      b = *reinterpret_cast<const uint4*>(p.block + t * p.ldb + v * 8);
      if (p.residual) res[i].load(p.residual, t * p.ldr + v * 8);
    }
    unpack8<ACT>(b, r[i]);
  }
  if (p.post) {
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[0] += r[i][k] * r[i][k];
    row_reduce<1, false>(s, slots[0], warp_row);
    const float inv = rsqrtf(s[0] * inv_d + p.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
      if (v < nvec) {
        float w[8];
        unpack8<ACT>(*reinterpret_cast<const uint4*>(p.post + v * 8), w);
#pragma unroll
        for (int k = 0; k < 8; ++k) r[i][k] *= inv * w[k];
      }
    }
  }
  const unsigned short* gate = p.gate ? p.gate + (t / p.tokens_per_gate) * p.ldg : nullptr;
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    float q[8];
    if (gate && v < nvec) {
      unpack8<ACT>(*reinterpret_cast<const uint4*>(gate + v * 8), q);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[i][k] *= q[k];
    }
    res[i].get(q);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      r[i][k] += p.scale * q[k];
      s[0] += r[i][k] * r[i][k];
    }
    if (v < nvec) Wide<ACT, F32>::store(p.new_residual, t * p.ldn + v * 8, r[i]);
  }
  row_reduce<1, false>(s, slots[1], warp_row);
  const float inv = rsqrtf(s[0] * inv_d + p.eps);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    if (v < nvec) {
      float w[8];
      unpack8<ACT>(*reinterpret_cast<const uint4*>(p.weight + v * 8), w);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[i][k] *= inv * w[k];
      const uint4 x = pack8<ACT>(r[i]);
      if (p.x) {
        *reinterpret_cast<uint4*>(p.x + t * p.ldx + v * 8) = x;
      } else {
        unpack8<ACT>(x, r[i]);  // what is cast is the rounded x: the codes are those of a cast of it
        bits = top_bits(bits, x);
      }
    }
  }
  if (!p.x) {
    float top[1] = {top_value<ACT>(bits)};
    row_reduce<1, true>(top, slots[2], warp_row);
    float sf, qinv;
    int8_scale(top[0], &sf, &qinv);
    if (me == 0) p.x_sf[t] = sf;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
      if (v < nvec) *reinterpret_cast<uint2*>(p.x_int + t * p.ldx + v * 8) = int8_codes(r[i], qinv);
    }
  }
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
// (cp.async, each thread what it will read itself, so that nobody waits for anybody's copies): with a row at a time in registers and three
// reductions 8192 x 5120 took 386 us, of a floor of 117.
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_wait(int pending) {  // all but the latest `pending` groups have landed
  if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 2;" ::: "memory");
}

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
  for (int i = 0; i < 8; ++i) v[i] = __shfl_sync(0xffffffffu, x, i);
}

// V: vectors of eight channels to a thread.  Up to two, the weights of a thread's channels stay in registers too.
template <int ACT, bool F32, int V>
__global__ void __launch_bounds__(512) norm_backward_kernel(const NormBackwardParams p) {
  extern __shared__ __align__(16) unsigned char rows_smem[];
  __shared__ float slots[2][128], slots_block[512 / 32];
  constexpr int WIDE = F32 ? 2 : 1, UNITS = 2 + 2 * WIDE;  // 16-byte units of a vector: block, grad_x, residual, grad_new
  constexpr bool KEEP = V <= 2;
  start_behind();
  const int me = threadIdx.x, tpr = blockDim.x, nvec = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(rows_smem) + (uint32_t)me * 16u;
  // the unit u of vector i in stage s
  auto at = [&](int s, int u, int i) { return mine + (uint32_t)(((s * UNITS + u) * V + i) * tpr) * 16u; };
  auto wide_at = [&](int s, int u, int i, float (&f)[8]) {
    Wide<ACT, F32> w;
#pragma unroll
    for (int h = 0; h < WIDE; ++h) w.v[h] = lds_u4(at(s, u + h, i));
    w.get(f);
  };
  // The weights of a vector's channels: of the second norm, and of what stands in front of the residual (post and gate together)
  auto load_w = [&](int i, float (&w)[8]) {
    const int v = me + i * tpr;
    unpack8<ACT>(v < nvec ? *reinterpret_cast<const uint4*>(p.weight + v * 8) : make_uint4(0, 0, 0, 0), w);
  };
  auto load_pg = [&](int g, int i, float (&pg)[8]) {
    const int v = me + i * tpr;
#pragma unroll
    for (int k = 0; k < 8; ++k) pg[k] = 1.f;
    float x[8];
    if (p.post && v < nvec) unpack8<ACT>(*reinterpret_cast<const uint4*>(p.post + v * 8), pg);
    if (p.gate && v < nvec) {
      unpack8<ACT>(*reinterpret_cast<const uint4*>(p.gate + g * p.ldg + v * 8), x);
#pragma unroll
      for (int k = 0; k < 8; ++k) pg[k] *= x[k];
    }
  };
  float kept_w[KEEP ? V : 1][8], kept_pg[KEEP ? V : 1][8];
  float gw[V][8], S[V][8];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (KEEP) load_w(i, kept_w[i]);
#pragma unroll
    for (int k = 0; k < 8; ++k) gw[i][k] = 0.f;
  }
  // Three stages and more: a row's reduction takes the next row's sum of block block along, whose copies have landed by then.
  const bool ahead = p.stages >= 3;
  const int part = (int)(blockIdx.x % p.ctas_per_gate), stride = (int)(gridDim.x / p.ctas_per_gate);
  bool first_gate = true;
  for (int g = blockIdx.x / p.ctas_per_gate; g < p.gates; g += stride, first_gate = false) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (KEEP) load_pg(g, i, kept_pg[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) S[i][k] = 0.f;
    }
    const long long t0 = (long long)g * p.tokens_per_gate;
    const int r0 = (int)((long long)p.tokens_per_gate * part / p.ctas_per_gate);
    const int rows = (int)((long long)p.tokens_per_gate * (part + 1) / p.ctas_per_gate) - r0;
    auto fetch = [&](int n) {  // row n of this run, to stage n % stages
      if (n < rows) {
        const long long t = t0 + r0 + n;
        const int s = n % p.stages;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int v = me + i * tpr;
          if (v < nvec) {
            copy16(at(s, 0, i), p.block + t * p.ldb + v * 8);
            copy16(at(s, 1, i), p.grad_x + t * p.lddx + v * 8);
#pragma unroll
            for (int h = 0; h < WIDE; ++h) {
              if (p.residual) copy16(at(s, 2 + h, i), static_cast<const char*>(p.residual) + (t * p.ldr + v * 8) * (F32 ? 4 : 2) + h * 16);
              if (p.grad_new) copy16(at(s, 2 + WIDE + h, i), static_cast<const char*>(p.grad_new) + (t * p.lddn + v * 8) * (F32 ? 4 : 2) + h * 16);
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto block_square = [&](int s) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float b[8];
        unpack8<ACT>(lds_u4(at(s, 0, i)), b);
        if (me + i * tpr < nvec)
#pragma unroll
          for (int k = 0; k < 8; ++k) x += b[k] * b[k];
      }
      return x;
    };
    for (int n = 0; n < p.stages - 1; ++n) fetch(n);
    float s1 = 1.f;
    if (ahead && p.post && rows > 0) {
      copies_wait(p.stages - 2);
      float x[1] = {block_square(0)};
      row_reduce<1, false>(x, slots_block, false);
      s1 = rsqrtf(x[0] * inv_d + p.eps);
    }
    for (int n = 0; n < rows; ++n) {
      const int s = n % p.stages;
      fetch(n + p.stages - 1);
      copies_wait(ahead ? p.stages - 2 : p.stages - 1);
      if (!ahead && p.post) {
        float x[1] = {block_square(s)};
        row_reduce<1, false>(x, slots_block, false);
        s1 = rsqrtf(x[0] * inv_d + p.eps);
      }
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      float kept_r[1][8];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (me + i * tpr < nvec) {
          float b[8], d[8], res[8], dn[8], w[8], pg[8];
          unpack8<ACT>(lds_u4(at(s, 0, i)), b);
          unpack8<ACT>(lds_u4(at(s, 1, i)), d);
          if (p.residual) wide_at(s, 2, i, res);
          if (p.grad_new) wide_at(s, 2 + WIDE, i, dn);
          if constexpr (!KEEP) { load_w(i, w); load_pg(g, i, pg); }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float q = b[k] * s1 * (KEEP ? kept_pg[KEEP ? i : 0][k] : pg[k]), e = d[k] * (KEEP ? kept_w[KEEP ? i : 0][k] : w[k]);
            const float r = q + (p.residual ? p.scale * res[k] : 0.f);
            if constexpr (V == 1) kept_r[0][k] = r;
            sum[0] += r * r;
            sum[1] += e * r;
            sum[2] += q * (p.grad_new ? dn[k] : 0.f);
            sum[3] += q * e;
            sum[4] += q * r;
          }
        }
      }
      if (ahead && p.post && n + 1 < rows) sum[5] = block_square((n + 1) % p.stages);
      sums8(sum, slots[n & 1]);
      const float s2 = rsqrtf(sum[0] * inv_d + p.eps), mean = sum[1] * s2 * inv_d;         // of e xh
      const float mean_q = (sum[2] + s2 * (sum[3] - s2 * mean * sum[4])) * inv_d;          // of dr q
      const long long t = t0 + r0 + n;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        if (v < nvec) {
          float b[8], d[8], res[8], dn[8], w[8], pg[8], out[8];
          unpack8<ACT>(lds_u4(at(s, 0, i)), b);
          unpack8<ACT>(lds_u4(at(s, 1, i)), d);
          if (V > 1 && p.residual) wide_at(s, 2, i, res);
          if (p.grad_new) wide_at(s, 2 + WIDE, i, dn);
          if constexpr (!KEEP) { load_w(i, w); load_pg(g, i, pg); }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float m = KEEP ? kept_pg[KEEP ? i : 0][k] : pg[k], e = d[k] * (KEEP ? kept_w[KEEP ? i : 0][k] : w[k]);
            const float bh = b[k] * s1, q = bh * m;
            const float r = V == 1 ? kept_r[0][k] : q + (p.residual ? p.scale * res[k] : 0.f);
            const float xh = r * s2;
            gw[i][k] += d[k] * xh;
            const float dr = (p.grad_new ? dn[k] : 0.f) + s2 * (e - xh * mean);
            S[i][k] += dr * bh;
            res[k] = p.scale * dr;
            out[k] = p.post ? s1 * (dr * m - bh * mean_q) : dr * m;
          }
          if (p.grad_residual) Wide<ACT, F32>::store(p.grad_residual, t * p.lddr + v * 8, res);
          *reinterpret_cast<uint4*>(p.grad_block + t * p.lddb + v * 8) = pack8<ACT>(out);
        }
      }
      s1 = ahead && p.post ? rsqrtf(sum[5] * inv_d + p.eps) : s1;
    }
    // the gate's sums: its own gradient, and what the rows give post
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
      if (v >= nvec) continue;
      float x[8];
      if (p.grad_gate) {
        float* to = p.ctas_per_gate == 1 ? p.grad_gate + (long long)g * p.D : p.partial + ((long long)2 * p.grid + blockIdx.x) * p.D;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = 1.f;
        if (p.post) unpack8<ACT>(*reinterpret_cast<const uint4*>(p.post + v * 8), x);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] *= S[i][k];
        Wide<ACT, true>::store(to, v * 8, x);
      }
      if (p.post) {
        const long long to = ((long long)p.grid + blockIdx.x) * p.D + v * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = 1.f;
        if (p.gate) unpack8<ACT>(*reinterpret_cast<const uint4*>(p.gate + g * p.ldg + v * 8), x);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = x[k] * S[i][k] + (first_gate ? 0.f : p.partial[to + k]);
        Wide<ACT, true>::store(p.partial, to, x);
      }
    }
    copies_wait(0);  // (what was asked for past the run's end is nothing)
    __syncthreads();  // the slots of this run's last row have been read
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    if (v < nvec) Wide<ACT, true>::store(p.partial, (long long)blockIdx.x * p.D + v * 8, gw[i]);
  }
}

// The sums of the CTAs' shares: 32 columns a CTA, eight runs of CTAs' shares side by side, joined in order.  blockIdx.y: grad_weight,
// grad_post, then one for each gate.
__global__ void __launch_bounds__(256) norm_sums_kernel(const NormBackwardParams p) {
  __shared__ float part[8][33];
  start_behind();
  const int which = (int)blockIdx.y, col = (int)blockIdx.x * 32 + (threadIdx.x & 31), run = threadIdx.x >> 5;
  const float* from = p.partial;
  float* to = p.grad_weight;
  int n = p.grid;
  if (which == 1) {
    if (!p.post) return;
    from += (long long)p.grid * p.D;
    to = p.grad_post;
  } else if (which > 1) {
    const int g = which - 2;
    n = p.ctas_per_gate;
    from += ((long long)2 * p.grid + (long long)g * n) * p.D;
    to = p.grad_gate + (long long)g * p.D;
  }
  float s = 0.f;
  if (col < p.D) {
    const int i0 = n * run / 8, i1 = n * (run + 1) / 8;
#pragma unroll 8
    for (int i = i0; i < i1; ++i) s += from[(long long)i * p.D + col];
  }
  part[run][threadIdx.x & 31] = s;
  __syncthreads();
  if (run == 0 && col < p.D) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x & 31];
    to[col] = s;
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

// Threads of a row and vectors of a thread: a warp for up to 512 channels, else a CTA.
struct RowShape { int warp_rows, threads, vectors, ctas; };
static RowShape row_shape(int T, int D) {
  const int nvec = D / 8;
  RowShape s;
  s.warp_rows = nvec <= 64 ? 1 : 0;
  if (s.warp_rows) {
    s.vectors = nvec <= 32 ? 1 : 2;
    s.threads = 128;
    s.ctas = (T + 3) / 4;
    return s;
  }
  s.vectors = nvec <= 256 ? 1 : nvec <= 2048 ? 2 : 4;
  const int per = (nvec + s.vectors - 1) / s.vectors;
  s.threads = (per + 31) / 32 * 32;
  if (s.threads > 1024) s.threads = 1024;
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
    default: return launch_behind(cast_int_kernel<ACT, 4>, grid, s.threads, 0, stream, p, s.warp_rows);
  }
}
cudaError_t cast_int_launch(const CastIntParams& p, int act, cudaStream_t stream) {
  return act == 0 ? cast_int_act<0>(p, stream) : cast_int_act<1>(p, stream);
}

template <int ACT, bool F32>
static cudaError_t norm_type(const NormParams& p, cudaStream_t stream) {
  const RowShape s = row_shape(p.T, p.D);
  const dim3 grid((unsigned)s.ctas, 1, 1);
  switch (s.vectors) {
    case 1: return launch_behind(norm_kernel<ACT, F32, 1>, grid, s.threads, 0, stream, p, s.warp_rows);
    default: return launch_behind(norm_kernel<ACT, F32, 2>, grid, s.threads, 0, stream, p, s.warp_rows);
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
template <int ACT, bool F32>
static cudaError_t backward_type(const NormBackwardParams& p, cudaStream_t stream) {
  cudaError_t e;
  switch (p.vectors) {
    case 1: e = backward_rows<ACT, F32, 1>(p, stream); break;
    case 2: e = backward_rows<ACT, F32, 2>(p, stream); break;
    default: e = backward_rows<ACT, F32, 4>(p, stream); break;
  }
  if (e != cudaSuccess) return e;
  const int sums = 2 + (p.grad_gate && p.ctas_per_gate > 1 ? p.gates : 0);
  return launch_behind(norm_sums_kernel, dim3((unsigned)((p.D + 31) / 32), (unsigned)sums, 1), 256, 0, stream, p);
}
// The shape of the gradient's launch: threads and vectors of a row, CTAs (one for 512 threads of an SM), and stages for the rows ahead.
void norm_backward_shape(int D, bool residual_f32, int gates, int tokens_per_gate, int sms, int max_smem, NormBackwardParams* p) {
  const int nvec = D / 8;
  p->vectors = nvec <= 512 ? 1 : nvec <= 1024 ? 2 : 4;
  p->threads = ((nvec + p->vectors - 1) / p->vectors + 31) / 32 * 32;
  const int per_sm = 512 / p->threads < 4 ? 512 / p->threads : 4, most = sms * per_sm;
  if (gates >= most) {
    p->ctas_per_gate = 1;
    p->grid = most;
  } else {
    p->ctas_per_gate = most / gates < tokens_per_gate ? most / gates : tokens_per_gate;
    p->grid = gates * p->ctas_per_gate;
  }
  const int stage = p->vectors * p->threads * 16 * (residual_f32 ? 6 : 4), room = (max_smem + 1024) / per_sm - 1024 - 2048;
  p->stages = room / stage > 4 ? 4 : room / stage;
  p->smem = p->stages * stage;
}
cudaError_t norm_backward_launch(const NormBackwardParams& p, int act, bool residual_f32, cudaStream_t stream) {
  if (act == 0) return residual_f32 ? backward_type<0, true>(p, stream) : backward_type<0, false>(p, stream);
  return residual_f32 ? backward_type<1, true>(p, stream) : backward_type<1, false>(p, stream);
}

}  // namespace b200q
