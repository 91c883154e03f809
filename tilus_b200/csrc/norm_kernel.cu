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
//   bh = block s1, n = bh post;  r = scale residual + gate n;  xh = r s2;  e = grad_x weight
//   dr = grad_new + s2 (e - xh mean(e xh));   grad_residual = scale dr;   dn = gate dr
//   grad_block = s1 (f - bh mean(f bh)) with f = dn post   (dn without a norm after the block)
//   grad_weight = sum grad_x xh,  grad_post = sum dn bh,  grad_gate = sum dr n   over the rows (of the gate)
// A CTA takes a run of rows of one gate and keeps its share of the three sums in registers; a second kernel adds the CTAs' shares
// in a fixed order, so that a call gives the same bits each time.
template <int ACT, bool F32, int V>
__global__ void __launch_bounds__(512) norm_backward_kernel(const NormBackwardParams p) {
  __shared__ float slots[3][64];
  const int me = threadIdx.x, tpr = blockDim.x, nvec = p.D / 8;
  const float inv_d = 1.0f / (float)p.D;
  uint4 weight[V], post[V], gate[V];
  float gw[V][8], gp[V][8], gg[V][8];
  const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    weight[i] = v < nvec ? *reinterpret_cast<const uint4*>(p.weight + v * 8) : none;
    post[i] = p.post && v < nvec ? *reinterpret_cast<const uint4*>(p.post + v * 8) : none;
#pragma unroll
    for (int k = 0; k < 8; ++k) gw[i][k] = gp[i][k] = 0.f;
  }
  const int part = (int)(blockIdx.x % p.ctas_per_gate), stride = (int)(gridDim.x / p.ctas_per_gate);
  for (int g = blockIdx.x / p.ctas_per_gate; g < p.gates; g += stride) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = me + i * tpr;
      gate[i] = p.gate && v < nvec ? *reinterpret_cast<const uint4*>(p.gate + g * p.ldg + v * 8) : none;
#pragma unroll
      for (int k = 0; k < 8; ++k) gg[i][k] = 0.f;
    }
    const long long t0 = (long long)g * p.tokens_per_gate;
    const int r0 = (int)((long long)p.tokens_per_gate * part / p.ctas_per_gate);
    const int r1 = (int)((long long)p.tokens_per_gate * (part + 1) / p.ctas_per_gate);
    for (long long t = t0 + r0; t < t0 + r1; ++t) {
      uint4 block[V], dx[V];
      Wide<ACT, F32> res[V], dn[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        block[i] = dx[i] = none;
        res[i].zero();
        dn[i].zero();
        if (v < nvec) {
          block[i] = *reinterpret_cast<const uint4*>(p.block + t * p.ldb + v * 8);
          dx[i] = *reinterpret_cast<const uint4*>(p.grad_x + t * p.lddx + v * 8);
          if (p.residual) res[i].load(p.residual, t * p.ldr + v * 8);
          if (p.grad_new) dn[i].load(p.grad_new, t * p.lddn + v * 8);
        }
      }
      float s1 = 1.f;
      if (p.post) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float b[8];
          unpack8<ACT>(block[i], b);
#pragma unroll
          for (int k = 0; k < 8; ++k) s[0] += b[k] * b[k];
        }
        row_reduce<1, false>(s, slots[0], false);
        s1 = rsqrtf(s[0] * inv_d + p.eps);
      }
      float r[V][8], s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float b[8], w[8], q[8];
        unpack8<ACT>(block[i], b);
        if (p.post) {
          unpack8<ACT>(post[i], w);
#pragma unroll
          for (int k = 0; k < 8; ++k) b[k] *= s1 * w[k];
        }
        if (p.gate) {
          unpack8<ACT>(gate[i], w);
#pragma unroll
          for (int k = 0; k < 8; ++k) b[k] *= w[k];
        }
        res[i].get(q);
        unpack8<ACT>(weight[i], w);
        float d[8];
        unpack8<ACT>(dx[i], d);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          r[i][k] = b[k] + p.scale * q[k];
          s[0] += r[i][k] * r[i][k];
          s[1] += d[k] * w[k] * r[i][k];
        }
      }
      row_reduce<2, false>(s, slots[1], false);
      const float s2 = rsqrtf(s[0] * inv_d + p.eps), mean = s[1] * s2 * inv_d;
      float sf[1] = {0.f};
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        float b[8], w[8], q[8], d[8], wp[8];
        unpack8<ACT>(block[i], b);
        unpack8<ACT>(weight[i], w);
        unpack8<ACT>(dx[i], d);
        dn[i].get(q);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float xh = r[i][k] * s2;
          gw[i][k] += d[k] * xh;
          q[k] += s2 * (d[k] * w[k] - xh * mean);  // dr
          w[k] = p.scale * q[k];
        }
        if (p.grad_residual && v < nvec) Wide<ACT, F32>::store(p.grad_residual, t * p.lddr + v * 8, w);
        if (p.post) {
          unpack8<ACT>(post[i], wp);
#pragma unroll
          for (int k = 0; k < 8; ++k) b[k] *= s1;  // bh
        }
        if (p.gate) {
          unpack8<ACT>(gate[i], w);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            gg[i][k] += q[k] * (p.post ? b[k] * wp[k] : b[k]);
            q[k] *= w[k];  // dn
          }
        }
        if (p.post) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            gp[i][k] += q[k] * b[k];
            q[k] *= wp[k];  // f
            sf[0] += q[k] * b[k];
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) r[i][k] = q[k];
      }
      if (p.post) {
        row_reduce<1, false>(sf, slots[2], false);
        const float m = sf[0] * inv_d;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float b[8];
          unpack8<ACT>(block[i], b);
#pragma unroll
          for (int k = 0; k < 8; ++k) r[i][k] = s1 * (r[i][k] - b[k] * s1 * m);
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        if (v < nvec) *reinterpret_cast<uint4*>(p.grad_block + t * p.lddb + v * 8) = pack8<ACT>(r[i]);
      }
      if (!p.post) __syncthreads();  // (with one reduction a row its slots are in use until here)
    }
    if (p.grad_gate) {
      float* to = p.ctas_per_gate == 1 ? p.grad_gate + (long long)g * p.D : p.partial + ((long long)2 * p.grid + blockIdx.x) * p.D;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = me + i * tpr;
        if (v < nvec) Wide<ACT, true>::store(to, v * 8, gg[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = me + i * tpr;
    if (v < nvec) {
      Wide<ACT, true>::store(p.partial, (long long)blockIdx.x * p.D + v * 8, gw[i]);
      if (p.post) Wide<ACT, true>::store(p.partial, ((long long)p.grid + blockIdx.x) * p.D + v * 8, gp[i]);
    }
  }
}

// The sums of the CTAs' shares: 32 columns a CTA, eight runs of CTAs' shares side by side, joined in order.  blockIdx.y: grad_weight,
// grad_post, then one for each gate.
__global__ void __launch_bounds__(256) norm_sums_kernel(const NormBackwardParams p) {
  __shared__ float part[8][33];
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
#pragma unroll 4
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
static cudaError_t launch_behind(Kernel kern, dim3 grid, int threads, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
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
    case 1: return launch_behind(cast_int_kernel<ACT, 1>, grid, s.threads, stream, p, s.warp_rows);
    case 2: return launch_behind(cast_int_kernel<ACT, 2>, grid, s.threads, stream, p, s.warp_rows);
    default: return launch_behind(cast_int_kernel<ACT, 4>, grid, s.threads, stream, p, s.warp_rows);
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
    case 1: return launch_behind(norm_kernel<ACT, F32, 1>, grid, s.threads, stream, p, s.warp_rows);
    default: return launch_behind(norm_kernel<ACT, F32, 2>, grid, s.threads, stream, p, s.warp_rows);
  }
}
cudaError_t norm_launch(const NormParams& p, int act, bool residual_f32, cudaStream_t stream) {
  if (act == 0) return residual_f32 ? norm_type<0, true>(p, stream) : norm_type<0, false>(p, stream);
  return residual_f32 ? norm_type<1, true>(p, stream) : norm_type<1, false>(p, stream);
}

template <int ACT, bool F32>
static cudaError_t backward_type(const NormBackwardParams& p, cudaStream_t stream) {
  const int nvec = p.D / 8, vectors = nvec <= 512 ? 1 : nvec <= 1024 ? 2 : 4;
  const int threads = ((nvec + vectors - 1) / vectors + 31) / 32 * 32;
  switch (vectors) {
    case 1: norm_backward_kernel<ACT, F32, 1><<<p.grid, threads, 0, stream>>>(p); break;
    case 2: norm_backward_kernel<ACT, F32, 2><<<p.grid, threads, 0, stream>>>(p); break;
    default: norm_backward_kernel<ACT, F32, 4><<<p.grid, threads, 0, stream>>>(p); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int sums = 2 + (p.grad_gate && p.ctas_per_gate > 1 ? p.gates : 0);
  norm_sums_kernel<<<dim3((unsigned)((p.D + 31) / 32), (unsigned)sums, 1), 256, 0, stream>>>(p);
  return cudaGetLastError();
}
cudaError_t norm_backward_launch(const NormBackwardParams& p, int act, bool residual_f32, cudaStream_t stream) {
  if (act == 0) return residual_f32 ? backward_type<0, true>(p, stream) : backward_type<0, false>(p, stream);
  return residual_f32 ? backward_type<1, true>(p, stream) : backward_type<1, false>(p, stream);
}

}  // namespace b200q
