// C ABI of the 8-bit integer products, the per-token int8 cast and the block norms: argument checks, kernel choice, launches.
#include <cmath>

#include "../../include/b200q.h"
#include "int8.cuh"
#include "norm.cuh"

namespace b200q {

static bool misaligned(const void* p, unsigned bytes) { return ((uintptr_t)p & (bytes - 1)) != 0; }
static bool known_act(int act) { return act == B200Q_F16 || act == B200Q_BF16; }

// ---- products -----------------------------------------------------------------------------------------------
// int32 sums are exact up to this K: 128 * 128 * K < 2^31
static const int kInt8MaxK = 131056;
static const int kStreamRows = 256;

static int check_igemm(int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1) return ST_INVALID_ARG;
  if (N % 16 != 0 || K % 16 != 0 || K > kInt8MaxK) return ST_UNSUPPORTED;
  return ST_OK;
}
static int igemm_kblocks(int K) { return (K + 127) / 128; }

static int parts(int n, int of) { return (n - 1) / of + 1; }  // of `of` each that n >= 1 makes (n may be any int)
static long long pair_tiles(int M, int N, bool gated, int cols) { return (long long)parts(M, 256) * parts(N, gated ? cols / 2 : cols); }
// Shares of the columns in the stream kernel, of which `at_once` run at once: as many as that in as few rounds as the tensor core's
// 256 columns allow, but of two units of 8 columns at least.  They differ by a unit at most.  Where an SM
// has one, as few as have the widest width, since each reads A (64 x 12288 x 4096 11.6 us with 140, 12.1 with 148); where it has two,
// all, since what counts is the wider pair of them (64 x 28672 x 4096 gated 21.8 with 256, 21.4 with 296).
static const int kUnit = 8;
static int stream_width(int N, int shares) { return parts(N / kUnit, shares) * kUnit; }  // of the widest
static int stream_shares(int N, bool gated, int at_once, int per) {
  const int units = N / kUnit, most = gated ? 16 : 32;
  const int rounds = (units + most * at_once - 1) / (most * at_once), all = rounds * at_once;
  const int shares = all < units / 2 ? all : units / 2;
  return per == 1 ? parts(N, stream_width(N, shares)) : shares;
}
static int stream_stages(int M, bool gated, int width, int s, int budget) {
  int stages = 12;  // (with 16 64 x 1024 x 8192 takes 7.3 us, not 7.0)
  while (stages > 1 && int8_stream_smem_bytes(M, gated, width, s, stages) > budget) --stages;
  return stages;
}

// What a call takes, in us, by kernel: fitted to calls of 1 .. 8192 rows x 1024 .. 28672 columns x 128 .. 14336 on a B200, which they
// meet within some 15 %.  They decide between kernels, so that only their ratios matter.  (Fitted with B read early.  Without that the
// row kernel takes 0.3 to 1.1 us more and the stream kernel 0.1 to 0.6: over 60 shapes of up to 16 rows the choice between the two is 0.9 %
// from the better one on average, 0.6 % with.)
constexpr double kHbm = 6465.5e3;  // bytes a us

// Reading B at five sixths of the memory's rate up to eight rows of A (with twice as many, whose loads are as many as B's, at three
// fifths), but no less than the latency of each round of a CTA, which goes by its length of K.
static double row_cost(int M, double b_bytes, int rounds, int K) {
  const bool few = M <= 8;
  const double steps = K / 4096.0;
  const double memory = 1.6 + b_bytes / kHbm * (few ? 1.2 : 1.62);
  const double latency = 0.4 + rounds * (few ? 1.4 + 1.4 * steps : 1.9 + 2.4 * steps);
  return memory > latency ? memory : latency;
}

// Rows that start between two 32-byte sectors: their pieces of 128 bytes come in one sector more, of two lines.  (K = 4096 / 4128 / 4112, us:
// 1024 x 18944 50 / 53 / 65, 200 x 4736 12.9 / 14.1 / 19.7.)
static bool split_sectors(int K) { return K % 32 != 0; }

// A piece of 128 bytes of K takes what the slowest of three takes: reading B, bringing both operands' rows to the SM (121 GB/s a SM, or
// half of that), and the tensor core's reading them (about as fast, but whole accumulators' rows of A).  A cluster's exchange goes by the
// sums that it moves: 64 x 4096 x 14336 takes 20.1 us alone, 14.5 in pairs, 15.3 in fours; 128 rows 20.7, 17.1, 19.4.  Two CTAs to an SM
// (`per` 2) share it, but one starts and ends under the other: 8 x 28672 gated 22.5 us with one, 20.6 with two.
static double stream_cost(int M, int N, bool gated, int shares, int s, int at_once, int per, int K, const DeviceInfo& di) {
  const int kblocks = igemm_kblocks(K), both = gated ? 2 : 1, b_rows = both * stream_width(N, shares), ctas = shares * s;
  const int rows = (M + 15) / 16 * 16, accs = (rows + 127) / 128, slots = s * at_once;
  const int rounds = (ctas + slots - 1) / slots;
  const double tensor = per * accs * (128 + b_rows) * (per == 1 ? 0.95e-3 : 1.05e-3);
  const double in = per * (rows + b_rows) * (split_sectors(K) ? 2.1e-3 : 1.05e-3);
  // all of B's rows at the memory's rate, and those of the SM that has most at its own
  const double all = (double)both * N * s / rounds, alone = (double)both * kUnit * ((per * (N / kUnit) + shares - 1) / shares);
  const double most = 0.95 * di.sm_count * alone;
  const double memory = 128.0 / kHbm * (all > most ? all : most) * (per == 1 ? 1.08 : 1.03);
  const double piece = tensor > in ? (tensor > memory ? tensor : memory) : (in > memory ? in : memory);
  return (per == 1 ? 2.8 : 2.6) + rounds * piece * ((kblocks + s - 1) / s) + (s > 1 ? 0.55 + 0.17 * s + 5e-4 * M * b_rows * (s - 1) / s : 0.0) +
         0.004 * per * M;
}

// A piece of a tile of 256 x 256 takes 0.30 us (0.28 at rest, 0.35 under the power limit), of 256 x 128 two thirds: its operands come
// through the same SM.  A tile takes no less than its outputs do, 3.1 and 1.9 us (gated 2.6: half
// of the writers have none of a narrow tile).  Up front, and for the last tile's outputs: 5.6 and 3.9.  And
// B has to be read.
static double pair_cost(long long tiles, bool gated, int cols, int K, double b_bytes, const DeviceInfo& di) {
  const int pairs = di.sm_count / 2;
  const long long rounds = (tiles - 1) / pairs + 1;
  const double piece = split_sectors(K) ? (cols == 256 ? 0.42 : 0.32) : cols == 256 ? 0.30 : 0.195;
  const double products = igemm_kblocks(K) * piece, outputs = cols == 256 ? 3.1 : gated ? 2.6 : 1.9;
  const double start = cols == 256 ? 5.6 : 3.9, all = products + (rounds - 1) * (products > outputs ? products : outputs);
  const double memory = 1.15 * b_bytes / kHbm;
  return start + (all > memory ? all : memory);
}

static void make_igemm_plan(int M, int N, int K, bool gated, b200q_igemm_plan_t* pl) {
  const DeviceInfo di = device_info();
  const int kblocks = igemm_kblocks(K);
  *pl = b200q_igemm_plan_t();
  double best = 1e30;
  // (A last row tile of a few rows costs as much as any, but no more than that: 4097 x 12288 x 4096 takes 137.7 us, 4096 rows 132.5, and
  // 4096 rows with the last one in a kernel of its own beside them 142.2.)
  for (int cols = 256; cols >= 128; cols -= 128) {
    const long long tiles = pair_tiles(M, N, gated, cols);
    const double cost = pair_cost(tiles, gated, cols, K, (double)(gated ? 2 : 1) * N * K, di);
    if (cost >= best) continue;
    best = cost;
    *pl = {1, 256, cols, 2, cols == 256 ? 6 : 8, 2 * (int)(tiles < di.sm_count / 2 ? tiles : di.sm_count / 2)};
  }
  if (M > kStreamRows) return;
  const int* clusters = int8_stream_clusters(di);
  for (int s = 1, i = 0; s <= 8 && 4 * (s - 1) <= kblocks; s *= 2, ++i)
    for (int per = s == 1 && kblocks >= 10 ? 2 : 1; per >= 1; --per) {
      const int at_once = per * clusters[i], shares = stream_shares(N, gated, at_once, per), width = stream_width(N, shares);
      if (per == 2 && (M > 128 ? 2 : 1) * (((gated ? 2 : 1) * width + 15) / 16 * 16) > 256) continue;  // (both CTAs' tensor memory)
      const double cost = stream_cost(M, N, gated, shares, s, at_once, per, K, di);
      if (cost >= best) continue;
      // Half an SM's shared memory for one of two CTAs, or where that is depth enough for the length of K: a CTA of the stream's next
      // launch has room next to it then.  (us, K 1024 / 2048 / 4096, half an SM's stages / ten of a whole one's: 24 x 9472, 8 stages, 4.4
      // 7.6 10.7 / 5.0 7.7 10.1; 100 x 9472, 4 stages, 5.4 8.6 12.8 / 5.6 8.0 10.5; 24 x 4736, 12 stages, 3.8 5.2 8.4 / 4.2 5.8 9.0.)
      // A cluster has whole SMs in any case.
      int stages = stream_stages(M, gated, width, s, s > 1 ? di.max_smem : 113 * 1024);
      if (s == 1 && per == 1 && stages < 12 && (stages < 3 || 3 * kblocks > 8 * stages)) stages = stream_stages(M, gated, width, s, di.max_smem);
      if (stages < (per == 1 ? 2 : 3)) continue;
      best = cost;
      *pl = {2, (M + 15) / 16 * 16, width, s, stages, shares * s};
    }
  if (M <= 16) {
    const int items = N / (gated ? 8 : 16);
    const double cost = row_cost(M, (double)(gated ? 2 : 1) * N * K, (items + 2 * di.sm_count - 1) / (2 * di.sm_count), K);
    if (cost < best) *pl = {3, M, gated ? 8 : 16, 1, 1, items < 2 * di.sm_count ? items : 2 * di.sm_count};
  }
}

// A thread's latest plans: a model's layers come again with each token, and to weigh the kernels takes a tenth of a small call (0.3 us).
static void plan_igemm(int M, int N, int K, bool gated, b200q_igemm_plan_t* pl) {
  struct Known { int M = 0, N, K, gated, dev; b200q_igemm_plan_t plan; };
  static thread_local Known known[16];
  int dev = -1;
  (void)cudaGetDevice(&dev);
  Known& k = known[((unsigned)N / 16 * 7 + (unsigned)K / 16 * 3 + (unsigned)M + (gated ? 5 : 0)) % 16];
  if (k.M != M || k.N != N || k.K != K || k.gated != (int)gated || k.dev != dev) {
    make_igemm_plan(M, N, K, gated, &k.plan);
    k.M = M; k.N = N; k.K = K; k.gated = gated; k.dev = dev;
  }
  *pl = k.plan;
}

// 2-D map of 8-bit rows, a box of 128 bytes x `rows`
static int encode_rows(EncodeTiledFn enc, CUtensorMap* map, const void* base, int K, long long rows, long long ld, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {128u, (cuuint32_t)box_rows}, steps[2] = {1u, 1u};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ST_OK : cuda_failed((int)r);
}

static int run_igemm(const void* a, int lda, const void* b, int ldb, const float* a_sf, const float* b_sf, const void* bias, void* c,
                     int ldc, int M, int N, int K, int act, bool gated, int use_clamp, float clamp, int early_b, void* workspace, size_t ws_bytes,
                     cudaStream_t stream, const b200q_igemm_plan_t& pl) {
  if (!known_act(act)) return ST_UNSUPPORTED;
  int st = check_igemm(M, N, K);
  if (st != ST_OK) return st;
  if (!a || !b || !a_sf || !b_sf || !c) return ST_INVALID_ARG;
  if (lda < K || ldb < K || ldc < N || lda % 16 != 0 || ldb % 16 != 0 || ldc % 8 != 0) return ST_INVALID_ARG;
  if (misaligned(a, 16) || misaligned(b, 16) || misaligned(c, 16) || misaligned(a_sf, 4) || misaligned(b_sf, 16) || misaligned(bias, 16))
    return ST_INVALID_ARG;
  if (use_clamp && std::isnan(clamp)) return ST_INVALID_ARG;
  if (!workspace || ws_bytes < WS_HEADER_BYTES || misaligned(workspace, 256)) return ST_WORKSPACE;
  const EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return cuda_failed((int)cudaErrorNotSupported);
  Int8Params p = {};
  p.a = static_cast<const signed char*>(a); p.b = static_cast<const signed char*>(b);
  p.lda = lda; p.ldb = ldb;
  p.early = early_b ? 1 : 0;
  p.a_sf = a_sf; p.b_sf = b_sf;
  p.bias = static_cast<const unsigned short*>(bias);
  p.c = static_cast<unsigned short*>(c);
  p.status = static_cast<int*>(workspace);
  p.M = M; p.N = N; p.K = K; p.ldc = ldc;
  p.kblocks = igemm_kblocks(K);
  p.act = act;
  p.use_clamp = use_clamp ? 1 : 0;
  p.clamp = clamp;
  const long long b_rows = gated ? 2ll * N : N;
  CUtensorMap ta, tb, tb_less, tc;
  cudaError_t e;
  if (pl.kernel == 3) {
    e = int8_row_launch(p, gated, pl.ctas, stream);
  } else if (pl.kernel == 1) {
    const int pc = pl.width;
    st = encode_rows(enc, &ta, a, K, M, lda, 128);
    if (st == ST_OK) st = encode_rows(enc, &tb, b, K, b_rows, ldb, pc / 2);
    if (st != ST_OK) return st;
    const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    const cuuint64_t strides[1] = {(cuuint64_t)ldc * 2};
    const cuuint32_t box[2] = {64u, 32u}, steps[2] = {1u, 1u};
    const CUresult r = enc(&tc, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, c, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return cuda_failed((int)r);
    p.m_tiles = parts(M, 256);
    p.n_tiles = parts(N, gated ? pc / 2 : pc);
    // (more than any memory holds; a CTA's next tile stays an int)
    if ((long long)p.m_tiles * p.n_tiles > 0x7fffff00ll) return ST_UNSUPPORTED;
    p.tiles = p.m_tiles * p.n_tiles;
    // rows of A that stay in the L2 cache while the columns of B stream past them: about 32 MB
    const long long fit = (32ll << 20) / (256ll * K);
    p.m_group = (int)(fit < 1 ? 1 : fit > p.m_tiles ? p.m_tiles : fit);
    e = int8_pair_launch(p, gated, pc, ta, tb, tc, pl.ctas, stream);
  } else {
    st = encode_rows(enc, &ta, a, K, M, lda, pl.rows);
    if (st == ST_OK) st = encode_rows(enc, &tb, b, K, b_rows, ldb, pl.width);
    p.tiles = pl.ctas / pl.cluster;
    p.rows = pl.rows; p.width = pl.width; p.cluster = pl.cluster; p.stages = pl.stages;
    p.wide = p.tiles - (int)((long long)pl.width / kUnit * p.tiles - N / kUnit);
    if (p.wide == p.tiles) tb_less = tb;
    else if (st == ST_OK) st = encode_rows(enc, &tb_less, b, K, b_rows, ldb, pl.width - kUnit);
    if (st != ST_OK) return st;
    // A cluster's CTAs have an SM each to themselves.  Next to one another, two clusters (of one launch or of two streams) could each
    // hold the tensor memory that the other's second CTA waits for.
    p.smem = pl.cluster > 1 ? device_info().max_smem : int8_stream_smem_bytes(M, gated, pl.width, 1, pl.stages);
    e = int8_stream_launch(p, gated, ta, tb, tb_less, stream);
  }
  return e == cudaSuccess ? ST_OK : cuda_failed((int)e);
}

// Whether a (possibly edited) plan can be run: what its kernel needs of its fields.
static bool igemm_plan_ok(int M, int N, int K, bool gated, b200q_igemm_plan_t* pl) {
  const DeviceInfo di = device_info();
  if (pl->kernel == 1) {
    if (pl->width != 128 && pl->width != 256) return false;
    if (pl->ctas < 2 || pl->ctas % 2 != 0 || pl->ctas > di.sm_count) return false;
    return int8_pair_smem_bytes(pl->width) <= di.max_smem;
  }
  if (pl->kernel == 3) return M <= 16 && pl->ctas >= 1 && pl->ctas <= 8 * di.sm_count;
  if (pl->kernel != 2 || M > kStreamRows) return false;
  pl->rows = (M + 15) / 16 * 16;
  if (pl->cluster < 1 || pl->cluster > 8 || pl->cluster > igemm_kblocks(K)) return false;
  if (pl->width < kUnit || pl->width > (gated ? 128 : 256) || pl->width % kUnit != 0) return false;
  // (shares as the CTAs say, where these are of that width; else as few as there can be)
  int shares = pl->ctas > 0 && pl->ctas % pl->cluster == 0 ? pl->ctas / pl->cluster : 0;
  if (shares < 1 || shares > N / kUnit || stream_width(N, shares) != pl->width) shares = parts(N, pl->width);
  pl->width = stream_width(N, shares);
  pl->ctas = shares * pl->cluster;
  return pl->stages >= 1 && pl->stages <= 16 &&
         int8_stream_smem_bytes(M, gated, pl->width, pl->cluster, pl->stages) <= di.max_smem;
}

// ---- row-wise kernels -------------------------------------------------------------------------------------
static const int kNormMaxD = 16384;

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_igemm_plan(int M, int N, int K, int gated, b200q_igemm_plan_t* plan) {
  if (!plan) return ST_INVALID_ARG;
  const int st = check_igemm(M, N, K);
  if (st == ST_OK) plan_igemm(M, N, K, gated != 0, plan);
  return st;
}

int b200q_igemm(const void* a, int lda, const void* b, int ldb, const float* a_sf, const float* b_sf, const void* bias, void* c, int ldc,
                int M, int N, int K, int act_dtype, int early_b, void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_igemm(M, N, K);
  if (st != ST_OK) return st;
  b200q_igemm_plan_t pl;
  plan_igemm(M, N, K, false, &pl);
  return run_igemm(a, lda, b, ldb, a_sf, b_sf, bias, c, ldc, M, N, K, act_dtype, false, 0, 0.f, early_b, workspace, workspace_bytes,
                   static_cast<cudaStream_t>(stream), pl);
}

int b200q_igemm_swiglu(const void* a, int lda, const void* b, int ldb, const float* a_sf, const float* b_sf, void* c, int ldc, int M,
                       int N, int K, int act_dtype, int use_clamp, float clamp_value, int early_b, void* workspace,
                       size_t workspace_bytes, void* stream) {
  int st = check_igemm(M, N, K);
  if (st != ST_OK) return st;
  if (N > 0x7fffffff / 2) return ST_UNSUPPORTED;
  b200q_igemm_plan_t pl;
  plan_igemm(M, N, K, true, &pl);
  return run_igemm(a, lda, b, ldb, a_sf, b_sf, nullptr, c, ldc, M, N, K, act_dtype, true, use_clamp, clamp_value, early_b,
                   workspace, workspace_bytes, static_cast<cudaStream_t>(stream), pl);
}

int b200q_igemm_planned(const void* a, int lda, const void* b, int ldb, const float* a_sf, const float* b_sf, const void* bias, void* c,
                        int ldc, int M, int N, int K, int act_dtype, int gated, int use_clamp, float clamp_value,
                        int early_b, void* workspace, size_t workspace_bytes, void* stream, const b200q_igemm_plan_t* plan) {
  int st = check_igemm(M, N, K);
  if (st != ST_OK) return st;
  if (!plan || (gated && (bias || N > 0x7fffffff / 2))) return ST_INVALID_ARG;
  b200q_igemm_plan_t pl = *plan;
  if (!igemm_plan_ok(M, N, K, gated != 0, &pl)) return ST_UNSUPPORTED;
  return run_igemm(a, lda, b, ldb, a_sf, b_sf, bias, c, ldc, M, N, K, act_dtype, gated != 0, use_clamp, clamp_value, early_b,
                   workspace, workspace_bytes, static_cast<cudaStream_t>(stream), pl);
}

int b200q_per_token_cast_int(const void* x, int ldx, void* out, int ldo, float* out_sf, int tokens, int hidden, int act_dtype,
                             void* stream) {
  if (!known_act(act_dtype)) return ST_UNSUPPORTED;
  if (!x || !out || !out_sf || tokens < 1 || hidden < 1) return ST_INVALID_ARG;
  if (hidden % 8 != 0) return ST_UNSUPPORTED;
  if (ldx < hidden || ldo < hidden || ldx % 8 != 0 || ldo % 8 != 0) return ST_INVALID_ARG;
  if (misaligned(x, 16) || misaligned(out, 8) || misaligned(out_sf, 4)) return ST_INVALID_ARG;
  CastIntParams p;
  p.x = static_cast<const unsigned short*>(x);
  p.out = static_cast<signed char*>(out);
  p.out_sf = out_sf;
  p.T = tokens; p.D = hidden; p.ldx = ldx; p.ldo = ldo;
  const cudaError_t e = cast_int_launch(p, act_dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? ST_OK : cuda_failed((int)e);
}

static int check_norm(const b200q_block_norm_t* a) {
  if (!a) return ST_INVALID_ARG;
  if (!known_act(a->act_dtype)) return ST_UNSUPPORTED;
  if (!a->block || !a->weight || a->tokens < 1 || a->hidden < 1 || a->gates < 0) return ST_INVALID_ARG;
  if ((a->gates == 0) != (a->gate == nullptr)) return ST_INVALID_ARG;
  if (a->hidden % 8 != 0 || a->hidden > kNormMaxD) return ST_UNSUPPORTED;
  if (a->gates > 0 && a->tokens % a->gates != 0) return ST_INVALID_ARG;
  if (a->ldb < a->hidden || a->ldb % 8 != 0) return ST_INVALID_ARG;
  if (a->residual && (a->ldr < a->hidden || a->ldr % 8 != 0)) return ST_INVALID_ARG;
  if (a->gates > 1 && (a->ldg < a->hidden || a->ldg % 8 != 0)) return ST_INVALID_ARG;
  if (misaligned(a->block, 16) || misaligned(a->residual, 16) || misaligned(a->weight, 16) || misaligned(a->post_weight, 16) ||
      misaligned(a->gate, 16))
    return ST_INVALID_ARG;
  return ST_OK;
}

int b200q_block_norm(const b200q_block_norm_t* a, void* x, long long ldx, void* x_int, float* x_sf, void* new_residual, long long ldn,
                     void* stream) {
  const int st = check_norm(a);
  if (st != ST_OK) return st;
  if ((x == nullptr) == (x_int == nullptr) || (x_int && !x_sf) || !new_residual) return ST_INVALID_ARG;
  if (ldx < a->hidden || ldx % 8 != 0 || ldn < a->hidden || ldn % 8 != 0) return ST_INVALID_ARG;
  if (misaligned(x, 16) || misaligned(x_int, 8) || misaligned(x_sf, 4) || misaligned(new_residual, 16)) return ST_INVALID_ARG;
  NormParams p = {};
  p.block = static_cast<const unsigned short*>(a->block);
  p.weight = static_cast<const unsigned short*>(a->weight);
  p.post = static_cast<const unsigned short*>(a->post_weight);
  p.gate = static_cast<const unsigned short*>(a->gate);
  p.residual = a->residual;
  p.x = static_cast<unsigned short*>(x);
  p.x_int = static_cast<signed char*>(x_int);
  p.x_sf = x_sf;
  p.new_residual = new_residual;
  p.T = a->tokens; p.D = a->hidden;
  p.tokens_per_gate = a->gates > 0 ? a->tokens / a->gates : a->tokens;
  p.ldb = a->ldb; p.ldr = a->ldr; p.ldg = a->ldg; p.ldx = ldx; p.ldn = ldn;
  p.scale = a->residual_scale; p.eps = a->eps;
  p.sms = device_info().sm_count;
  const cudaError_t e = norm_launch(p, a->act_dtype, a->residual_f32 != 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? ST_OK : cuda_failed((int)e);
}

size_t b200q_block_norm_scratch_bytes(int tokens, int hidden, int gates) {
  if (tokens < 1 || hidden < 8 || hidden % 8 != 0 || hidden > kNormMaxD || gates < 0 || (gates > 0 && tokens % gates != 0)) return 0;
  NormBackwardParams p;
  const DeviceInfo di = device_info();
  norm_backward_shape(hidden, false, gates > 0 ? gates : 1, tokens / (gates > 0 ? gates : 1), di.sm_count, di.max_smem, &p);
  return (size_t)2 * p.grid * hidden * sizeof(float);
}

int b200q_block_norm_backward(const b200q_block_norm_t* a, const void* grad_x, long long lddx, const void* grad_new, long long lddn,
                              void* grad_block, long long lddb, void* grad_residual, long long lddr, float* grad_weight,
                              float* grad_post, float* grad_gate, void* scratch, size_t scratch_bytes, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const int st = check_norm(a);
  if (st != ST_OK) return st;
  if (!grad_x || !grad_block || !grad_weight || (grad_post == nullptr) != (a->post_weight == nullptr) ||
      (grad_gate == nullptr) != (a->gate == nullptr) || (grad_residual && !a->residual))
    return ST_INVALID_ARG;
  if (lddx < a->hidden || lddx % 8 != 0 || lddb < a->hidden || lddb % 8 != 0) return ST_INVALID_ARG;
  if ((grad_new && (lddn < a->hidden || lddn % 8 != 0)) || (grad_residual && (lddr < a->hidden || lddr % 8 != 0))) return ST_INVALID_ARG;
  if (misaligned(grad_x, 16) || misaligned(grad_new, 16) || misaligned(grad_block, 16) || misaligned(grad_residual, 16) ||
      misaligned(grad_weight, 16) || misaligned(grad_post, 16) || misaligned(grad_gate, 16))
    return ST_INVALID_ARG;
  if (!scratch || misaligned(scratch, 16) || scratch_bytes < b200q_block_norm_scratch_bytes(a->tokens, a->hidden, a->gates))
    return ST_WORKSPACE;
  if (!workspace || workspace_bytes < WS_HEADER_BYTES || misaligned(workspace, 256)) return ST_WORKSPACE;
  NormBackwardParams p = {};
  p.status = static_cast<int*>(workspace);
  p.block = static_cast<const unsigned short*>(a->block);
  p.weight = static_cast<const unsigned short*>(a->weight);
  p.post = static_cast<const unsigned short*>(a->post_weight);
  p.gate = static_cast<const unsigned short*>(a->gate);
  p.grad_x = static_cast<const unsigned short*>(grad_x);
  p.residual = a->residual; p.grad_new = grad_new;
  p.grad_block = static_cast<unsigned short*>(grad_block);
  p.grad_residual = grad_residual;
  p.grad_weight = grad_weight; p.grad_post = grad_post; p.grad_gate = grad_gate;
  p.partial = static_cast<float*>(scratch);
  p.T = a->tokens; p.D = a->hidden;
  p.gates = a->gates > 0 ? a->gates : 1;
  p.tokens_per_gate = a->tokens / p.gates;
  const DeviceInfo di = device_info();
  norm_backward_shape(p.D, a->residual_f32 != 0, p.gates, p.tokens_per_gate, di.sm_count, di.max_smem, &p);
  p.ldb = a->ldb; p.ldr = a->ldr; p.ldg = a->ldg;
  p.lddx = lddx; p.lddn = lddn; p.lddb = lddb; p.lddr = lddr;
  p.scale = a->residual_scale; p.eps = a->eps;
  const cudaError_t e = norm_backward_launch(p, a->act_dtype, a->residual_f32 != 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? ST_OK : cuda_failed((int)e);
}

}  // extern "C"
