// LayerNorm for training its own weights: forward, and backward with dgamma / dbeta.
//   y = (x - mean) rstd gamma + beta,   xh = (x - mean) rstd,   g = dy gamma
//   dx = rstd (g - mean_C(g) - xh mean_C(g xh)) [+ dres],   dgamma = sum_rows dy xh,   dbeta = sum_rows dy
// bf16 or fp32 rows of any width up to 8192 and any row stride; every sum and statistic in fp32.  With a checkpoint (aql_act8.cuh) the
// forward pass also writes the 8-bit codes of x and the backward pass reads them in x's place (mean and rstd stay those of x itself).
//
// A row is held in the registers of TPR threads (16, 64, 256 or 512, by width), 8 columns per thread and slot: x is read once forward, x and
// dy once backward, so the kernels are bound by HBM.  The column sums dgamma / dbeta stay in the registers of a thread over all rows of
// its group, are joined over the workgroup in LDS and written as one fp32 row pair per workgroup; a second launch adds those
// rows in a fixed order (no atomics: the same bits every time).
#include "aql_act8.cuh"

using namespace act8;

namespace {

constexpr int MAXC = 8192;
constexpr int BWD_T = 512;
constexpr int fwd_threads(int tpr) { return tpr > 256 ? tpr : 256; }
constexpr int BWD_BLOCKS = 512;   // two workgroups per CU, 16 wavefronts

template <int TPR>
__device__ __forceinline__ float group_sum(float v, float* red) {
  if constexpr (TPR == 16) {   // the four row rotations of wave_sum stay inside 16 lanes
    v += aql_dpp_row<0x128>(v);
    v += aql_dpp_row<0x124>(v);
    v += aql_dpp_row<0x122>(v);
    v += aql_dpp_row<0x121>(v);
    return v;
  } else if constexpr (TPR == 64) {
    return wave_sum(v);
  } else {
    v = wave_sum(v);
    const int wave = threadIdx.x >> 6, base = (threadIdx.x / TPR) * (TPR / 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = red[base];
#pragma unroll
    for (int k = 1; k < TPR / 64; ++k) v += red[base + k];
    return v;
  }
}

__device__ __forceinline__ void load_param(const void* p, int bf, int col, int n, float* o) {
  if (bf) {
    Raw8<bf16_t> r;
    load_raw((const bf16_t*)p + col, n, r);
    widen(r, o);
  } else {
    Raw8<float> r;
    load_raw((const float*)p + col, n, r);
    widen(r, o);
  }
}

template <class T, int TPR, int NT>
__global__ __launch_bounds__(fwd_threads(TPR)) void fwd_kernel(const T* __restrict__ x, long M, int C, long ldx, const void* __restrict__ gamma,
                                                    const void* __restrict__ beta, int pbf, float eps, T* __restrict__ y, long ldy,
                                                    float2* __restrict__ stats, uint8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  constexpr int FWD_T = fwd_threads(TPR);
  __shared__ float red[FWD_T / 64];
  const int lane = threadIdx.x % TPR;
  const long row = (long)blockIdx.x * (FWD_T / TPR) + threadIdx.x / TPR;
  if (TPR < 256 && row >= M) return;   // (256 and more: one row per workgroup, the grid is M)
  float v[NT][8];
  float s = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int col = (lane + t * TPR) * 8;
    Raw8<T> r;
    load_raw(x + row * ldx + (col < C ? col : 0), C - col, r);
    widen(r, v[t]);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) s += v[t][j];
  const float mean = group_sum<TPR>(s, red) / C;
  float q = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = C - (lane + t * TPR) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = v[t][j] - mean;
      q += j < n ? d * d : 0.f;
    }
  }
  const float rstd = rsqrtf(group_sum<TPR>(q, red) / C + eps);
  if (lane == 0) stats[row] = make_float2(mean, rstd);
  const int nchunk = ((C + 31) / 32) * 4;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = lane + t * TPR, col = c * 8, n = C - col;
    if (codes != nullptr) {
      const uint32_t b = exp_byte(quad_umax(amax_bits8(v[t])));   // (every lane of the quad is here: nothing above branches per chunk)
      if (c < nchunk) {
        const float inv = inv_step(b);
        *reinterpret_cast<uint2*>(codes + (row * nchunk + c) * 8) =
            make_uint2(codes4(v[t][0], v[t][1], v[t][2], v[t][3], inv), codes4(v[t][4], v[t][5], v[t][6], v[t][7], inv));
        if ((c & 3) == 0) exps[row * (nchunk >> 2) + (c >> 2)] = (uint8_t)b;
      }
    }
    if (n > 0) {
      float ga[8], be[8], o[8];
      load_param(gamma, pbf, col, n, ga);
      if (beta != nullptr) load_param(beta, pbf, col, n, be);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf((v[t][j] - mean) * rstd, ga[j], beta != nullptr ? be[j] : 0.f);
      store8(y + row * ldy + col, n, o);
    }
  }
}

template <class T, int TPR, int NT, bool CK>
__global__ __launch_bounds__(BWD_T) void bwd_kernel(const T* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                    const T* __restrict__ dy, const T* __restrict__ dres, long M, int C, long ldx, long lddy,
                                                    long lddres, const void* __restrict__ gamma, int pbf, const float2* __restrict__ stats,
                                                    T* __restrict__ dx, long lddx, float* __restrict__ part) {
  constexpr int GROUPS = BWD_T / TPR;
  __shared__ float red[BWD_T / 64];
  __shared__ float acc_lds[2][TPR * NT * 8];
  const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const int nchunk = ((C + 31) / 32) * 4;
  float ga[NT][8], ag[NT][8], ab[NT][8];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int col = (lane + t * TPR) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) ga[t][j] = ag[t][j] = ab[t][j] = 0.f;
    if (col < C) load_param(gamma, pbf, col, C - col, ga[t]);
  }
  // 256 and more threads reduce over workgroup barriers: all groups of the workgroup make the same number of rounds (a dead row is a row of zeros)
  const long rounds = (M + (long)gridDim.x * GROUPS - 1) / ((long)gridDim.x * GROUPS);
  for (long it = 0; it < rounds; ++it) {
    const long row = (it * gridDim.x + blockIdx.x) * GROUPS + grp;
    const bool live = row < M;
    if (TPR < 256 && !live) break;
    const float2 st = live ? stats[row] : make_float2(0.f, 0.f);
    float xh[NT][8], g[NT][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int c = lane + t * TPR, col = c * 8, n = live ? C - col : 0;
      if constexpr (CK) {
        uint2 q = make_uint2(0u, 0u);
        float sp = 0.f;
        if (n > 0) {
          q = *reinterpret_cast<const uint2*>(codes + (row * nchunk + c) * 8);
          sp = step(exps[row * (nchunk >> 2) + (c >> 2)]);
        }
        values4(q.x, sp, xh[t]);
        values4(q.y, sp, xh[t] + 4);
      } else {
        Raw8<T> r;
        load_raw(n > 0 ? x + row * ldx + col : x, n, r);
        widen(r, xh[t]);
      }
      Raw8<T> r;
      load_raw(n > 0 ? dy + row * lddy + col : dy, n, r);
      widen(r, g[t]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[t][j] = (xh[t][j] - st.x) * st.y;
        ag[t][j] = fmaf(g[t][j], xh[t][j], ag[t][j]);
        ab[t][j] += g[t][j];
        g[t][j] *= ga[t][j];
        s1 += g[t][j];
        s2 = fmaf(g[t][j], xh[t][j], s2);
      }
    s1 = group_sum<TPR>(s1, red) / C;
    s2 = group_sum<TPR>(s2, red) / C;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = (lane + t * TPR) * 8, n = live ? C - col : 0;
      if (n > 0) {
        float o[8], rs[8];
        if (dres != nullptr) {
          Raw8<T> r;
          load_raw(dres + row * lddres + col, n, r);
          widen(r, rs);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[j] = st.y * (g[t][j] - s1 - xh[t][j] * s2);
          if (dres != nullptr) o[j] += rs[j];
        }
        store8(dx + row * lddx + col, n, o);
      }
    }
  }
  // the groups add to the workgroup's sums one after the other: a fixed order
  for (int k = 0; k < GROUPS; ++k) {
    if (grp == k) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = (lane + t * TPR) * 8 + j;
          acc_lds[0][i] = k ? acc_lds[0][i] + ag[t][j] : ag[t][j];
          acc_lds[1][i] = k ? acc_lds[1][i] + ab[t][j] : ab[t][j];
        }
    }
    __syncthreads();
  }
  float* out = part + (long)blockIdx.x * 2 * C;
  for (int i = threadIdx.x; i < C; i += BWD_T) {
    out[i] = acc_lds[0][i];
    out[C + i] = acc_lds[1][i];
  }
}

// out[j] = sum over the nblk partial rows, j < n = 2C: 64 columns x 16 row groups per workgroup
__global__ __launch_bounds__(1024) void reduce_kernel(const float* __restrict__ part, int nblk, int n, int C, float* __restrict__ dgamma,
                                                      float* __restrict__ dbeta) {
  __shared__ float acc[16][64];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), grp = threadIdx.x >> 6;
  float s = 0.f;
  if (col < n)
#pragma unroll 8
    for (int b = grp; b < nblk; b += 16) s += part[(long)b * n + col];
  acc[grp][threadIdx.x & 63] = s;
  __syncthreads();
  if (grp == 0 && col < n) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += acc[k][threadIdx.x];
    float* o = col < C ? dgamma : dbeta;
    if (o != nullptr) o[col < C ? col : col - C] = s;
  }
}

int bwd_blocks(long M, int C) {
  const int groups = C <= 256 ? BWD_T / 16 : C <= 2048 ? BWD_T / 64 : C <= 4096 ? BWD_T / 256 : 1;
  const long b = (M + groups - 1) / groups;
  return (int)(b < BWD_BLOCKS ? b : BWD_BLOCKS);
}

struct Args {
  const void *x, *dy, *dres, *gamma, *beta;
  uint8_t *codes, *exps;
  void* out;
  long M, ldx, lddy, lddres, ldo;
  int C, pbf;
  float eps;
  float2* stats;
  float* part;
};

template <class T, int TPR, int NT>
void launch(int mode, const Args& a, hipStream_t st) {
  if (mode == 0)
    hipLaunchKernelGGL((fwd_kernel<T, TPR, NT>), dim3((unsigned)((a.M + fwd_threads(TPR) / TPR - 1) / (fwd_threads(TPR) / TPR))), dim3(fwd_threads(TPR)), 0, st, (const T*)a.x, a.M,
                       a.C, a.ldx, a.gamma, a.beta, a.pbf, a.eps, (T*)a.out, a.ldo, a.stats, a.codes, a.exps);
  else if (a.codes)
    hipLaunchKernelGGL((bwd_kernel<T, TPR, NT, true>), dim3(bwd_blocks(a.M, a.C)), dim3(BWD_T), 0, st, (const T*)a.x, a.codes, a.exps, (const T*)a.dy,
                       (const T*)a.dres, a.M, a.C, a.ldx, a.lddy, a.lddres, a.gamma, a.pbf, a.stats, (T*)a.out, a.ldo, a.part);
  else
    hipLaunchKernelGGL((bwd_kernel<T, TPR, NT, false>), dim3(bwd_blocks(a.M, a.C)), dim3(BWD_T), 0, st, (const T*)a.x, a.codes, a.exps, (const T*)a.dy,
                       (const T*)a.dres, a.M, a.C, a.ldx, a.lddy, a.lddres, a.gamma, a.pbf, a.stats, (T*)a.out, a.ldo, a.part);
}

template <class T>
void dispatch(int mode, const Args& a, hipStream_t st) {
  const int chunks = (a.C + 7) / 8;
  if (chunks <= 16) launch<T, 16, 1>(mode, a, st);
  else if (chunks <= 32) launch<T, 16, 2>(mode, a, st);
  else if (chunks <= 64) launch<T, 64, 1>(mode, a, st);
  else if (chunks <= 128) launch<T, 64, 2>(mode, a, st);
  else if (chunks <= 192) launch<T, 64, 3>(mode, a, st);
  else if (chunks <= 256) launch<T, 64, 4>(mode, a, st);
  else if (chunks <= 512) launch<T, 256, 2>(mode, a, st);
  else launch<T, 512, 2>(mode, a, st);
}

}  // namespace

// fp32 elements of the workspace of aql_layernorm_train_bwd
extern "C" int aql_layernorm_train_scratch_floats(long M, int C) { return M <= 0 || C <= 0 || C > MAXC ? 0 : bwd_blocks(M, C) * 2 * C; }

extern "C" int aql_layernorm_train_fwd(const void* x, int dtype, long M, int C, long ldx, const void* gamma, const void* beta, int param_dtype,
                                       float eps, void* y, long ldy, float* stats, uint8_t* codes, uint8_t* exps, hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && M < (1L << 31) && C > 0 && C <= MAXC && ldx >= C && ldy >= C, "aql_layernorm_train_fwd: bad shape M=%ld C=%d (at most %d columns)", M, C, MAXC);
  AQL_CHECK_ARG((dtype == 0 || dtype == 1) && (param_dtype == 0 || param_dtype == 1) && !codes == !exps, "aql_layernorm_train_fwd: bad types");
  if (M == 0) return AQL_OK;
  AQL_CHECK_ARG(x && gamma && y && stats, "aql_layernorm_train_fwd: null operand");
  Args a{};
  a.x = x, a.gamma = gamma, a.beta = beta, a.codes = codes, a.exps = exps, a.out = y, a.M = M, a.ldx = ldx, a.ldo = ldy, a.C = C;
  a.pbf = param_dtype == 0, a.eps = eps, a.stats = (float2*)stats;
  if (dtype == 0) dispatch<bf16_t>(0, a, stream);
  else dispatch<float>(0, a, stream);
  AQL_CHECK_LAUNCH("aql_layernorm_train_fwd");
  return AQL_OK;
}

extern "C" int aql_layernorm_train_bwd(const void* x, const uint8_t* codes, const uint8_t* exps, const void* dy, const void* dres, int dtype, long M,
                                       int C, long ldx, long lddy, long lddres, const void* gamma, int param_dtype, const float* stats, void* dx,
                                       long lddx, float* dgamma, float* dbeta, float* scratch, long scratch_floats, hipStream_t stream) {
  AQL_CHECK_ARG(M > 0 && M < (1L << 31) && C > 0 && C <= MAXC && lddy >= C && lddx >= C && (!dres || lddres >= C) && (!x || ldx >= C),
                "aql_layernorm_train_bwd: bad shape M=%ld C=%d (at most %d columns)", M, C, MAXC);
  AQL_CHECK_ARG((dtype == 0 || dtype == 1) && (param_dtype == 0 || param_dtype == 1) && !codes == !exps && !x != !codes,
                "aql_layernorm_train_bwd: bad types, or not exactly one of x and its codes");
  AQL_CHECK_ARG(dy && gamma && stats && dx && scratch, "aql_layernorm_train_bwd: null operand");
  AQL_CHECK_ARG(scratch_floats >= aql_layernorm_train_scratch_floats(M, C), "aql_layernorm_train_bwd: workspace of %ld floats, %d needed",
                scratch_floats, aql_layernorm_train_scratch_floats(M, C));
  Args a{};
  a.x = x ? x : dy;   // (codes: never read)
  a.codes = const_cast<uint8_t*>(codes), a.exps = const_cast<uint8_t*>(exps), a.dy = dy, a.dres = dres, a.gamma = gamma, a.out = dx, a.M = M;
  a.C = C, a.ldx = ldx, a.lddy = lddy, a.lddres = lddres, a.ldo = lddx, a.pbf = param_dtype == 0;
  a.stats = (float2*)const_cast<float*>(stats), a.part = scratch;
  if (dtype == 0) dispatch<bf16_t>(1, a, stream);
  else dispatch<float>(1, a, stream);
  AQL_CHECK_LAUNCH("aql_layernorm_train_bwd");
  if (dgamma || dbeta) {
    hipLaunchKernelGGL(reduce_kernel, dim3((2 * C + 63) / 64), dim3(1024), 0, stream, scratch, bwd_blocks(M, C), 2 * C, C, dgamma, dbeta);
    AQL_CHECK_LAUNCH("aql_layernorm_train_bwd (weight gradients)");
  }
  return AQL_OK;
}
