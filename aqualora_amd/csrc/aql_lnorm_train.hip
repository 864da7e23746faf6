// LayerNorm for training its own weights: forward, and backward with dgamma / dbeta.
//   y = (x - mean) rstd gamma + beta,   xh = (x - mean) rstd,   g = dy gamma
//   dx = rstd (g - mean_C(g) - xh mean_C(g xh)) [+ dres],   dgamma = sum_rows dy xh,   dbeta = sum_rows dy
// bf16 or fp32 rows of any width up to 8192 and any row stride; every sum and statistic in fp32.  With a checkpoint (aql_act8.cuh) the
// forward pass also writes the 8-bit codes of x and the backward pass reads them in x's place (mean and rstd stay those of x itself).
//
// A row is held in the registers of TPR threads (16, 64, 256 or 512, by width), 8 columns per thread and slot: x is read once forward, x and
// dy once backward, so the kernels are bound by HBM.  A group of threads walks over its rows with the next row's loads in flight under the
// arithmetic of this one (16384 x 1280 bf16 with codes: 19.7 us forward and 23.0 backward, 5.3 and 4.6 TB/s; one row after the other 31 and 35; 32768 x
// 320: 10.8 and 16.4).  The column sums dgamma
// / dbeta stay in the registers of a thread over all rows of its group, are joined over the workgroup in LDS and written as one fp32 row pair
// per workgroup; a second launch adds those rows in a fixed order (no atomics: the same bits every time).
#include "aql_act8.cuh"

using namespace act8;

namespace {

constexpr int MAXC = 8192;
constexpr int threads(int tpr) { return tpr > 256 ? tpr : 256; }
// workgroups that fit on the 256 CUs together, by registers
constexpr int fwd_most(int nt) { return nt == 1 ? 2048 : nt == 2 ? 1280 : 1024; }
constexpr int BWD_BLOCKS = 768;

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

// a parameter row as fp32 in LDS, zeros past its end (and all zeros for an absent one)
template <int THREADS, int W>
__device__ __forceinline__ void stage_param(const void* p, int bf, int C, float* out) {
  for (int c = threadIdx.x; c < W / 8; c += THREADS) {
    float g[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (p != nullptr && c * 8 < C) load_param(p, bf, c * 8, C - c * 8, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) out[c * 8 + j] = g[j];
  }
}

// A chunk of a row.  TAIL: C is no multiple of 8, the last chunk is read element by element.  Otherwise a chunk is whole or dead, all are read without a
// branch (dead ones from the row's first columns) and `mask` makes zeros of the dead ones: the compiler can count the loads in flight.
template <bool TAIL, class T>
__device__ __forceinline__ void fetch(const T* p, int n, Raw8<T>& r) {
  load_raw(p, TAIL ? n : 8, r);
}
template <bool TAIL, class T>
__device__ __forceinline__ void mask(Raw8<T>& r, int n) {
  if constexpr (!TAIL) {
#pragma unroll
    for (uint32_t& w : r.w) w = n > 0 ? w : 0u;
  }
}

template <class T, int TPR, int NT, bool TAIL>
__global__ __launch_bounds__(threads(TPR), TPR > 256 ? 2 : 4) void fwd_kernel(const T* __restrict__ x, long M, int C, long ldx, const void* __restrict__ gamma,
                                                                              const void* __restrict__ beta, int pbf, float eps, T* __restrict__ y, long ldy,
                                                                              float2* __restrict__ stats, uint8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  constexpr int THREADS = threads(TPR), GROUPS = THREADS / TPR, W = TPR * NT * 8;
  __shared__ float red[THREADS / 64];
  __shared__ __attribute__((aligned(16))) float gl[W], bl[W];   // gamma and beta: from memory they would be four times the loads of a bf16 row
  const int lane = threadIdx.x % TPR;
  const int nchunk = ((C + 31) / 32) * 4;
  stage_param<THREADS, W>(gamma, pbf, C, gl);
  stage_param<THREADS, W>(beta, pbf, C, bl);
  __syncthreads();
  const long stride = (long)gridDim.x * GROUPS;
  long row = (long)blockIdx.x * GROUPS + threadIdx.x / TPR;   // (256 threads and more: one group per workgroup, so barriers are met together)
  Raw8<T> raw[NT];
  auto load = [&](long r) {
    const T* p = x + min(r, M - 1) * ldx;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = (lane + t * TPR) * 8;
      fetch<TAIL>(p + (col < C ? col : 0), C - col, raw[t]);
    }
  };
  load(row);
  for (; row < M; row += stride) {
    float v[NT][8];
    uint32_t am[NT];
    float s = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      mask<TAIL>(raw[t], C - (lane + t * TPR) * 8);
      widen(raw[t], v[t]);
      am[t] = amax_bits8(raw[t]);
    }
    load(row + stride);
    if (codes != nullptr) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int c = lane + t * TPR;
        const uint32_t b = exp_byte(quad_umax(am[t]));   // (every lane of the quad is here)
        if (c < nchunk) {
          *reinterpret_cast<uint2*>(codes + (row * nchunk + c) * 8) = codes8(v[t], b);
          if ((c & 3) == 0) exps[row * (nchunk >> 2) + (c >> 2)] = (uint8_t)b;
        }
      }
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
      if (n >= 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[t][j] -= mean;
          q = fmaf(v[t][j], v[t][j], q);
        }
      } else if (n > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[t][j] -= mean;
          q += j < n ? v[t][j] * v[t][j] : 0.f;
        }
      }
    }
    const float rstd = rsqrtf(group_sum<TPR>(q, red) / C + eps);
    if (lane == 0) stats[row] = make_float2(mean, rstd);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = (lane + t * TPR) * 8, n = C - col;
      if (n > 0) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = fmaf(v[t][j] * rstd, gl[col + j], bl[col + j]);
        store8(y + row * ldy + col, n, o);
      }
    }
  }
}

template <class T, int TPR, int NT, bool CK, bool RES, bool TAIL>
__global__ __launch_bounds__(threads(TPR), TPR > 256 || (NT == 3 && (RES || sizeof(T) == 4)) ? 2 : 3) void bwd_kernel(const T* __restrict__ x, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                                              const T* __restrict__ dy, const T* __restrict__ dres, long M, int C, long ldx, long lddy,
                                                                              long lddres, const void* __restrict__ gamma, int pbf, const float2* __restrict__ stats,
                                                                              T* __restrict__ dx, long lddx, float* __restrict__ part) {
  constexpr int THREADS = threads(TPR), GROUPS = THREADS / TPR, W = TPR * NT * 8;
  __shared__ float red[THREADS / 64];
  __shared__ __attribute__((aligned(16))) float gl[W], acc_lds[2][W];   // gamma; the workgroup's column sums
  const int lane = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const int nchunk = ((C + 31) / 32) * 4;
  stage_param<THREADS, W>(gamma, pbf, C, gl);
  __syncthreads();
  float ag[NT][8], ab[NT][8];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) ag[t][j] = ab[t][j] = 0.f;
  const long stride = (long)gridDim.x * GROUPS;
  long row = (long)blockIdx.x * GROUPS + grp;
  Raw8<T> rx[NT], rd[NT], rr[NT];
  uint2 rc[NT];
  uint32_t re[NT];
  float2 st;
  auto load = [&](long r) {   // past the end: the last row again, never used
    r = min(r, M - 1);
    st = stats[r];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int c = lane + t * TPR, col = c * 8, at = col < C ? col : 0;
      if constexpr (CK) {
        const int ca = col < C ? c : 0;
        rc[t] = *reinterpret_cast<const uint2*>(codes + (r * nchunk + ca) * 8);
        re[t] = exps[r * (nchunk >> 2) + (ca >> 2)];
      } else {
        fetch<TAIL>(x + r * ldx + at, C - col, rx[t]);
      }
      fetch<TAIL>(dy + r * lddy + at, C - col, rd[t]);
      if constexpr (RES) fetch<TAIL>(dres + r * lddres + at, C - col, rr[t]);
    }
  };
  load(row);
  for (; row < M; row += stride) {
    float xh[NT][8], g[NT][8];
    Raw8<T> res[NT];
    const float mean = st.x, rstd = st.y;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (CK) {
        const float sp = step(re[t]);
        values4(rc[t].x, sp, xh[t]);
        values4(rc[t].y, sp, xh[t] + 4);
      } else {
        widen(rx[t], xh[t]);
      }
      mask<TAIL>(rd[t], C - (lane + t * TPR) * 8);
      widen(rd[t], g[t]);   // (columns past C: dy reads as zero, so they add nothing to any sum ...
      if constexpr (RES) res[t] = rr[t];
    }
    load(row + stride);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if ((lane + t * TPR) * 8 >= C) continue;   // ... and chunks past C are left out: x may hold a NaN there)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[t][j] = (xh[t][j] - mean) * rstd;
        ag[t][j] = fmaf(g[t][j], xh[t][j], ag[t][j]);
        ab[t][j] += g[t][j];
        g[t][j] *= gl[(lane + t * TPR) * 8 + j];
        s1 += g[t][j];
        s2 = fmaf(g[t][j], xh[t][j], s2);
      }
    }
    s1 = group_sum<TPR>(s1, red) / C;
    s2 = group_sum<TPR>(s2, red) / C;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = (lane + t * TPR) * 8, n = C - col;
      if (n > 0) {
        float o[8], rs[8];
        if constexpr (RES) widen(res[t], rs);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[j] = rstd * (g[t][j] - s1 - xh[t][j] * s2);
          if constexpr (RES) o[j] += rs[j];
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
  for (int i = threadIdx.x; i < C; i += THREADS) {
    out[i] = acc_lds[0][i];
    out[C + i] = acc_lds[1][i];
  }
}

// out[j] = sum over the nblk partial rows, j < n = 2C: 32 columns x 32 row groups per workgroup
__global__ __launch_bounds__(1024) void reduce_kernel(const float* __restrict__ part, int nblk, int n, int C, float* __restrict__ dgamma,
                                                      float* __restrict__ dbeta) {
  __shared__ float acc[32][32];
  const int c = threadIdx.x & 31, col = blockIdx.x * 32 + c, grp = threadIdx.x >> 5;
  float s = 0.f;
  if (col < n)
#pragma unroll 8
    for (int b = grp; b < nblk; b += 32) s += part[(long)b * n + col];
  acc[grp][c] = s;
  __syncthreads();
  if (grp == 0 && col < n) {
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += acc[k][c];
    float* o = col < C ? dgamma : dbeta;
    if (o != nullptr) o[col < C ? col : col - C] = s;
  }
}

int tpr_of(int C) { return C <= 256 ? 16 : C <= 1536 ? 64 : C <= 4096 ? 256 : 512; }   // of the backward pass: see dispatch
// at least eight rows to a workgroup: its two rows of sums are then small change next to the rows it reads
int bwd_blocks(long M, int C) {
  const int groups = threads(tpr_of(C)) / tpr_of(C), rows = groups < 8 ? 8 : groups;
  const long b = (M + rows - 1) / rows, most = tpr_of(C) > 256 ? 512 : BWD_BLOCKS;
  return (int)(b < most ? b : most);
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

template <class T, int TPR, int NT, bool TAIL>
void launch_tail(int mode, const Args& a, hipStream_t st) {
  constexpr int GROUPS = threads(TPR) / TPR;
  if (mode == 0) {
    const long b = (a.M + GROUPS - 1) / GROUPS;
    hipLaunchKernelGGL((fwd_kernel<T, TPR, NT, TAIL>), dim3((unsigned)(b < fwd_most(NT) ? b : fwd_most(NT))), dim3(threads(TPR)), 0, st, (const T*)a.x, a.M, a.C, a.ldx,
                       a.gamma, a.beta, a.pbf, a.eps, (T*)a.out, a.ldo, a.stats, a.codes, a.exps);
    return;
  }
  const dim3 grid(bwd_blocks(a.M, a.C));
#define AQL_LNB(CK, RES)                                                                                                                                  \
  hipLaunchKernelGGL((bwd_kernel<T, TPR, NT, CK, RES, TAIL>), grid, dim3(threads(TPR)), 0, st, (const T*)a.x, a.codes, a.exps, (const T*)a.dy, (const T*)a.dres, \
                     a.M, a.C, a.ldx, a.lddy, a.lddres, a.gamma, a.pbf, a.stats, (T*)a.out, a.ldo, a.part)
  if (a.codes && a.dres) AQL_LNB(true, true);
  else if (a.codes) AQL_LNB(true, false);
  else if (a.dres) AQL_LNB(false, true);
  else AQL_LNB(false, false);
#undef AQL_LNB
}

template <class T, int TPR, int NT>
void launch(int mode, const Args& a, hipStream_t st) {
  if (a.C % 8) launch_tail<T, TPR, NT, true>(mode, a, st);
  else launch_tail<T, TPR, NT, false>(mode, a, st);
}

template <class T>
void dispatch(int mode, const Args& a, hipStream_t st) {
  const int chunks = (a.C + 7) / 8;
  if (chunks <= 16) launch<T, 16, 1>(mode, a, st);
  else if (chunks <= 32) launch<T, 16, 2>(mode, a, st);
  // (forward only: four rows to a wavefront put four times the bytes in flight, 32768 x 320 10.7 against 16.6 us; backward the sixteen groups of a workgroup
  // take longer to join than that saves, 19.7 against 15.8 us)
  else if (chunks <= 48 && mode == 0) launch<T, 16, 3>(mode, a, st);
  else if (chunks <= 64) launch<T, 64, 1>(mode, a, st);
  else if (chunks <= 128) launch<T, 64, 2>(mode, a, st);
  else if (chunks <= 192) launch<T, 64, 3>(mode, a, st);
  else if (chunks <= 256) launch<T, 256, 1>(mode, a, st);
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
    hipLaunchKernelGGL(reduce_kernel, dim3((2 * C + 31) / 32), dim3(1024), 0, stream, scratch, bwd_blocks(M, C), 2 * C, C, dgamma, dbeta);
    AQL_CHECK_LAUNCH("aql_layernorm_train_bwd (weight gradients)");
  }
  return AQL_OK;
}
