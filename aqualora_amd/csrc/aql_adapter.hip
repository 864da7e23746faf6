// Low-rank adapters of many requests at once beside a shared projection.
//
// The rows of X belong to requests, the requests to adapters (or to none):  with g the adapter of row m
//     T[m] = s_g A_g x_m          (aql_adapter_linear, first launch; aql_adapter_down alone, also from 8-bit codes of X)
//     Y[m] = W x_m + b + B_g T[m] + residual_m        (second launch: one fp32 accumulator, one rounding)
// The backward-data pass is the same entry with exchanged operands (X = dY, W = W^T, A = B^T, B = A^T: T becomes dT, Y becomes dX), and
//     P_g = sum over the rows of g of  U[m] V[m]^T     (aql_adapter_wgrad: dA from (dT, X), dB from (T, dY))
// are the weight gradients.
//
// Rows are described by segments: rows [start[s] unit, start[s + 1] unit) have adapter id[s], -1 for none.  A tile of rows finds its segments by
// binary search, so tiles stay dense whatever the requests' lengths; where several segments meet in a tile, the low-rank term runs once
// per segment with the other segments' T rows taken as zeros (a select: what they hold cannot reach the sum).
//
// T is kept in fp32: the gradients dA and dB are fp32 sums of its products and would lose half their digits to a bf16 T.  Their matrix products
// split T into three bf16 parts (24 bits); the second launch of the linear rounds T to bf16 once, where it multiplies B.
#include "aql_act8.cuh"

namespace {

constexpr int BK = 64;
constexpr uint32_t OOB = 0x80000000u;

struct Segs {
  const int* start;   // [n + 1], in units
  const int* id;      // [n]
  int n, unit;
};

// the segment that holds `row` (0 <= row < rows of the plan); uniform arguments, scalar loads
__device__ __forceinline__ int seg_of(const Segs& s, long row) {
  int lo = 0, hi = s.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((long)s.start[mid] * s.unit <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ bf16x8_t zero8() { return bf16x8_t{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ bf16x8_t load8(const bf16_t* p) { return *reinterpret_cast<const bf16x8_t*>(p); }
__device__ __forceinline__ bf16x8_t pack8(const float* v) {
  union { uint32_t w[4]; bf16x8_t f; } u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  return u.f;
}
// eight fp32 T values as an operand fragment (rounded to bf16: the one rounding of T in the linear), zeros where `on` is false
__device__ __forceinline__ bf16x8_t t_frag(const float* p, bool on) {
  if (!on) return zero8();
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  return pack8(v);
}
__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// ---------------------------------------------------------------------------------------------------------------------- T = s A x
// One workgroup: 16 rows x 16 RT adapter rows of ONE segment (blockIdx.y counts the segments of the row tile); its four wavefronts split the
// contraction and join in LDS.  Fragments come straight from memory: lane (i = lane & 15, q = lane >> 4) holds row i, columns k + 8 q ..
// k + 8 q + 7 of either operand, and gets T[m = lane & 15][r = 4 q + e] back.
template <int RT, bool CODES>
__global__ __launch_bounds__(256) void down_kernel(const bf16_t* __restrict__ X, long ldx, const uint8_t* __restrict__ codes,
                                                   const uint8_t* __restrict__ exps, long M, int K, const bf16_t* __restrict__ A,
                                                   const int* __restrict__ ranks, const float* __restrict__ scales, int R, Segs sg,
                                                   float* __restrict__ T) {
  __shared__ float red[3][RT][64][4];
  const long m0 = (long)blockIdx.x * 16;
  const int s = seg_of(sg, m0) + blockIdx.y;
  if (s >= sg.n) return;
  const long lo = max(m0, (long)sg.start[s] * sg.unit), hi = min(m0 + 16, (long)sg.start[s + 1] * sg.unit);
  const int g = sg.id[s];
  if (lo >= hi || g < 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int r0 = blockIdx.z * 16 * RT;
  const int ksteps = (K + 31) / 32, kb = ksteps * wave / 4, ke = ksteps * (wave + 1) / 4;
  const long m = min(m0 + i, M - 1);
  const bf16_t* Ag = A + (long)g * R * K;
  f32x4_t acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int ks = kb; ks < ke; ++ks) {
    const int k = ks * 32 + q * 8;
    const bool in = k < K;
    bf16x8_t xf = zero8();
    if constexpr (CODES) {
      if (in) {
        const uint2 c = *reinterpret_cast<const uint2*>(codes + m * (long)(ksteps * 32) + k);
        const float st = act8::step(exps[m * (long)ksteps + ks]);
        float v[8];
        act8::values4(c.x, st, v);
        act8::values4(c.y, st, v + 4);
        xf = pack8(v);
      }
    } else {
      if (in) xf = load8(X + m * ldx + k);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = r0 + t * 16 + i;
      const bf16x8_t af = in && r < R ? load8(Ag + (long)r * K + k) : zero8();
      acc[t] = mfma(af, xf, acc[t]);
    }
  }
  if (wave) {
#pragma unroll
    for (int t = 0; t < RT; ++t) *reinterpret_cast<f32x4_t*>(red[wave - 1][t][lane]) = acc[t];
  }
  __syncthreads();
  if (wave) return;
  const float sc = scales[g];
  const int rank = ranks[g];
  const long mr = m0 + i;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + t * 16 + q * 4;
    float4 o;
    float* ov = &o.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = ((acc[t][e] + red[0][t][lane][e]) + red[1][t][lane][e]) + red[2][t][lane][e];
      ov[e] = r + e < rank ? sc * v : 0.f;   // columns past the adapter's rank are 0 whatever x holds
    }
    if (mr >= lo && mr < hi && r < R) *reinterpret_cast<float4*>(T + mr * R + r) = o;
  }
}

struct LinArgs {
  const bf16_t *X, *W, *bias, *res, *B;
  bf16_t* Y;
  const float* T;
  long ldx, ldw, ldr, ldy, M;
  int N, K, R;
  Segs sg;   // n = 0: no low-rank term
};

// ------------------------------------------------------------------------------------------- few rows: 16 x 16 NF tiles, split contraction
// Eight wavefronts split the contraction of one tile (and the tile's (segment, rank step) pairs) and join in LDS: with few rows the launch is
// bound by the latency of the weight loads, so the loads of a tile are spread over as many wavefronts as it can feed.
template <int NF>
__global__ __launch_bounds__(512) void skinny_kernel(const LinArgs a) {
  __shared__ float red[8][NF][64][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const long m0 = (long)blockIdx.y * 16;
  const int n0 = blockIdx.x * 16 * NF;
  const int ksteps = (a.K + 31) / 32, kb = ksteps * wave / 8, ke = ksteps * (wave + 1) / 8;
  const long m = min(m0 + i, a.M - 1);
  f32x4_t acc[NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int ks = kb; ks < ke; ++ks) {
    const int k = ks * 32 + q * 8;
    const bool in = k < a.K;
    const bf16x8_t xf = in ? load8(a.X + m * a.ldx + k) : zero8();
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const int n = n0 + j * 16 + i;
      const bf16x8_t wf = in && n < a.N ? load8(a.W + (long)n * a.ldw + k) : zero8();
      acc[j] = mfma(wf, xf, acc[j]);
    }
  }
  if (a.sg.n) {
    const int s0 = seg_of(a.sg, m0), rsteps = (a.R + 31) / 32;
    int turn = 0;
    for (int s = s0; s < a.sg.n && (long)a.sg.start[s] * a.sg.unit < m0 + 16; ++s) {
      const int g = a.sg.id[s];
      if (g < 0) continue;
      const bool mine = m0 + i >= (long)a.sg.start[s] * a.sg.unit && m0 + i < (long)a.sg.start[s + 1] * a.sg.unit;
      const bf16_t* Bg = a.B + (long)g * a.N * a.R;
      for (int rs = 0; rs < rsteps; ++rs, ++turn) {
        if ((turn & 7) != wave) continue;
        const int r = rs * 32 + q * 8;
        const bool in = r < a.R;
        const bf16x8_t tf = t_frag(a.T + m * a.R + r, in && mine);
#pragma unroll
        for (int j = 0; j < NF; ++j) {
          const int n = n0 + j * 16 + i;
          const bf16x8_t bf = in && n < a.N ? load8(Bg + (long)n * a.R + r) : zero8();
          acc[j] = mfma(bf, tf, acc[j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NF; ++j) *reinterpret_cast<f32x4_t*>(red[wave][j][lane]) = acc[j];
  __syncthreads();
  for (int id = threadIdx.x; id < NF * 64; id += 512) {
    const int j = id >> 6, l = id & 63;
    const long mr = m0 + (l & 15);
    const int n = n0 + j * 16 + (l >> 4) * 4;
    if (mr >= a.M || n >= a.N) continue;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v[e] += red[w][j][l][e];
    }
    if (a.bias) {
      const uint2 b = *reinterpret_cast<const uint2*>(a.bias + n);
      v[0] += bf16lo(b.x), v[1] += bf16hi(b.x), v[2] += bf16lo(b.y), v[3] += bf16hi(b.y);
    }
    if (a.res) {
      const uint2 b = *reinterpret_cast<const uint2*>(a.res + mr * a.ldr + n);
      v[0] += bf16lo(b.x), v[1] += bf16hi(b.x), v[2] += bf16lo(b.y), v[3] += bf16hi(b.y);
    }
    *reinterpret_cast<uint2*>(a.Y + mr * a.ldy + n) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  }
}

// ------------------------------------------------------------------------------------------------------------- many rows: LDS tiles
__device__ __forceinline__ int lds_off(int row, int chunk) { return row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4); }   // conflict-free fragment reads

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, voff, soff, 0, 0);
}

// rows x 64 columns of one operand, global -> LDS; lane (row = tid >> 3, slot = tid & 7) fetches source chunk slot ^ ((row >> 1) & 7)
template <int ROWS>
struct Stage {
  static constexpr int NL = ROWS / 32;
  __amdgpu_buffer_rsrc_t rs;
  uint32_t voff[NL], soff;
  int krem, kc;
  __device__ __forceinline__ void init(const bf16_t* base, long ld, int live, int K, int tid) {   // base: first row of the tile
    rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(base), 0, 0x40000000, 0x00020000);
    kc = ((tid & 7) ^ ((tid >> 4) & 7)) * 8;
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int r = (tid >> 3) + 32 * l;
      voff[l] = r < live ? (uint32_t)r * (uint32_t)(ld * 2) + kc * 2 : OOB;
    }
    soff = 0;
    krem = K;
  }
  __device__ __forceinline__ void fetch(char* dst, int wave) {
    const bool bad = kc >= krem;
#pragma unroll
    for (int l = 0; l < NL; ++l) dma16(rs, dst + (32 * l + 8 * wave) * 128, bad ? OOB : voff[l], soff);
    soff += BK * 2;
    krem -= BK;
  }
};

// 256 threads, 2 x 2 wavefronts, BM x BN outputs; NSTG LDS stages with NSTG - 1 tiles of the contraction in flight.  The weight-side
// fragment is MFMA operand A, so a lane ends with four consecutive columns of one row.  The low-rank term runs on fragments loaded straight
// from memory, under the first tiles' DMA.
template <int BM, int BN, int NSTG>
__global__ __launch_bounds__(256) void tile_kernel(const LinArgs a) {
  constexpr int WM = BM / 2, WN = BN / 2, FM = WM / 16, FN = WN / 16;
  constexpr int STAGE = (BM + BN) * 128, PITCH = (BN + 4) * 4;
  constexpr int LDS = NSTG * STAGE > BM * PITCH ? NSTG * STAGE : BM * PITCH;
  constexpr int NLD = BM / 32 + BN / 32;
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i16 = lane & 15, q = lane >> 4;
  const int tiles_n = (a.N + BN - 1) / BN;
  const long m0 = (long)(blockIdx.x / tiles_n) * BM;
  const int n0 = (blockIdx.x % tiles_n) * BN;
  const int wm0 = (wave >> 1) * WM, wn0 = (wave & 1) * WN;
  Stage<BM> sx;
  Stage<BN> sw;
  sx.init(a.X + m0 * a.ldx, a.ldx, (int)min((long)BM, a.M - m0), a.K, tid);
  sw.init(a.W + (long)n0 * a.ldw, a.ldw, min(BN, a.N - n0), a.K, tid);
  f32x4_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto issue = [&](int st) {
    sx.fetch(lds + st * STAGE, wave);
    sw.fetch(lds + st * STAGE + BM * 128, wave);
  };
#pragma unroll
  for (int u = 0; u < NSTG - 1; ++u) issue(u);

  if (a.sg.n) {
    const long w0 = m0 + wm0;   // this wavefront's rows
    const int rsteps = (a.R + 31) / 32;
    if (w0 < a.M)
      for (int s = seg_of(a.sg, w0); s < a.sg.n && (long)a.sg.start[s] * a.sg.unit < w0 + WM; ++s) {
        const int g = a.sg.id[s];
        if (g < 0) continue;
        const long lo = (long)a.sg.start[s] * a.sg.unit, hi = (long)a.sg.start[s + 1] * a.sg.unit;
        const bf16_t* Bg = a.B + (long)g * a.N * a.R;
        for (int rs = 0; rs < rsteps; ++rs) {
          const int r = rs * 32 + q * 8;
          const bool in = r < a.R;
          bf16x8_t tf[FM], bf[FN];
#pragma unroll
          for (int i = 0; i < FM; ++i) {
            const long m = w0 + i * 16 + i16;
            tf[i] = t_frag(a.T + m * a.R + r, in && m >= lo && m < hi);
          }
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            const int n = n0 + wn0 + j * 16 + i16;
            bf[j] = in && n < a.N ? load8(Bg + (long)n * a.R + r) : zero8();
          }
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mfma(bf[j], tf[i], acc[i][j]);
        }
      }
  }

  const int kt = (a.K + BK - 1) / BK;
  int rd = 0, wr = NSTG - 1;
  for (int t = 0; t < kt; ++t) {
    // every step issues NLD copies (past the end: out of range, zero fill), so the count of those still allowed in flight is a constant
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NSTG - 2) * NLD) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue(wr);
    const char *pa = lds + rd * STAGE, *pb = pa + BM * 128;
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      bf16x8_t fa[FM], fb[FN];
      const int chunk = ks * 4 + q;
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[i] = *reinterpret_cast<const bf16x8_t*>(pa + lds_off(wm0 + i * 16 + i16, chunk));
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = *reinterpret_cast<const bf16x8_t*>(pb + lds_off(wn0 + j * 16 + i16, chunk));
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma(fb[j], fa[i], acc[i][j]);
    }
    rd = rd + 1 == NSTG ? 0 : rd + 1;
    wr = wr + 1 == NSTG ? 0 : wr + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the zero-filling copies still write LDS
  __syncthreads();
  // the fp32 tile through LDS: rows leave as 16-byte stores, bias and residual are added before the one rounding
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
      *reinterpret_cast<f32x4_t*>(lds + (wm0 + i * 16 + i16) * PITCH + (wn0 + j * 16 + q * 4) * 4) = acc[i][j];
  __syncthreads();
  for (int id = tid; id < BM * (BN / 8); id += 256) {
    const int row = id / (BN / 8), c = id % (BN / 8);
    const long m = m0 + row;
    const int n = n0 + c * 8;
    if (m >= a.M || n >= a.N) continue;
    const float4 u = *reinterpret_cast<const float4*>(lds + row * PITCH + c * 32), w = *reinterpret_cast<const float4*>(lds + row * PITCH + c * 32 + 16);
    float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
    auto add = [&](const bf16_t* p) {
      const uint4 b = *reinterpret_cast<const uint4*>(p);
      v[0] += bf16lo(b.x), v[1] += bf16hi(b.x), v[2] += bf16lo(b.y), v[3] += bf16hi(b.y);
      v[4] += bf16lo(b.z), v[5] += bf16hi(b.z), v[6] += bf16lo(b.w), v[7] += bf16hi(b.w);
    };
    if (a.bias) add(a.bias + n);
    if (a.res) add(a.res + m * a.ldr + n);
    *reinterpret_cast<uint4*>(a.Y + m * a.ldy + n) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
}

// ------------------------------------------------------------------------------------------------------------------ weight gradients
// The rows of all adapters in sorted order (adapter by adapter, segment by segment) are one axis of `rows` positions, cut into chunks of `chunk`
// positions.  A workgroup takes one chunk x 128 columns of V x RB columns of U; where adapters change inside its chunk it finishes one and
// begins the next.  Piece (chunk b, j-th used adapter) is partial sum b + j: along the axis every new piece raises b or j.  A second launch adds
// an adapter's partial sums in their order: no atomics, the same bits every time.
struct Order {
  const int* seg_start;   // [n] first row of the k-th segment in sorted order, in units
  const int* seg_pos;     // [n + 1] its first position, in units
  const int* used_pos;    // [nused + 1] first position of the j-th used adapter, in units
  const int* used_id;     // [nused]
  const int* slot;        // [nslot] j of adapter g, or -1
  int n, nused, nslot, unit;
  long rows;
};

typedef short v4s_t __attribute__((ext_vector_type(4)));
template <int PB>
__device__ __forceinline__ int tr_off(int row, int chunk) { return row * PB + ((chunk ^ ((row & 7) << 1)) << 4); }   // PB >= 256: the XOR moves a chunk by up to 14
// 16 columns of 32 rows of a row-major LDS tile as an operand fragment whose contraction runs over the rows.  Both operands are read with
// the same gather, so the order in which it puts the 32 rows into the fragment's slots does not matter.
template <int PB>
__device__ __forceinline__ bf16x8_t tr_frag(const char* tile, int r32, int col0, int lane) {
  const int p = lane & 15, row = r32 * 32 + (lane >> 4) * 4 + (p >> 2);   // rows row and row + 16 have the same row & 7
  const char* b = tile + tr_off<PB>(row, (col0 >> 3) + ((p & 3) >> 1)) + (p & 1) * 8;
  const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_t __attribute__((address_space(3)))*)(b));
  const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s_t __attribute__((address_space(3)))*)(b + 16 * PB));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <int RB, bool CODES, bool TRANS>   // TRANS: partial sums as [C][R] (dB), else [R][C] (dA)
__global__ __launch_bounds__(256) void wgrad_kernel(const float* __restrict__ U, int R, const bf16_t* __restrict__ V, long ldv,
                                                    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, int C, Order o,
                                                    int chunk, float* __restrict__ part) {
  constexpr int TK = 64, CB = 128, PV = 256, PU = RB == 32 ? 256 : 512, FU = RB / 16;
  __shared__ __attribute__((aligned(16))) char vt[TK * PV], ut[TK * PU];
  __shared__ int rowof[TK];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c0 = blockIdx.y * CB, r0 = blockIdx.z * RB;
  const long p_begin = (long)blockIdx.x * chunk, p_end = min(p_begin + chunk, o.rows);
  int j = 0;   // the used adapter that holds p_begin
  for (int hi = o.nused; hi - j > 1;) {
    const int mid = (j + hi) >> 1;
    if ((long)o.used_pos[mid] * o.unit <= p_begin) j = mid;
    else hi = mid;
  }
  const int cp = (C + 31) / 32 * 32;
  for (long p = p_begin; p < p_end; ++j) {
    const long piece_end = min(p_end, (long)o.used_pos[j + 1] * o.unit);
    f32x4_t acc[2][FU];   // 32 columns of V per wavefront
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int u = 0; u < FU; ++u) acc[v][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (; p < piece_end; p += TK) {
      const int nrow = (int)min((long)TK, piece_end - p);
      __syncthreads();   // the last tile's fragments have been read
      if (tid < TK) {
        int row = -1;
        if (tid < nrow) {
          const long pos = p + tid;
          int lo = 0, hi = o.n;
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((long)o.seg_pos[mid] * o.unit <= pos) lo = mid;
            else hi = mid;
          }
          row = (int)((long)o.seg_start[lo] * o.unit + (pos - (long)o.seg_pos[lo] * o.unit));
        }
        rowof[tid] = row;
      }
      __syncthreads();
#pragma unroll
      for (int l = 0; l < TK * CB / 8 / 256; ++l) {
        const int row = (tid >> 4) + 16 * l, ch = tid & 15, c = c0 + ch * 8;
        const long m = rowof[row];
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (m >= 0 && c < C) {
          if constexpr (CODES) {
            const uint2 k = *reinterpret_cast<const uint2*>(codes + m * cp + c);
            const float st = act8::step(exps[m * (cp >> 5) + (c >> 5)]);
            float v[8];
            act8::values4(k.x, st, v);
            act8::values4(k.y, st, v + 4);
            w = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
          } else {
            w = *reinterpret_cast<const uint4*>(V + m * ldv + c);
          }
        }
        *reinterpret_cast<uint4*>(vt + tr_off<PV>(row, ch)) = w;
      }
#pragma unroll
      for (int l = 0; l < TK * RB / 8 / 256; ++l) {
        const int id = tid + 256 * l, row = id / (RB / 8), ch = id % (RB / 8), r = r0 + ch * 8;
        const long m = rowof[row];
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (m >= 0 && r < R) {
          const float4 x = *reinterpret_cast<const float4*>(U + m * R + r), y = *reinterpret_cast<const float4*>(U + m * R + r + 4);
          v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
        }
        // v = h + m + l, three bf16 parts that hold 24 bits (each difference is exact)
#pragma unroll
        for (int part3 = 0; part3 < 3; ++part3) {
          const uint4 w = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
          *reinterpret_cast<uint4*>(ut + tr_off<PU>(row, part3 * (RB / 8) + ch)) = w;
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[2 * e] -= bf16lo(ww[e]);
            v[2 * e + 1] -= bf16hi(ww[e]);
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < TK / 32; ++s) {
        bf16x8_t fv[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) fv[v] = tr_frag<PV>(vt, s, wave * 32 + v * 16, lane);
#pragma unroll
        for (int part3 = 2; part3 >= 0; --part3)
#pragma unroll
          for (int u = 0; u < FU; ++u) {
            const bf16x8_t fu = tr_frag<PU>(ut, s, part3 * RB + u * 16, lane);
#pragma unroll
            for (int v = 0; v < 2; ++v) acc[v][u] = TRANS ? mfma(fu, fv[v], acc[v][u]) : mfma(fv[v], fu, acc[v][u]);
          }
      }
    }
    p = piece_end;
    float* out = part + (long)(blockIdx.x + j) * R * C;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int u = 0; u < FU; ++u) {
        const int cb = c0 + wave * 32 + v * 16, rb = r0 + u * 16, a = (lane >> 4) * 4, b = lane & 15;
        if (TRANS) {   // lane: column b of V, columns a .. a + 3 of U
          if (cb + b < C && rb + a < R) *reinterpret_cast<f32x4_t*>(out + (long)(cb + b) * R + rb + a) = acc[v][u];
        } else {       // lane: column b of U, columns a .. a + 3 of V
          if (rb + b < R && cb + a < C) *reinterpret_cast<f32x4_t*>(out + (long)(rb + b) * C + cb + a) = acc[v][u];
        }
      }
  }
}

// out[g] = sum of the partial sums of adapter g; zeros for an adapter without rows and past an adapter's rank
template <bool TRANS>
__global__ __launch_bounds__(256) void wgrad_reduce_kernel(const float* __restrict__ part, int R, int C, int r_out, const int* __restrict__ ranks, Order o,
                                                           int chunk, float* __restrict__ out) {
  const int g = blockIdx.y;
  const long id = (long)blockIdx.x * 256 + threadIdx.x, n = (long)r_out * C;
  if (id >= n) return;
  const int r = (int)(TRANS ? id % r_out : id / C);
  const long at = TRANS ? id / r_out * R + r : id;
  const int j = g < o.nslot ? o.slot[g] : -1;
  float s = 0.f;
  if (j >= 0 && r < ranks[g]) {
    const long first = (long)o.used_pos[j] * o.unit, last = (long)o.used_pos[j + 1] * o.unit - 1;
    const long b1 = last / chunk + j;
    for (long b = first / chunk + j; b <= b1; ++b) s += part[b * R * C + at];
  }
  out[g * n + id] = s;
}

int wgrad_chunk(long rows, int C, int R) {
  const long tiles = (long)((C + 127) / 128) * (R <= 32 ? 1 : (R + 63) / 64);
  long want = 1024 / tiles;   // workgroups: four per CU
  if (want < 1) want = 1;
  long ch = (rows + want - 1) / want;
  ch = (ch + 63) / 64 * 64;
  return (int)(ch < 64 ? 64 : ch > (1 << 20) ? (1 << 20) : ch);
}

void launch_down(const bf16_t* X, long ldx, const uint8_t* codes, const uint8_t* exps, long M, int K, const bf16_t* A, const int* ranks, const float* scales, int R,
                 const Segs& sg, int slots, float* T, hipStream_t st) {
  const int t16 = (R + 15) / 16, rt = t16 == 1 ? 1 : 2;
  const dim3 grid((unsigned)((M + 15) / 16), slots, (t16 + rt - 1) / rt);
#define AQL_DOWN(RT, CODES) hipLaunchKernelGGL((down_kernel<RT, CODES>), grid, dim3(256), 0, st, X, ldx, codes, exps, M, K, A, ranks, scales, R, sg, T)
  if (codes) {
    if (rt == 1) AQL_DOWN(1, true);
    else AQL_DOWN(2, true);
  } else {
    if (rt == 1) AQL_DOWN(1, false);
    else AQL_DOWN(2, false);
  }
#undef AQL_DOWN
}

bool seg_ok(const void* start, const void* id, int n, int unit) { return n >= 0 && (n == 0 || (start && id && unit >= 1)); }

}  // namespace

// Y = X W^T + bias + residual + the low-rank term; T: [M][R] fp32, written for the rows that have an adapter.  slots: the most segments that meet in one tile
// of 16 rows (16-aligned tiles of rows).
extern "C" int aql_adapter_linear(const bf16_t* X, long ldx, const bf16_t* W, long ldw, const bf16_t* bias, const bf16_t* residual, long ldr, bf16_t* Y,
                                  long ldy, long M, int N, int K, const bf16_t* A, const bf16_t* B, const int* ranks, const float* scales, int R,
                                  const int* seg_start, const int* seg_id, int nseg, int unit, int slots, float* T, hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && M < (1L << 31) - 256 && N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0, "aql_adapter_linear: bad shape M=%ld N=%d K=%d (N, K: multiples of 8)", M, N, K);
  if (M == 0) return AQL_OK;
  AQL_CHECK_ARG(X && W && Y, "aql_adapter_linear: null operand");
  AQL_CHECK_ARG(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N) && ldx % 8 == 0 && ldw % 8 == 0 && ldy % 8 == 0 && ldr % 8 == 0 && ldx < (1L << 21) &&
                    ldw < (1L << 21), "aql_adapter_linear: leading dimensions (multiples of 8, at least the width, below 2^21)");
  AQL_CHECK_ARG((((uintptr_t)X | (uintptr_t)W | (uintptr_t)bias | (uintptr_t)residual | (uintptr_t)Y) & 15) == 0, "aql_adapter_linear: operands must be 16-byte aligned");
  AQL_CHECK_ARG(seg_ok(seg_start, seg_id, nseg, unit) && (nseg == 0 || (A && B && ranks && scales && T && R > 0 && R % 8 == 0 && slots >= 1 && slots <= 16)),
                "aql_adapter_linear: bad adapters (R=%d: a multiple of 8) or segments", R);
  const Segs sg{seg_start, seg_id, nseg, unit};
  if (nseg) {
    launch_down(X, ldx, nullptr, nullptr, M, K, A, ranks, scales, R, sg, slots, T, stream);
    AQL_CHECK_LAUNCH("aql_adapter_linear (down)");
  }
  const LinArgs a{X, W, bias, residual, B, Y, T, ldx, ldw, ldr, ldy, M, N, K, R, sg};
  if (M <= 256) {
    hipLaunchKernelGGL((skinny_kernel<1>), dim3((N + 15) / 16, (unsigned)((M + 15) / 16)), dim3(512), 0, stream, a);
  } else {
    const long big = ((M + 127) / 128) * ((N + 127) / 128);
    if (big >= 256)
      hipLaunchKernelGGL((tile_kernel<128, 128, 2>), dim3((unsigned)big), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((tile_kernel<64, 64, 3>), dim3((unsigned)(((M + 63) / 64) * ((N + 63) / 64))), dim3(256), 0, stream, a);
  }
  AQL_CHECK_LAUNCH("aql_adapter_linear");
  return AQL_OK;
}

// T = s A x alone, from X or from its 8-bit codes
extern "C" int aql_adapter_down(const bf16_t* X, long ldx, const uint8_t* codes, const uint8_t* exps, long M, int K, const bf16_t* A, const int* ranks,
                                const float* scales, int R, const int* seg_start, const int* seg_id, int nseg, int unit, int slots, float* T,
                                hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && M < (1L << 31) - 256 && K > 0 && K % 8 == 0 && R > 0 && R % 8 == 0, "aql_adapter_down: bad shape M=%ld K=%d R=%d", M, K, R);
  AQL_CHECK_ARG(seg_ok(seg_start, seg_id, nseg, unit), "aql_adapter_down: bad segments");
  if (M == 0 || nseg == 0) return AQL_OK;
  AQL_CHECK_ARG(!codes == !exps && !X != !codes && (!X || (ldx >= K && ldx % 8 == 0 && ((uintptr_t)X & 15) == 0)) && A && ranks && scales && T && slots >= 1 && slots <= 16,
                "aql_adapter_down: bad operands (exactly one of X and its codes)");
  launch_down(X, ldx, codes, exps, M, K, A, ranks, scales, R, Segs{seg_start, seg_id, nseg, unit}, slots, T, stream);
  AQL_CHECK_LAUNCH("aql_adapter_down");
  return AQL_OK;
}

// fp32 elements of the workspace of aql_adapter_wgrad (rows: those that have an adapter; nused: adapters that have rows), or -1: more than 2^31 - 1
extern "C" int aql_adapter_wgrad_scratch_floats(long rows, int nused, int C, int R) {
  if (rows <= 0 || nused <= 0 || C <= 0 || R <= 0) return 0;
  const int ch = wgrad_chunk(rows, C, R);
  const double n = (double)((rows + ch - 1) / ch + nused - 1) * R * C;
  return n < 2147483647.0 ? (int)n : -1;
}

extern "C" int aql_adapter_wgrad(const float* U, int R, const bf16_t* V, long ldv, const uint8_t* codes, const uint8_t* exps, long M, int C, int G, int r_out,
                                 const int* ranks, const int* seg_start, const int* seg_pos, const int* used_pos, const int* used_id, const int* slot, int nseg,
                                 int nused, int nslot, int unit, long rows, int trans, float* out, float* scratch, long scratch_floats, hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && M < (1L << 31) - 256 && C > 0 && C % 8 == 0 && R > 0 && R % 8 == 0 && G > 0 && G <= 65535 && r_out > 0 && r_out <= R && rows >= 0 && rows <= M,
                "aql_adapter_wgrad: bad shape M=%ld C=%d R=%d G=%d", M, C, R, G);
  AQL_CHECK_ARG(out && ranks && !codes == !exps && !V != !codes && (V == nullptr || (ldv >= C && ldv % 8 == 0 && ((uintptr_t)V & 15) == 0)), "aql_adapter_wgrad: bad operands");
  AQL_CHECK_ARG(rows == 0 || (U && seg_start && seg_pos && used_pos && used_id && slot && nseg > 0 && nused > 0 && nslot > 0 && unit >= 1), "aql_adapter_wgrad: bad segments");
  const int need = aql_adapter_wgrad_scratch_floats(rows, nused, C, R);
  AQL_CHECK_ARG(need >= 0 && scratch_floats >= need && (need == 0 || scratch), "aql_adapter_wgrad: workspace of %ld floats, %d needed", scratch_floats, need);
  Order o{seg_start, seg_pos, used_pos, used_id, slot, nseg, nused, rows ? nslot : 0, unit, rows};
  const int ch = rows ? wgrad_chunk(rows, C, R) : 64;
  if (rows) {
    const dim3 grid((unsigned)((rows + ch - 1) / ch), (C + 127) / 128, R <= 32 ? 1 : (R + 63) / 64);
#define AQL_WG(RB, CODES, TRANS) hipLaunchKernelGGL((wgrad_kernel<RB, CODES, TRANS>), grid, dim3(256), 0, stream, U, R, V, ldv, codes, exps, C, o, ch, scratch)
    if (R <= 32) {
      if (codes && trans) AQL_WG(32, true, true);
      else if (codes) AQL_WG(32, true, false);
      else if (trans) AQL_WG(32, false, true);
      else AQL_WG(32, false, false);
    } else {
      if (codes && trans) AQL_WG(64, true, true);
      else if (codes) AQL_WG(64, true, false);
      else if (trans) AQL_WG(64, false, true);
      else AQL_WG(64, false, false);
    }
#undef AQL_WG
    AQL_CHECK_LAUNCH("aql_adapter_wgrad");
  }
  const dim3 rgrid((unsigned)(((long)r_out * C + 255) / 256), G);
  if (trans)
    hipLaunchKernelGGL(wgrad_reduce_kernel<true>, rgrid, dim3(256), 0, stream, scratch, R, C, r_out, ranks, o, ch, out);
  else
    hipLaunchKernelGGL(wgrad_reduce_kernel<false>, rgrid, dim3(256), 0, stream, scratch, R, C, r_out, ranks, o, ch, out);
  AQL_CHECK_LAUNCH("aql_adapter_wgrad (sum)");
  return AQL_OK;
}
