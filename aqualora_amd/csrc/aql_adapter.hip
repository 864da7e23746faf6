// Low-rank adapters of many requests at once beside a shared projection.
//
// The rows of X belong to requests, the requests to adapters (or to none):  with g the adapter of row m
//     T[m] = s_g A_g x_m          (aql_adapter_linear, first launch; aql_adapter_down alone, also from 8-bit codes of X)
//     Y[m] = W x_m + b + B_g T[m] + residual_m        (second launch: one fp32 accumulator, one rounding)
// The backward-data pass is the same entry with exchanged operands (X = dY, W = W^T, A = B^T, B = A^T: T becomes dT, Y becomes dX), and
//     P_g = sum over the rows of g of  U[m] V[m]^T     (aql_adapter_wgrad: dA from (dT, X), dB from (T, dY))
// are the weight gradients.
//
// Row m has adapter id[m / unit], -1 for none: one load, whatever the requests' lengths (a binary search over their starts cost a chain of
// scalar loads: 15 us against 6 us where 16 requests meet in a tile of 16 rows).  Tiles of rows stay dense; the low-rank term runs once for each
// adapter that a tile meets, with the other adapters' T rows taken as zeros and their sums left alone (selects: neither what those rows hold
// nor an infinity or a NaN in this adapter's weights reaches another request).
//
// T is written as bf16 parts: T = hi + mid + lo, hi = T rounded to bf16, mid = the rest rounded, lo = the rest of that.  The second launch reads
// hi alone (the one rounding of T in the linear, as in the single-adapter kernels).  The gradients dA and dB are fp32 sums of T's products
// and would lose two thirds of their digits to a bf16 T: they read all three parts (24 bits), which only a training pass writes.
#include "aql_act8.cuh"

namespace {

constexpr int BK = 64;
constexpr uint32_t OOB = 0x80000000u;
constexpr int SPAN = 0x40000000;     // bytes from a tile's first row that its buffer descriptor covers: 256 rows of any leading dimension below 2^21
constexpr int MAX_R = 1 << 16;       // of the stacks: so that rows of T's three parts, and of B, do as well

struct Rows {
  const int* id;   // adapter of each unit of rows; null: no adapters at all
  int unit;
};
__device__ __forceinline__ int id_of(const Rows& r, long row) { return r.id[r.unit == 1 ? (uint32_t)row : (uint32_t)row / (uint32_t)r.unit]; }

__device__ __forceinline__ bf16x8_t zero8() { return bf16x8_t{0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ bf16x8_t load8(const bf16_t* p) { return *reinterpret_cast<const bf16x8_t*>(p); }
// loads that may be dead go to a clamped address and are selected afterwards: a load under a branch costs the branch, and the compiler, which no
// longer knows how many loads are in flight behind it, waits for all of them
__device__ __forceinline__ bf16x8_t keep(bf16x8_t v, bool on) {
  union { bf16x8_t f; uint32_t w[4]; } u;
  u.f = v;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.w[i] = on ? u.w[i] : 0u;
  return u.f;
}
__device__ __forceinline__ uint4 keep(uint4 v, bool on) { return make_uint4(on ? v.x : 0u, on ? v.y : 0u, on ? v.z : 0u, on ? v.w : 0u); }
__device__ __forceinline__ bf16x8_t pack8(const float* v) {
  union { uint32_t w[4]; bf16x8_t f; } u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  return u.f;
}
// T's parts of row m: hi at T + m P R, mid and lo R and 2 R further on (P = 1: hi alone, P = 3)
__device__ __forceinline__ void store_t4(bf16_t* t, int R, int P, const float (&v)[4]) {   // four consecutive columns
  float r[4] = {v[0], v[1], v[2], v[3]};
  for (int p = 0; p < P; ++p) {
    const uint2 w = make_uint2(pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]));
    *reinterpret_cast<uint2*>(t + p * R) = w;
    r[0] -= bf16lo(w.x), r[1] -= bf16hi(w.x), r[2] -= bf16lo(w.y), r[3] -= bf16hi(w.y);   // exact
  }
}
__device__ __forceinline__ void store_t8(bf16_t* t, int R, int P, const float (&v)[8]) {   // eight
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
  for (int p = 0; p < P; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = pack_bf16x2(r[2 * k], r[2 * k + 1]);
      r[2 * k] -= bf16lo(w[k]), r[2 * k + 1] -= bf16hi(w[k]);
    }
    *reinterpret_cast<uint4*>(t + p * R) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// ---------------------------------------------------------------------------------------------------------------------- T = s A x
struct DownArgs {
  const bf16_t* X;
  const uint8_t *codes, *exps;
  const bf16_t* A;
  const int* ranks;
  const float* scales;
  bf16_t* T;
  long ldx, M;
  int K, R, P;
  Rows rows;
};

// Few rows or short requests: bound by the latency of row -> adapter -> loads (8 x 1280, rank 32: 4.0 us).  One workgroup: 16 rows x 16 RT adapter rows of ONE adapter (blockIdx.y counts the adapters that the row
// tile meets); its NW wavefronts split the contraction and join in LDS.  Fragments come straight from memory, four steps of 32 columns at a time
// (all their loads in flight together): lane (i = lane & 15, q = lane >> 4) holds row i, columns k + 8 q .. k + 8 q + 7 of either operand, and
// gets T[m = lane & 15][r = 4 q + e] back.
template <int RT, int NW, bool CODES>
__global__ __launch_bounds__(NW * 64) void down_kernel(const DownArgs a) {
  constexpr int UN = 4;
  __shared__ float red[NW - 1][RT][64][4];
  const long m0 = (long)blockIdx.x * 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const int gi = m0 + i < a.M ? id_of(a.rows, m0 + i) : -1;
  uint32_t left = (uint32_t)__ballot(gi >= 0) & 0xffffu;   // rows whose adapter has not been met yet
  int g = -1;
  for (int k = blockIdx.y; left; --k) {                    // the blockIdx.y-th adapter of the tile, in order of its first row
    g = __builtin_amdgcn_readlane(gi, __builtin_ctz(left));
    if (k == 0) break;
    left &= ~(uint32_t)__ballot(gi == g);
    g = -1;
  }
  if (g < 0) return;
  const float sc = a.scales[g];   // (here, and bias and residual in the next kernel likewise: behind the join their latency would show)
  const int rank = a.ranks[g];
  const int r0 = blockIdx.z * 16 * RT;
  const int ksteps = (a.K + 31) / 32;
  const long m = min(m0 + i, a.M - 1);
  const bf16_t* Ag = a.A + (long)g * a.R * a.K;
  f32x4_t acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave * UN; kb < ksteps; kb += NW * UN) {
    bf16x8_t xf[UN], af[UN][RT];
    uint2 cd[UN];
    uint32_t ex[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int k = (kb + u) * 32 + q * 8;
      const bool in = k < a.K;
      const int kc = in ? k : 0;
      if constexpr (CODES) {
        cd[u] = *reinterpret_cast<const uint2*>(a.codes + m * (long)(ksteps * 32) + kc);
        ex[u] = a.exps[m * (long)ksteps + (kc >> 5)];
      } else {
        xf[u] = load8(a.X + m * a.ldx + kc);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) af[u][t] = load8(Ag + (long)min(r0 + t * 16 + i, a.R - 1) * a.K + kc);   // (rows past R are never stored)
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if constexpr (CODES) {
        float v[8];
        act8::values4(cd[u].x, act8::step(ex[u]), v);
        act8::values4(cd[u].y, act8::step(ex[u]), v + 4);
        xf[u] = pack8(v);
      }
      const bool in = (kb + u) * 32 + q * 8 < a.K;
      xf[u] = keep(xf[u], in);
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[t] = mfma(keep(af[u][t], in), xf[u], acc[t]);
    }
  }
  if (wave) {
#pragma unroll
    for (int t = 0; t < RT; ++t) *reinterpret_cast<f32x4_t*>(red[wave - 1][t][lane]) = acc[t];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + t * 16 + q * 4;
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = acc[t][e];
#pragma unroll
      for (int w = 0; w < NW - 1; ++w) v += red[w][t][lane][e];
      o[e] = r + e < rank ? sc * v : 0.f;   // columns past the adapter's rank are 0 whatever x holds
    }
    if (gi == g && r < a.R) store_t4(a.T + m * a.P * a.R + r, a.R, a.P, o);
  }
}

struct LinArgs {
  const bf16_t *X, *W, *bias, *res, *B;
  bf16_t* Y;
  const bf16_t* T;
  long ldx, ldw, ldr, ldy, M;
  int N, K, R, P;
  Rows rows;   // id null: no low-rank term
};

// ------------------------------------------------------------------------------------------- few rows: 16 x 16 NF tiles, split contraction
// Eight wavefronts split the contraction of one tile (and the tile's (adapter, rank step) pairs) and join in LDS: with few rows the launch is
// bound by the latency of the weight loads, so the loads of a tile are spread over as many wavefronts as it can feed and issued UN steps at a time
// (8 x 1280 x 1280, eight adapters: 5.3 us, a whole call without adapters 3.7; 193 x 1280 x 320, 48 adapters: 8.0).
template <int NF>
__global__ __launch_bounds__(512) void skinny_kernel(const LinArgs a) {
  constexpr int UN = 4;
  __shared__ float red[8][NF][64][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
  const long m0 = (long)blockIdx.y * 16;
  const int n0 = blockIdx.x * 16 * NF;
  const int ksteps = (a.K + 31) / 32;
  const long m = min(m0 + i, a.M - 1);
  const int gi = a.rows.id && m0 + i < a.M ? id_of(a.rows, m0 + i) : -1;
  // wavefront j < NF writes fragment j at the end: row m0 + i, columns n0 + 16 j + 4 q ..
  const long mw = m0 + i;
  const int nw = n0 + wave * 16 + q * 4;
  const bool writes = wave < NF && mw < a.M && nw < a.N;
  uint2 add[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
  if (writes && a.bias) add[0] = *reinterpret_cast<const uint2*>(a.bias + nw);
  if (writes && a.res) add[1] = *reinterpret_cast<const uint2*>(a.res + mw * a.ldr + nw);
  f32x4_t acc[NF];
#pragma unroll
  for (int j = 0; j < NF; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave * UN; kb < ksteps; kb += 8 * UN) {
    bf16x8_t xf[UN], wf[UN][NF];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int k = (kb + u) * 32 + q * 8;
      const bool in = k < a.K;
      const int kc = in ? k : 0;
      xf[u] = load8(a.X + m * a.ldx + kc);
#pragma unroll
      for (int j = 0; j < NF; ++j) wf[u][j] = load8(a.W + (long)min(n0 + j * 16 + i, a.N - 1) * a.ldw + kc);   // (rows past N are never stored)
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const bool in = (kb + u) * 32 + q * 8 < a.K;
      xf[u] = keep(xf[u], in);
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[j] = mfma(keep(wf[u][j], in), xf[u], acc[j]);
    }
  }
  uint32_t left = (uint32_t)__ballot(gi >= 0) & 0xffffu;   // rows whose adapter is still to come
  const int rsteps = (a.R + 31) / 32;
  for (int turn = 0; left;) {
    const int g = __builtin_amdgcn_readlane(gi, __builtin_ctz(left));
    left &= ~(uint32_t)__ballot(gi == g);
    const bf16_t* Bg = a.B + (long)g * a.N * a.R;
    for (int rs = 0; rs < rsteps; ++rs, ++turn) {
      if ((turn & 7) != wave) continue;
      const int r = rs * 32 + q * 8;
      const bool in = r < a.R;
      const bf16x8_t tf = in && gi == g ? load8(a.T + m * a.P * a.R + r) : zero8();
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const int n = n0 + j * 16 + i;
        const bf16x8_t bf = in && n < a.N ? load8(Bg + (long)n * a.R + r) : zero8();
        const f32x4_t v = mfma(bf, tf, acc[j]);   // the other rows keep their sums by a select: B may hold an infinity or a NaN
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = gi == g ? v[e] : acc[j][e];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NF; ++j) *reinterpret_cast<f32x4_t*>(red[wave][j][lane]) = acc[j];
  __syncthreads();
  if (!writes) return;
  float v[4] = {bf16lo(add[0].x) + bf16lo(add[1].x), bf16hi(add[0].x) + bf16hi(add[1].x), bf16lo(add[0].y) + bf16lo(add[1].y), bf16hi(add[0].y) + bf16hi(add[1].y)};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) t += red[w][wave][lane][e];
    v[e] += t;
  }
  *reinterpret_cast<uint2*>(a.Y + mw * a.ldy + nw) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// ------------------------------------------------------------------------------------------------------------- many rows: LDS tiles
// Rows of 128 bytes; the chunks of a row are exchanged by a number made of its bits so that the 16 rows of a fragment, neighbours or as pair_row takes
// them, fall on different banks
__device__ __forceinline__ int lds_mix(int row) { return ((row >> 1) & 1) | ((row >> 2) & 2) | (((row >> 2) ^ (row >> 4)) & 1) << 2; }
__device__ __forceinline__ int lds_off(int row, int chunk) { return row * 128 + ((chunk ^ lds_mix(row)) << 4); }
// the row of W that fragment j, lane row i, of FN fragments reads: two neighbouring fragments together cover 32 columns such that a lane ends with eight
// consecutive ones of its row (4 of each) and moves them 16 bytes at a time; the last of an odd number is read as it is
template <int FN>
__device__ __forceinline__ int pair_row(int j, int i) {
  return j + 1 == FN && FN % 2 ? j * 16 + i : (j >> 1) * 32 + (i >> 2) * 8 + (j & 1) * 4 + (i & 3);
}

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, voff, soff, 0, 0);
}

// rows x 64 columns of one operand, global -> LDS, by NW wavefronts; lane (row = tid >> 3, slot = tid & 7) fetches source chunk slot ^ lds_mix(row)
template <int ROWS, int NW>
struct Stage {
  static constexpr int RPI = 8 * NW, NL = ROWS / RPI;
  static_assert(ROWS % RPI == 0 && RPI % 32 == 0, "whole copies, of rows with the same lds_mix");
  __amdgpu_buffer_rsrc_t rs;
  uint32_t voff[NL], soff;
  int krem, kc;
  // base: first row of the tile; live(r): whether row r of the tile is read (others are zeros)
  template <class L>
  __device__ __forceinline__ void begin(const bf16_t* base, long ld, int K, int tid, L live) {
    rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(base), 0, SPAN, 0x00020000);
    kc = ((tid & 7) ^ lds_mix(tid >> 3)) * 8;
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int r = (tid >> 3) + RPI * l;
      voff[l] = live(r) ? (uint32_t)r * (uint32_t)(ld * 2) + kc * 2 : OOB;
    }
    soff = 0;
    krem = K;
  }
  __device__ __forceinline__ void fetch(char* dst, int wave) {
    const bool bad = kc >= krem;
#pragma unroll
    for (int l = 0; l < NL; ++l) dma16(rs, dst + (RPI * l + 8 * wave) * 128, bad ? OOB : voff[l], soff);
    soff += BK * 2;
    krem -= BK;
  }
};

// A ring of NSTG LDS stages of 64 columns, NSTG - 1 in flight, one barrier per stage.  issue(st) starts the next stage's copies (NLD per wavefront,
// always: past the end they are out of range and fill zeros, so the count of copies still allowed in flight is a constant).
template <int BM, int BN, int NW, int NSTG>
struct Ring {
  static constexpr int STAGE = (BM + BN) * 128, NLD = (BM + BN) / (8 * NW);
  char* lds;
  int rd = 0, wr = NSTG - 1;
  template <class I>
  __device__ __forceinline__ const char* turn(I issue) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NSTG - 2) * NLD) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue(wr);
    const char* p = lds + rd * STAGE;
    rd = rd + 1 == NSTG ? 0 : rd + 1;
    wr = wr + 1 == NSTG ? 0 : wr + 1;
    return p;
  }
  __device__ __forceinline__ void drain() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }   // the zero-filling copies still write LDS
};

// acc += one stage's product.  The weight-side fragment is MFMA operand A, so a lane ends with four consecutive columns (4 q + e; PAIRS: see pair_row)
// of one row (lane & 15).  SOME: only rows of fragments i with bit i of `own` set in their lanes take part; the others keep their sums by a select, whatever the weight
// side holds (a zero row against an infinity or a NaN would add a NaN).
template <int BM, int BN, int WGM, int WGN, bool PAIRS, bool SOME = false>
__device__ __forceinline__ void products(const char* pa, int wave, int lane, f32x4_t (&acc)[BM / WGM / 16][BN / WGN / 16], uint32_t own = 0) {
  constexpr int WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16;
  if constexpr (SOME) asm volatile("" : "+v"(lane));   // (its addresses are made anew: kept beside the other loop's they would spill)
  const int i16 = lane & 15, q = lane >> 4, wm0 = (wave / WGN) * WM, wn0 = (wave % WGN) * WN;
  const char* pb = pa + BM * 128;
#pragma unroll
  for (int ks = 0; ks < BK / 32; ++ks) {
    bf16x8_t fa[FM], fb[FN];
    const int chunk = ks * 4 + q;
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[j] = *reinterpret_cast<const bf16x8_t*>(pb + lds_off(wn0 + (PAIRS ? pair_row<FN>(j, i16) : j * 16 + i16), chunk));
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = *reinterpret_cast<const bf16x8_t*>(pa + lds_off(wm0 + i * 16 + i16, chunk));
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const f32x4_t v = mfma(fb[j], fa[i], acc[i][j]);
        if constexpr (SOME) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = own >> i & 1 ? v[e] : acc[i][j][e];
        } else {
          acc[i][j] = v;
        }
      }
  }
}

// consecutive workgroups go to the eight XCDs in turn: XCD x takes the x-th eighth of the tiles, so that tiles that share operands share an L2
__device__ __forceinline__ uint32_t xcd_tile(uint32_t b, uint32_t n) {
  const uint32_t x = b & 7, i = b >> 3, q = n >> 3, r = n & 7;
  return x * q + min(x, r) + i;
}

template <int CTRL>
__device__ __forceinline__ uint32_t row_umin(uint32_t v) { return min(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false)); }
__device__ __forceinline__ uint32_t wave_umin(uint32_t v) {   // four rotations of 16 lanes, then the four rows: a scalar
  v = row_umin<0x121>(row_umin<0x122>(row_umin<0x124>(row_umin<0x128>(v))));
  const auto at = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return min(min(at(0), at(16)), min(at(32), at(48)));
}

// the smallest adapter above `after` among the BM rows of a tile (ids in LDS), or -1; the same in every lane of every wavefront
template <int BM>
__device__ __forceinline__ int next_adapter(const int* ids, int after, int lane) {
  uint32_t best = 0x7fffffffu;
#pragma unroll
  for (int k = 0; k < BM / 64; ++k) {
    const int g = ids[k * 64 + lane];
    best = min(best, g > after ? (uint32_t)g : 0x7fffffffu);
  }
  best = wave_umin(best);
  const int g = (int)best;
  return g == 0x7fffffff ? -1 : g;
}

// whether all `live` rows of a tile have adapter g
template <int BM>
__device__ __forceinline__ bool one_adapter(const int* ids, int g, int live, int lane) {
  bool all = true;
#pragma unroll
  for (int k = 0; k < BM / 64; ++k) all = all && (ids[k * 64 + lane] == g || k * 64 + lane >= live);
  return __ballot(all) == ~0ull;
}

// WGM x WGN wavefronts, BM x BN outputs.  The low-rank term of each adapter that the tile meets goes through the same ring, behind the projection's
// own columns: R further columns of the contraction, the adapter's rows of T against its B.  (Fragments of T and B
// straight from memory instead cost a load latency per 32 columns of rank: 28 against 18 us at 4096 x 640 x 640, rank 320.)  Large calls are bound by the
// matrix cores and the LDS reads that feed them (4096 x 10240 x 1280, rank 32: 109 us, 1.0 PFLOP/s), small ones by the latency of their stages
// (1001 x 640 x 768, rank 64: 8.6 us for 12 + 1 stages).
// What the tile may meet: ANY adapters; ONE or none (the caller knows); or FIND out -- where it is not one or none, false comes back and nothing is written.
enum Meets { ANY, ONE, FIND };
template <int BM, int BN, int WGM, int WGN, int NSTG, Meets MEETS>
__device__ __forceinline__ bool tile_body(const LinArgs& a, char* lds, long m0, int n0) {
  constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16, STAGE = (BM + BN) * 128;
  int* ids = reinterpret_cast<int*>(lds + NSTG * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i16 = lane & 15, q = lane >> 4;
  const int mlive = (int)min((long)BM, a.M - m0), nlive = min(BN, a.N - n0);
  const long w0 = m0 + (wave / WGN) * WM;          // this wavefront's rows and columns
  const int v0 = n0 + (wave % WGN) * WN;
  // the fp32 sums begin with bias and residual: their loads run under the first copies instead of behind the last product, and there is one rounding
  f32x4_t acc[FM][FN];
  constexpr int FP = FN / 2, FO = FN % 2;   // pairs of fragments, and a last one
  const auto low = [](uint4 b) { return f32x4_t{bf16lo(b.x), bf16hi(b.x), bf16lo(b.y), bf16hi(b.y)}; };
  const auto high = [](uint4 b) { return f32x4_t{bf16lo(b.z), bf16hi(b.z), bf16lo(b.w), bf16hi(b.w)}; };
  // eight columns of pair p, four of the last fragment; past the end: the last columns, never stored
  const auto load = [&](const bf16_t* row, int j) {
    if (j < 2 * FP) return *reinterpret_cast<const uint4*>(row + min(v0 + j * 16 + q * 8, a.N - 8));
    const uint2 v = *reinterpret_cast<const uint2*>(row + min(v0 + j * 16 + q * 4, a.N - 4));
    return make_uint4(v.x, v.y, 0u, 0u);
  };
#pragma unroll
  for (int j = 0; j < FN; j += 2) {
    const uint4 b = a.bias ? load(a.bias, j) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      acc[i][j] = low(b);
      if (j < 2 * FP) acc[i][j + 1 < FN ? j + 1 : j] = high(b);
    }
  }
  if (a.res) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const bf16_t* p = a.res + min(w0 + i * 16 + i16, a.M - 1) * a.ldr;
#pragma unroll
      for (int j = 0; j < FN; j += 2) {
        const uint4 r = load(p, j);
        acc[i][j] += low(r);
        if (j < 2 * FP) acc[i][j + 1 < FN ? j + 1 : j] += high(r);
      }
    }
  }
  Stage<BM, NW> sx;
  Stage<BN, NW> sw;
  sx.begin(a.X + m0 * a.ldx, a.ldx, a.K, tid, [&](int r) { return r < mlive; });
  sw.begin(a.W + (long)n0 * a.ldw, a.ldw, a.K, tid, [&](int r) { return r < nlive; });
  const int nk = (a.K + BK - 1) / BK;
  int left = nk, g = -1;   // stages still to be copied of the current part; its adapter
  const int rk = (a.R + BK - 1) / BK;
  auto issue = [&](int st) {
    if (left == 0 && a.rows.id != nullptr) {   // (uniform)
      g = next_adapter<BM>(ids, g, lane);
      left = g < 0 ? 1 << 30 : rk;
      if (g >= 0) {
        int t2 = tid;
        asm volatile("" : "+v"(t2));   // (made anew, as in products)
        sx.begin(a.T + m0 * a.P * a.R, (long)a.P * a.R, a.R, t2, [&](int r) { return ids[r] == g; });
        sw.begin(a.B + ((long)g * a.N + n0) * a.R, a.R, a.R, t2, [&](int r) { return r < nlive; });
      }
    }
    --left;
    sx.fetch(lds + st * STAGE, wave);
    sw.fetch(lds + st * STAGE + BM * 128, wave);
  };
  // the first copies leave before the row -> adapter loads come back, where the projection's own columns are enough for them
  const bool early = nk >= NSTG - 1;
  if (early) {
#pragma unroll
    for (int u = 0; u < NSTG - 1; ++u) issue(u);
  }
  if (a.rows.id != nullptr) {
    for (int r = tid; r < BM; r += NW * 64) ids[r] = r < mlive ? id_of(a.rows, m0 + r) : -1;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  if (!early) {
#pragma unroll
    for (int u = 0; u < NSTG - 1; ++u) issue(u);
  }
  Ring<BM, BN, NW, NSTG> ring{lds};
  if constexpr (MEETS == ANY) {
    for (int t = 0; t < nk; ++t) products<BM, BN, WGM, WGN, true>(ring.turn(issue), wave, lane, acc);
    if (a.rows.id != nullptr) {
      for (int h = next_adapter<BM>(ids, -1, lane); h >= 0; h = next_adapter<BM>(ids, h, lane)) {
        uint32_t own = 0;
#pragma unroll
        for (int i = 0; i < FM; ++i) own |= (uint32_t)(ids[(wave / WGN) * WM + i * 16 + i16] == h) << i;
        for (int t = 0; t < rk; ++t) products<BM, BN, WGM, WGN, true, true>(ring.turn(issue), wave, lane, acc, own);
      }
    }
  } else {
    const int h = a.rows.id != nullptr ? next_adapter<BM>(ids, -1, lane) : -1;
    if (MEETS == FIND && h >= 0 && !one_adapter<BM>(ids, h, mlive, lane)) {
      ring.drain();
      return false;
    }
    const int n = nk + (h < 0 ? 0 : rk);
    for (int t = 0; t < n; ++t) products<BM, BN, WGM, WGN, true>(ring.turn(issue), wave, lane, acc);
  }
  ring.drain();
  int l2 = lane;
  asm volatile("" : "+v"(l2));   // (what the stores need is made anew: kept over the loops it would spill)
  const int i2 = l2 & 15, q2 = l2 >> 4;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const long m = w0 + i * 16 + i2;
    if (m >= a.M) continue;
#pragma unroll
    for (int p = 0; p < FP; ++p) {
      const int n = v0 + p * 32 + q2 * 8;
      if (n >= a.N) continue;
      const f32x4_t v = acc[i][2 * p], w = acc[i][2 * p + 1];
      *reinterpret_cast<uint4*>(a.Y + m * a.ldy + n) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3]));
    }
    if constexpr (FO) {
      const int n = v0 + FP * 32 + q2 * 4;
      if (n >= a.N) continue;
      const f32x4_t v = acc[i][FN - 1];
      *reinterpret_cast<uint2*>(a.Y + m * a.ldy + n) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
  }
  return true;
}

template <int BM, int BN, int WGM, int WGN, int NSTG, Meets MEETS = ANY>
__global__ __launch_bounds__(WGM * WGN * 64, 2) void tile_kernel(const LinArgs a) {
  // ONE shared array: with a second one the compiler tells the two apart, takes the fragment reads for readers of the copies in flight, and waits
  // for all of them (s_waitcnt vmcnt(0)) in every step
  __shared__ __attribute__((aligned(16))) char lds[NSTG * (BM + BN) * 128 + BM * 4];
  const uint32_t tiles_n = (a.N + BN - 1) / BN, tile = xcd_tile(blockIdx.x, gridDim.x);
  const long m0 = (long)(tile / tiles_n) * BM;
  const int n0 = (int)(tile % tiles_n) * BN;
  const bool done = tile_body<BM, BN, WGM, WGN, NSTG, MEETS>(a, lds, m0, n0);
  if constexpr (MEETS == FIND) {   // the selects of ANY need registers that this tile does not have: in two halves
    for (int half = 0; half < 2 && !done; ++half) {
      __syncthreads();
      if (m0 + half * (BM / 2) < a.M) tile_body<BM / 2, BN, WGM, WGN, NSTG, ANY>(a, lds, m0 + half * (BM / 2), n0);
    }
  }
}

// a tile's sums -> T, the rows of adapter g.  mr0, r0: the wavefront's first row in the tile, its first column
template <int FM, int FN>
__device__ __forceinline__ void store_tile(const DownArgs& a, const f32x4_t (&acc)[FM][FN], const int* ids, int g, float sc, int rank, long m0, int mr0, int r0, int lane) {
  const int i16 = lane & 15, q = lane >> 4;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int mr = mr0 + i * 16 + i16;
    bf16_t* row = a.T + (m0 + mr) * a.P * a.R;
    if (ids[mr] != g) continue;
    if constexpr (FN == 1) {
      const int r = r0 + q * 4;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = r + e < rank ? sc * acc[i][0][e] : 0.f;
      if (r < a.R) store_t4(row + r, a.R, a.P, o);
    } else {
#pragma unroll
      for (int j = 0; j < FN; j += 2) {
        const int r = r0 + j * 16 + q * 8;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = r + e < rank ? sc * acc[i][j + e / 4][e % 4] : 0.f;
        if (r < a.R) store_t8(row + r, a.R, a.P, o);
      }
    }
  }
}

// T = s A x for many rows of long requests: 64 rows x BN adapter rows per workgroup, once for each adapter that the rows meet (mostly one).  Bound by reading
// X once per BN adapter rows (32768 x 2560, rank 32: 38.6 us, 4.4 TB/s; 32768 x 320: 5.7 us, 3.7 TB/s)
template <int BN, int NSTG>
__global__ __launch_bounds__(256) void down_tile_kernel(const DownArgs a) {
  constexpr int BM = 64, FM = 2, FN = BN / 32, STAGE = (BM + BN) * 128;
  __shared__ __attribute__((aligned(16))) char lds[NSTG * STAGE + BM * 4];   // (one array: see tile_kernel)
  int* ids = reinterpret_cast<int*>(lds + NSTG * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t tiles_r = (a.R + BN - 1) / BN, tile = xcd_tile(blockIdx.x, gridDim.x);
  const long m0 = (long)(tile / tiles_r) * BM;
  const int r0 = (int)(tile % tiles_r) * BN;
  const int mlive = (int)min((long)BM, a.M - m0), rlive = min(BN, a.R - r0);
  if (tid < BM) ids[tid] = tid < mlive ? id_of(a.rows, m0 + tid) : -1;
  __syncthreads();
  int turn = 0;   // where the rows meet several adapters, blockIdx.y = 0 and 1 take them in turn
  for (int g = next_adapter<BM>(ids, -1, lane); g >= 0; g = next_adapter<BM>(ids, g, lane), ++turn) {
    if ((turn & 1) != (int)blockIdx.y) continue;
    const float sc = a.scales[g];   // (here: behind the product their latency would show)
    const int rank = a.ranks[g];
    f32x4_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    Stage<BM, 4> sx;
    Stage<BN, 4> sa;
    sx.begin(a.X + m0 * a.ldx, a.ldx, a.K, tid, [&](int r) { return r < mlive; });
    sa.begin(a.A + ((long)g * a.R + r0) * a.K, a.K, a.K, tid, [&](int r) { return r < rlive; });
    auto issue = [&](int st) {
      sx.fetch(lds + st * STAGE, wave);
      sa.fetch(lds + st * STAGE + BM * 128, wave);
    };
#pragma unroll
    for (int u = 0; u < NSTG - 1; ++u) issue(u);
    Ring<BM, BN, 4, NSTG> ring{lds};
    for (int t = 0; t < (a.K + BK - 1) / BK; ++t) products<BM, BN, 2, 2, FN % 2 == 0>(ring.turn(issue), wave, lane, acc);
    ring.drain();
    store_tile(a, acc, ids, g, sc, rank, m0, (wave >> 1) * 32, r0 + (wave & 1) * (BN / 2), lane);
    __syncthreads();   // the stages are free for the next adapter
  }
}

// The same from 8-bit codes: a thread turns 16 codes of a row into bf16 on their way into LDS (exact), one stage ahead of the product, with the codes of
// the three stages behind it on their way from memory (9001 x 1280, rank 64: 12.9 us, with one stage 18.6); A comes by copies as above.
template <int BN>
__global__ __launch_bounds__(256) void down8_tile_kernel(const DownArgs a) {
  constexpr int BM = 64, FM = 2, FN = BN / 32, NSTG = 4, STAGE = (BM + BN) * 128;
  __shared__ __attribute__((aligned(16))) char lds[NSTG * STAGE + BM * 4];   // (one array: see tile_kernel)
  int* ids = reinterpret_cast<int*>(lds + NSTG * STAGE);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i16 = lane & 15, q = lane >> 4;
  const uint32_t tiles_r = (a.R + BN - 1) / BN, tile = xcd_tile(blockIdx.x, gridDim.x);
  const long m0 = (long)(tile / tiles_r) * BM;
  const int r0 = (int)(tile % tiles_r) * BN;
  const int mlive = (int)min((long)BM, a.M - m0), rlive = min(BN, a.R - r0);
  if (tid < BM) ids[tid] = tid < mlive ? id_of(a.rows, m0 + tid) : -1;
  __syncthreads();
  const int nb = (a.K + 31) / 32, nk = (a.K + BK - 1) / BK;   // blocks of a row, stages
  const int xr = tid >> 2, xc = (tid & 3) * 16;               // this thread's row, and its 16 columns of a stage
  const uint8_t* cr = a.codes + (m0 + min(xr, mlive - 1)) * (long)nb * 32;
  const uint8_t* er = a.exps + (m0 + min(xr, mlive - 1)) * (long)nb;
  int turn = 0;
  for (int g = next_adapter<BM>(ids, -1, lane); g >= 0; g = next_adapter<BM>(ids, g, lane), ++turn) {
    if ((turn & 1) != (int)blockIdx.y) continue;
    const float sc = a.scales[g];   // (here: behind the product their latency would show)
    const int rank = a.ranks[g];
    f32x4_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    Stage<BN, 4> sa;
    sa.begin(a.A + ((long)g * a.R + r0) * a.K, a.K, a.K, tid, [&](int r) { return r < rlive; });
    uint4 code[NSTG];          // of stage t at t % 4, like the LDS stages
    uint32_t ex[NSTG];
    // (the fences keep copies and loads in this order: the wait below counts them)
    auto load = [&](int t, int u) {   // past the row's last block: the first again
      const int k = t * BK + xc, kk = k < nb * 32 ? k : 0;
      code[u] = *reinterpret_cast<const uint4*>(cr + kk);
      ex[u] = er[kk >> 5];
      asm volatile("" ::: "memory");
    };
    auto fetch = [&](int u) {
      sa.fetch(lds + u * STAGE + BM * 128, wave);
      asm volatile("" ::: "memory");
    };
    auto put = [&](int t, int u) {
      // (the values are first used here, not ahead of the barriers, where the compiler would wait for all of them together)
      asm volatile("" : "+v"(code[u].x), "+v"(code[u].y), "+v"(code[u].z), "+v"(code[u].w), "+v"(ex[u]));
      // past the last block A is zero: any finite step (chosen here: with the load it would wait for it)
      const float sp = act8::step(t * BK + xc < nb * 32 ? ex[u] : 1u);
      float v[8];
      act8::values4(code[u].x, sp, v);
      act8::values4(code[u].y, sp, v + 4);
      *reinterpret_cast<bf16x8_t*>(lds + u * STAGE + lds_off(xr, xc >> 3)) = pack8(v);
      act8::values4(code[u].z, sp, v);
      act8::values4(code[u].w, sp, v + 4);
      *reinterpret_cast<bf16x8_t*>(lds + u * STAGE + lds_off(xr, (xc >> 3) + 1)) = pack8(v);
    };
    load(0, 0);
#pragma unroll
    for (int u = 0; u < NSTG - 1; ++u) {
      fetch(u);
      load(u + 1, u + 1);
    }
    put(0, 0);
    auto stage = [&](int t, int u) {   // u = t % 4
      // still in flight: the copies of two stages and three stages' codes (two loads each).  Stage t's codes are in LDS when everybody's writes are done
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * (BN / 32) + 6) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      put(t + 1, (u + 1) % NSTG);
      fetch((u + 3) % NSTG);
      load(t + 4, u);
      const char *pa = lds + u * STAGE, *pb = pa + BM * 128;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        bf16x8_t fa[FM], fb[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[j] = *reinterpret_cast<const bf16x8_t*>(pb + lds_off((wave & 1) * (BN / 2) + pair_row<FN>(j, i16), ks * 4 + q));
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[i] = *reinterpret_cast<const bf16x8_t*>(pa + lds_off((wave >> 1) * 32 + i * 16 + i16, ks * 4 + q));
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mfma(fb[j], fa[i], acc[i][j]);
      }
    };
    int t = 0;
    for (; t + NSTG <= nk; t += NSTG) {   // (whole turns without a branch inside: at a branch the compiler waits for all loads)
#pragma unroll
      for (int u = 0; u < NSTG; ++u) stage(t + u, u);
    }
#pragma unroll
    for (int u = 0; u < NSTG - 1; ++u)
      if (t + u < nk) stage(t + u, u);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    store_tile(a, acc, ids, g, sc, rank, m0, (wave >> 1) * 32, r0 + (wave & 1) * (BN / 2), lane);
    __syncthreads();   // the stages are free for the next adapter
  }
}

// ------------------------------------------------------------------------------------------------------------------ weight gradients
// The rows of all adapters in sorted order (adapter by adapter) are one axis of `rows` positions, cut into chunks of `chunk` positions.  A workgroup
// takes one chunk x 128 columns of V x RB columns of U; where adapters change inside its chunk it finishes one and begins the next.  Piece
// (chunk b, j-th used adapter) is partial sum b + j: along the axis every new piece raises b or j.  A second launch adds an adapter's partial
// sums in their order: no atomics, the same bits every time.  Bound by the latency of a tile's loads and LDS reads (4096 x 640 and 640, rank 320: 22.0 us, 460
// TFLOP/s, and 5.2 for the sums).
struct Order {
  const int* perm;       // [rows / unit] the unit of rows at each position of the axis, in units
  const int* used_pos;   // [nused + 1] first position of the j-th used adapter, in units
  const int* slot;       // [nslot] j of adapter g, or -1
  int nused, nslot, unit;
  uint32_t magic, shift; // p / unit = (2 p magic) >> 32 >> shift for p < 2^31
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

struct Grad {            // one gradient: dA (U = dT, V = X or its codes) or dB (U = T, V = dY)
  const bf16_t *U, *V;
  const uint8_t *codes, *exps;
  long ldv;
  int C, chunk, blocks;  // columns of V, positions per chunk, workgroups
  float *part, *out;     // partial sums, result
};

// One workgroup's share of one gradient.  The next tile is on its way from memory (registers) while a tile is multiplied; the rest
// of the latency is hidden by the other workgroups of the CU (three: the registers allow no more; with two tiles on their way one fits, 41 against 25 us).
template <int RB, bool CODES, bool TRANS>   // TRANS: partial sums as [C][R] (dB), else [R][C] (dA)
__device__ __forceinline__ void wgrad_body(const Grad& G, int R, const Order& o, uint32_t id, char* vt, char* ut) {
  constexpr int TK = 64, CB = 128, PV = 256, PU = RB == 32 ? 256 : 512;
  constexpr int WU = RB / 32, WV = 4 / WU, FV = CB / WV / 16, FU = 2;   // wavefronts WV x WU, FV x FU fragments each (fewer LDS reads than 4 x 1)
  constexpr int NV = TK * CB / 8 / 256, NU = TK * RB / 8 / 256;   // 16-byte chunks of V, and of each part of U, per thread
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int C = G.C, tc = (C + CB - 1) / CB, tr = (R + RB - 1) / RB;
  const uint32_t ck = id / (tc * tr), rest = id - ck * (tc * tr);   // neighbours share rows
  const int c0 = (int)(rest % tc) * CB, r0 = (int)(rest / tc) * RB;
  const long p_begin = (long)ck * G.chunk, p_end = min(p_begin + G.chunk, o.rows);
  int j = 0;   // the used adapter that holds p_begin
  for (int hi = o.nused; hi - j > 1;) {
    const int mid = (j + hi) >> 1;
    if ((long)o.used_pos[mid] * o.unit <= p_begin) j = mid;
    else hi = mid;
  }
  const int wv0 = wave / WU * (CB / WV), wu0 = wave % WU * 32;
  const int cp = (C + 31) / 32 * 32;
  const int vrow = tid >> 4, vch = tid & 15, vc = c0 + vch * 8;
  const int urow = tid / (RB / 8), uch = tid % (RB / 8), ur = r0 + uch * 8;
  struct Tile {
    uint4 v[NV], u[NU][3];
    uint2 c[NV];
    uint32_t e[NV];
  } next;
  int mv[NV], mu[NU], qv[NV], qu[NU];   // the tile to fetch next: unit of each row, and the row in it (nothing uses a load before the fetch)
  auto unit_of = [&](long p, int& m, int& q) {
    const uint32_t u = __umulhi((uint32_t)p << 1, o.magic) >> o.shift;
    m = o.perm[u];
    q = (int)((uint32_t)p - u * (uint32_t)o.unit);
  };
  auto rows_of = [&](long p, long end) {
#pragma unroll
    for (int l = 0; l < NV; ++l) unit_of(min(p + vrow + 16 * l, end - 1), mv[l], qv[l]);   // (dead rows: the piece's last)
#pragma unroll
    for (int l = 0; l < NU; ++l) unit_of(min(p + urow + (2048 / RB) * l, end - 1), mu[l], qu[l]);
  };
  const int vcl = vc < C ? vc : 0, url = ur < R ? ur : 0;   // (columns past the end: loaded from column 0, never stored)
  auto fetch = [&](Tile& t) {
#pragma unroll
    for (int l = 0; l < NV; ++l) {
      const uint32_t row = mv[l] * o.unit + qv[l];
      if constexpr (CODES) {
        t.c[l] = *reinterpret_cast<const uint2*>(G.codes + (uint64_t)row * (uint32_t)cp + vcl);
        t.e[l] = G.exps[(uint64_t)row * (uint32_t)(cp >> 5) + (vcl >> 5)];
      } else {
        t.v[l] = *reinterpret_cast<const uint4*>(G.V + (uint64_t)row * (uint32_t)G.ldv + vcl);
      }
    }
#pragma unroll
    for (int l = 0; l < NU; ++l) {
      const bf16_t* q = G.U + (uint64_t)(uint32_t)(mu[l] * o.unit + qu[l]) * (uint32_t)(3 * R) + url;
#pragma unroll
      for (int h = 0; h < 3; ++h) t.u[l][h] = *reinterpret_cast<const uint4*>(q + h * R);
    }
  };
  for (long p = p_begin; p < p_end; ++j) {
    const long piece_end = min(p_end, (long)o.used_pos[j + 1] * o.unit);
    f32x4_t acc[FV][FU];
#pragma unroll
    for (int v = 0; v < FV; ++v)
#pragma unroll
      for (int u = 0; u < FU; ++u) acc[v][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    rows_of(p, piece_end);
    fetch(next);
    rows_of(p + TK, piece_end);
    for (; p < piece_end; p += TK) {
      const Tile& t = next;
      __syncthreads();   // the last tile's fragments have been read
#pragma unroll
      for (int l = 0; l < NV; ++l) {
        uint4 w;
        if constexpr (CODES) {
          float v[8];
          act8::values4(t.c[l].x, act8::step(t.e[l]), v);
          act8::values4(t.c[l].y, act8::step(t.e[l]), v + 4);
          w = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        } else {
          w = t.v[l];
        }
        *reinterpret_cast<uint4*>(vt + tr_off<PV>(vrow + 16 * l, vch)) = keep(w, p + vrow + 16 * l < piece_end);
      }
#pragma unroll
      for (int l = 0; l < NU; ++l)
#pragma unroll
        for (int h = 0; h < 3; ++h)
          *reinterpret_cast<uint4*>(ut + tr_off<PU>(urow + (2048 / RB) * l, h * (RB / 8) + uch)) = keep(t.u[l][h], p + urow + (2048 / RB) * l < piece_end);
      __syncthreads();
      fetch(next);   // the next tile's loads run under this tile's products (past the piece: its last row again)
      rows_of(p + 2 * TK, piece_end);
#pragma unroll
      for (int s = 0; s < TK / 32; ++s) {
        bf16x8_t fv[FV];
#pragma unroll
        for (int v = 0; v < FV; ++v) fv[v] = tr_frag<PV>(vt, s, wv0 + v * 16, lane);
#pragma unroll
        for (int h = 2; h >= 0; --h)
#pragma unroll
          for (int u = 0; u < FU; ++u) {   // (all of U's fragments of a step read ahead spill registers: 30 against 25 us)
            const bf16x8_t fu = tr_frag<PU>(ut, s, h * RB + wu0 + u * 16, lane);
#pragma unroll
            for (int v = 0; v < FV; ++v) acc[v][u] = TRANS ? mfma(fu, fv[v], acc[v][u]) : mfma(fv[v], fu, acc[v][u]);
          }
      }
    }
    p = piece_end;
    float* out = G.part + (long)(ck + j) * R * C;
#pragma unroll
    for (int v = 0; v < FV; ++v)
#pragma unroll
      for (int u = 0; u < FU; ++u) {
        const int cb = c0 + wv0 + v * 16, rb = r0 + wu0 + u * 16, a = (lane >> 4) * 4, b = lane & 15;
        if (TRANS) {   // lane: column b of V, columns a .. a + 3 of U
          if (cb + b < C && rb + a < R) *reinterpret_cast<f32x4_t*>(out + (long)(cb + b) * R + rb + a) = acc[v][u];
        } else {       // lane: column b of U, columns a .. a + 3 of V
          if (rb + b < R && cb + a < C) *reinterpret_cast<f32x4_t*>(out + (long)(rb + b) * C + cb + a) = acc[v][u];
        }
      }
  }
}

// dA and dB in one launch: the first da.blocks workgroups work on dA, the others on dB
template <int RB, bool CODES>
__global__ __launch_bounds__(256, 3) void wgrad_kernel(const Grad da, const Grad db, int R, const Order o) {
  __shared__ __attribute__((aligned(16))) char vt[64 * 256], ut[64 * (RB == 32 ? 256 : 512)];
  const uint32_t id = xcd_tile(blockIdx.x, gridDim.x);
  if (id < (uint32_t)da.blocks) wgrad_body<RB, CODES, false>(da, R, o, id, vt, ut);
  else wgrad_body<RB, false, true>(db, R, o, id - da.blocks, vt, ut);
}

// out[g] = sum of the partial sums of adapter g; zeros for an adapter without rows and past an adapter's rank.  VEC outputs per thread
template <bool TRANS, int VEC>
__device__ __forceinline__ void wgrad_sum(const Grad& G, int R, int r_out, const int* ranks, const Order& o, uint32_t block) {
  typedef float vec_t __attribute__((ext_vector_type(VEC)));
  const int g = blockIdx.y, C = G.C;
  const uint32_t id = (block * 256u + threadIdx.x) * VEC, n = (uint32_t)r_out * (uint32_t)C;
  if (id >= n) return;
  const int w = TRANS ? r_out : C;                       // VEC divides a row of the output
  const uint32_t row = id / w, col = id - row * w;
  const int r = (int)(TRANS ? col : row);
  const uint32_t at = TRANS ? row * R + col : id;
  const int j = g < o.nslot ? o.slot[g] : -1;
  vec_t s = 0.f;
  if (j >= 0) {
    const long first = (long)o.used_pos[j] * o.unit, last = (long)o.used_pos[j + 1] * o.unit - 1;
    const float* q = G.part + (first / G.chunk + j) * R * C + at;
    const int nb = (int)(last / G.chunk - first / G.chunk) + 1;
#pragma unroll 8
    for (int b = 0; b < nb; ++b) s += *reinterpret_cast<const vec_t*>(q + (long)b * R * C);
    const int rank = ranks[g];
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (r + (TRANS ? e : 0) >= rank) s[e] = 0.f;
  }
  *reinterpret_cast<vec_t*>(G.out + (long)g * n + id) = s;
}

template <int VEC>   // of dB; dA's rows are a multiple of 8 long
__global__ __launch_bounds__(256) void wgrad_reduce_kernel(const Grad da, const Grad db, int R, int r_out, const int* __restrict__ ranks, const Order o, int blocks_a) {
  if ((int)blockIdx.x < blocks_a) wgrad_sum<false, 4>(da, R, r_out, ranks, o, blockIdx.x);
  else wgrad_sum<true, VEC>(db, R, r_out, ranks, o, blockIdx.x - blocks_a);
}

// positions per chunk, of both gradients (K, N: 0 for one that is not asked for): whole tiles of 64, at most 512 workgroups, two for each CU (4096 x 640,
// rank 320, with the sum: 27.6 us; 576: 30.4, 768: 29.0, 384: 31.6)
int wgrad_chunk(long rows, int K, int N, int R) {
  const long tiles = (long)((K + 127) / 128 + (N + 127) / 128) * (R <= 32 ? 1 : (R + 63) / 64);
  const long want = tiles < 512 ? 512 / tiles : 1;
  const long ch = ((rows + want - 1) / want + 63) / 64 * 64;
  return (int)(ch < 64 ? 64 : ch > (1 << 20) ? (1 << 20) : ch);
}

// partial sums of one gradient with C columns, in floats
double wgrad_floats(long rows, int nused, int C, int R, int chunk) {
  if (rows <= 0 || nused <= 0 || C <= 0 || R <= 0) return 0;
  return (double)((rows + chunk - 1) / chunk + nused - 1) * R * C;
}

// T by 64-row tiles where a tile rarely meets a second adapter (each costs another pass over its rows) and the tiles fill the chip or 16-row tiles are more
// than one for each CU, by 16-row tiles otherwise.  Measured (us, 64-row / 16-row tiles): 32768 x 320, rank 32: 5.3 / 9.8; 9001 x 1280, rank 64: 10.0 /
// 19.9; 4096 x 640, rank 320: 7.6 / 17.6; 4096 x 1280, rank 32 (64 tiles): 6.9 / 6.0; 1001 x 768, rank 64 (16 tiles): 6.7 / 6.3; 1000 x 2560, rank 32 (16
// tiles): 10.7 / 9.0; with the second launch 4678 x 1896, rank 64 (74 tiles, 293 16-row workgroups): 21.1 / 32.6; 1000 x 640, rank 320 (80, 315): 10.9 / 16.6.
void launch_down(const DownArgs& a, int runs, int slots, hipStream_t st) {
  const long tiles = (a.M + 63) / 64 * (a.R <= 32 ? 1 : (a.R + 63) / 64);
  const int t16 = (a.R + 15) / 16;
  // few workgroups: fewer adapter rows each, so that more CUs share the loads (8 x 1280, rank 32: 3.8 us with 16 rows, 5.0 with 32; 64 x 1280, rank 64:
  // 4.3 / 5.5 / 8.0 with 16 / 32 / 64); many: more, so that X is read less often (9001 x 1280 codes, rank 64: 30 / 23 / 20)
  const long b16 = (a.M + 15) / 16 * t16;
  const int rt = t16 == 1 || b16 <= 256 ? 1 : t16 == 2 || b16 <= 512 ? 2 : 4;
  if (a.M / runs >= 64 && (tiles >= 96 || (a.M + 15) / 16 * ((t16 + rt - 1) / rt) > 256)) {
    const dim3 grid((unsigned)tiles, a.rows.unit % 64 ? 2 : 1);   // whole tiles of one adapter need no second workgroup
    if (a.codes && a.R <= 32) hipLaunchKernelGGL((down8_tile_kernel<32>), grid, dim3(256), 0, st, a);
    else if (a.codes) hipLaunchKernelGGL((down8_tile_kernel<64>), grid, dim3(256), 0, st, a);
    else if (a.R <= 32) hipLaunchKernelGGL((down_tile_kernel<32, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((down_tile_kernel<64, 4>), grid, dim3(256), 0, st, a);
    return;
  }
  const dim3 grid((unsigned)((a.M + 15) / 16), slots, (t16 + rt - 1) / rt);
#define AQL_DOWN(RT)                                                                          \
  do {                                                                                        \
    if (a.codes) hipLaunchKernelGGL((down_kernel<RT, 4, true>), grid, dim3(256), 0, st, a);   \
    else hipLaunchKernelGGL((down_kernel<RT, 4, false>), grid, dim3(256), 0, st, a);          \
  } while (0)
  if (rt == 1) AQL_DOWN(1);
  else if (rt == 2) AQL_DOWN(2);
  else AQL_DOWN(4);
#undef AQL_DOWN
}

bool rows_ok(const void* id, int runs, int unit) { return runs >= 0 && (runs == 0 || (id && unit >= 1)); }

}  // namespace

// Y = X W^T + bias + residual + the low-rank term; T: [M][parts][R] bf16, written for the rows that have an adapter.  slots: at least the number of adapters that
// any 16 rows [16 i, 16 i + 16) meet; runs: stretches of neighbouring rows with one adapter; used: adapters that have rows (these two decide between forms only).
extern "C" int aql_adapter_linear(const bf16_t* X, long ldx, const bf16_t* W, long ldw, const bf16_t* bias, const bf16_t* residual, long ldr, bf16_t* Y,
                                  long ldy, long M, int N, int K, const bf16_t* A, const bf16_t* B, const int* ranks, const float* scales, int R,
                                  const int* unit_id, int unit, int runs, int slots, int used, bf16_t* T, int parts, hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && M < (1L << 31) - 256 && N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0, "aql_adapter_linear: bad shape M=%ld N=%d K=%d (N, K: multiples of 8)", M, N, K);
  if (M == 0) return AQL_OK;
  AQL_CHECK_ARG(X && W && Y, "aql_adapter_linear: null operand");
  AQL_CHECK_ARG(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N) && ldx % 8 == 0 && ldw % 8 == 0 && ldy % 8 == 0 && ldr % 8 == 0 && ldx < (1L << 21) &&
                    ldw < (1L << 21), "aql_adapter_linear: leading dimensions (multiples of 8, at least the width, below 2^21)");
  AQL_CHECK_ARG((((uintptr_t)X | (uintptr_t)W | (uintptr_t)bias | (uintptr_t)residual | (uintptr_t)Y) & 15) == 0, "aql_adapter_linear: operands must be 16-byte aligned");
  AQL_CHECK_ARG(rows_ok(unit_id, runs, unit) && (runs == 0 || (A && B && ranks && scales && T && R > 0 && R <= MAX_R && R % 8 == 0 && slots >= 1 && slots <= 16 && (parts == 1 || parts == 3))),
                "aql_adapter_linear: bad adapters (R=%d: a multiple of 8, at most %d) or rows", R, MAX_R);
  const Rows rows{runs ? unit_id : nullptr, unit};
  if (runs) {
    launch_down(DownArgs{X, nullptr, nullptr, A, ranks, scales, T, ldx, M, K, R, parts, rows}, runs, slots, stream);
    AQL_CHECK_LAUNCH("aql_adapter_linear (down)");
  }
  const LinArgs a{X, W, bias, residual, B, Y, T, ldx, ldw, ldr, ldy, M, N, K, R, parts, rows};
  // Sixteen rows at a time, or tiles of 64 rows and more: by the number of 16 x 16 outputs, and by the adapters that 64 rows meet, each of which costs a
  // tile another turn of its ring per 64 columns of rank.  Both launches of a call together, us, 16 rows / 64 x 64 tiles, rank 32, four requests and
  // single rows of eight adapters: 256 x 1280 x 1280 (1280 outputs): 16.4 / 13.1 and 20.8 / 20.9; 128 x 1280 x 1280 (640): 13.2 / 13.8 and 14.9 / 18.7;
  // 64 x 10240 x 1280 (2560): 24.6 / 16.2 and 27.0 / 20.0
  const long outs = ((M + 15) / 16) * ((N + 15) / 16);
  const long met = runs ? (64L * runs / M + 1 < used ? 64L * runs / M + 1 : used) : 0;
  if (outs < 960 + 32 * met * ((R + BK - 1) / BK)) {
    const unsigned my = (unsigned)((M + 15) / 16);
    // two fragments of columns per wavefront where one each gives more workgroups than CUs (64 x 1280 x 1280: 9.9 us, with one 10.8; 8 x 1280 x 1280: 10.5 / 9.0)
    if (outs > 256) hipLaunchKernelGGL((skinny_kernel<2>), dim3((N + 31) / 32, my), dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((skinny_kernel<1>), dim3((N + 15) / 16, my), dim3(512), 0, stream, a);
  } else {
#define AQL_TILE(BM, BN, WGM, WGN, ...) \
  hipLaunchKernelGGL((tile_kernel<BM, BN, WGM, WGN, __VA_ARGS__>), dim3((unsigned)(((M + BM - 1) / BM) * ((N + BN - 1) / BN))), dim3(WGM * WGN * 64), 0, stream, a)
    // Which tile (us without adapters, all tiles measured at each size): 256 x 320 where the width allows it and every CU gets one (4096 x 10240 x
    // 1280: 99, 256 x 192 116, 128 x 320 142, 128 x 128 145).  Where 128 x 128 still gives every CU one: the least of rounds x time per round -- one
    // 256 x 192 per CU, 29.5 us at K = 1280; one 128 x 320 (where that divides the width) or two 128 x 160, 29.2, a single 128 x 160, 19.8; two 128 x 128,
    // 28.2, one 14.1 (9001 x 1280 x 1280 with 256 x 192, 128 x 320, 128 x 128: 31.9, 50, 37.1; 16384 x 640 x 640: 19.4, 18.6, 21.0; 20480 x 640 x 640: 31.9,
    // 31.2, 25.0; 32768 x 320 x 320 with 128 x 160: 16.1, 128 x 320: 13.0; 4096 x 1280 x 1280 with 128 x 160: 19.8, 128 x 128: 21.5).  Smaller ones where
    // those leave CUs idle (2048 x 1280 x 1280: 13.2 with 64 x 128, 14.8 with 128 x 128; 1001 x 640 x 768: 6.0 with 64 x 64, 6.6 with 64 x 128; both
    // launches of 300 x 1280 x 5120: 31.3 with 64 x 32, 37.5 with 64 x 64).  256 x 320 with requests of whole 256-row tiles: no tile meets two
    // adapters, and the kernel need not find out (109 / 115 with rank 32).
    const auto tiles = [&](long bm, long bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
    const long t192 = (tiles(256, 192) + 255) / 256 * 295, t160 = tiles(128, 160) <= 256 ? 198 : (tiles(128, 160) + 511) / 512 * 292;
    const long t128 = (tiles(128, 128) + 255) / 256 * 141;
    const bool wide = N % 320 == 0 && 320 * ldw * 2 <= SPAN;   // (320 rows of W under one descriptor)
    if (wide && tiles(256, 320) >= 256 && (runs == 0 || unit % 256 == 0)) AQL_TILE(256, 320, 2, 4, 2, ONE);
    else if (wide && tiles(256, 320) >= 256) AQL_TILE(256, 320, 2, 4, 2, FIND);
    else if (tiles(128, 128) >= 256) {
      if (t128 <= t160 && t128 <= t192) AQL_TILE(128, 128, 2, 4, 2);
      else if (t192 < t160) AQL_TILE(256, 192, 4, 2, 2);
      else if (wide && tiles(128, 160) > 256) AQL_TILE(128, 320, 2, 4, 2);
      else AQL_TILE(128, 160, 2, 2, 2);
    }
    else if (tiles(64, 128) >= 256) AQL_TILE(64, 128, 2, 4, 3);
    else if (tiles(64, 64) > 128) AQL_TILE(64, 64, 2, 2, 3);
    else AQL_TILE(64, 32, 4, 1, 4);
#undef AQL_TILE
  }
  AQL_CHECK_LAUNCH("aql_adapter_linear");
  return AQL_OK;
}

// T = s A x alone, from X or from its 8-bit codes
extern "C" int aql_adapter_down(const bf16_t* X, long ldx, const uint8_t* codes, const uint8_t* exps, long M, int K, const bf16_t* A, const int* ranks,
                                const float* scales, int R, const int* unit_id, int unit, int runs, int slots, bf16_t* T, int parts,
                                hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && M < (1L << 31) - 256 && K > 0 && K % 8 == 0 && K < (1 << 21) && R > 0 && R <= MAX_R && R % 8 == 0, "aql_adapter_down: bad shape M=%ld K=%d R=%d", M, K, R);
  AQL_CHECK_ARG(rows_ok(unit_id, runs, unit), "aql_adapter_down: bad rows");
  if (M == 0 || runs == 0) return AQL_OK;
  AQL_CHECK_ARG(!codes == !exps && !X != !codes && (!X || (ldx >= K && ldx % 8 == 0 && ldx < (1L << 21) && ((uintptr_t)X & 15) == 0)) && A && ranks && scales && T && slots >= 1 && slots <= 16 && (parts == 1 || parts == 3),
                "aql_adapter_down: bad operands (exactly one of X and its codes)");
  launch_down(DownArgs{X, codes, exps, A, ranks, scales, T, ldx, M, K, R, parts, Rows{unit_id, unit}}, runs, slots, stream);
  AQL_CHECK_LAUNCH("aql_adapter_down");
  return AQL_OK;
}

// fp32 elements of the workspace of aql_adapter_wgrad (rows: those that have an adapter; nused: adapters that have rows; K, N: 0 for a gradient that is
// not asked for), or -1: more than 2^31 - 1
extern "C" int aql_adapter_wgrad_scratch_floats(long rows, int nused, int K, int N, int R) {
  if (K < 0) K = 0;
  if (N < 0) N = 0;
  if (K + N == 0) return 0;
  const int ch = wgrad_chunk(rows, K, N, R);
  const double n = wgrad_floats(rows, nused, K, R, ch) + wgrad_floats(rows, nused, N, R, ch);
  return n < 2147483647.0 ? (int)n : -1;
}

extern "C" int aql_adapter_wgrad(const bf16_t* dT, const bf16_t* X, long ldx, const uint8_t* codes, const uint8_t* exps, int K, float* dA, const bf16_t* T,
                                 const bf16_t* dY, long lddy, int N, float* dB, long M, int G, int R, int r_out, const int* ranks, const int* perm,
                                 const int* used_pos, const int* slot, int nused, int nslot, int unit, long rows, float* scratch, long scratch_floats,
                                 hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && M < (1L << 31) - 256 && R > 0 && R % 8 == 0 && G > 0 && G <= 65535 && r_out > 0 && r_out <= R && rows >= 0 && rows <= M,
                "aql_adapter_wgrad: bad shape M=%ld R=%d G=%d", M, R, G);
  AQL_CHECK_ARG((dA || dB) && ranks, "aql_adapter_wgrad: null operand");
  AQL_CHECK_ARG(!dA || (K > 0 && K % 8 == 0 && (long)R * K < (1L << 31) && !codes == !exps && !X != !codes && (!X || (ldx >= K && ldx % 8 == 0 && ldx < (1L << 31) && ((uintptr_t)X & 15) == 0))),
                "aql_adapter_wgrad: bad operands of dA (exactly one of X and its codes)");
  AQL_CHECK_ARG(!dB || (N > 0 && N % 8 == 0 && (long)R * N < (1L << 31) && dY && lddy >= N && lddy % 8 == 0 && lddy < (1L << 31) && ((uintptr_t)dY & 15) == 0), "aql_adapter_wgrad: bad operands of dB");
  AQL_CHECK_ARG(rows == 0 || ((!dA || dT) && (!dB || T) && perm && used_pos && slot && nused > 0 && nslot > 0 && unit >= 1 && rows % unit == 0), "aql_adapter_wgrad: bad rows");
  if (!dA) K = 0;
  if (!dB) N = 0;
  const int need = aql_adapter_wgrad_scratch_floats(rows, nused, K, N, R);
  AQL_CHECK_ARG(need >= 0 && scratch_floats >= need && (need == 0 || scratch), "aql_adapter_wgrad: workspace of %ld floats, %d needed", scratch_floats, need);
  uint32_t L = 0;   // 2^L >= unit: magic = floor(2^(31 + L) / unit) + 1 < 2^32, and the quotient is exact below 2^31
  while (rows && (1L << L) < unit) ++L;
  const Order o{perm, used_pos, slot, nused, rows ? nslot : 0, unit, rows ? (uint32_t)((1UL << (31 + L)) / (uint32_t)unit + 1) : 0u, L, rows};
  const int rb = R <= 32 ? 32 : 64, tr = (R + rb - 1) / rb, chunk = wgrad_chunk(rows, K, N, R);
  const auto job = [&](const bf16_t* U, const bf16_t* V, long ldv, int C, float* part, float* out) {
    Grad g{U, V, nullptr, nullptr, ldv, C, 64, 0, part, out};
    if (C && rows) {
      g.chunk = chunk;
      g.blocks = (int)((rows + g.chunk - 1) / g.chunk) * ((C + 127) / 128) * tr;
    }
    return g;
  };
  Grad a = job(dT, X, ldx, K, scratch, dA);
  a.codes = codes, a.exps = exps;
  const Grad b = job(T, dY, lddy, N, scratch + (long)wgrad_floats(rows, nused, K, R, chunk), dB);
  if (rows) {
    const dim3 grid(a.blocks + b.blocks);
    if (R <= 32) {
      if (codes) hipLaunchKernelGGL((wgrad_kernel<32, true>), grid, dim3(256), 0, stream, a, b, R, o);
      else hipLaunchKernelGGL((wgrad_kernel<32, false>), grid, dim3(256), 0, stream, a, b, R, o);
    } else {
      if (codes) hipLaunchKernelGGL((wgrad_kernel<64, true>), grid, dim3(256), 0, stream, a, b, R, o);
      else hipLaunchKernelGGL((wgrad_kernel<64, false>), grid, dim3(256), 0, stream, a, b, R, o);
    }
    AQL_CHECK_LAUNCH("aql_adapter_wgrad");
  }
  const bool vec = r_out % 4 == 0;
  const int ba = (int)(((long)r_out * K / 4 + 255) / 256), bb = (int)(((long)r_out * N / (vec ? 4 : 1) + 255) / 256);
  if (vec) hipLaunchKernelGGL(wgrad_reduce_kernel<4>, dim3(ba + bb, G), dim3(256), 0, stream, a, b, R, r_out, ranks, o, ba);
  else hipLaunchKernelGGL(wgrad_reduce_kernel<1>, dim3(ba + bb, G), dim3(256), 0, stream, a, b, R, r_out, ranks, o, ba);
  AQL_CHECK_LAUNCH("aql_adapter_wgrad (sum)");
  return AQL_OK;
}
