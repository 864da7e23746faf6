// 8-bit activation checkpoints (format: aql_act8.cuh): codes int8 [M][Cp], exponent bytes [M][Cp / 32], Cp = C rounded up to 32.
// Both kernels are one pass over the data, bound by HBM: a thread takes 8 columns, a quad of lanes one block of 32 (65536 x 640 bf16: pack 20.8 us,
// unpack 19.8 us, 6.1 and 6.4 TB/s of 127 MB that partly stay in the last-level cache; a copy of 2 GiB runs at 4.9).
#include "aql_act8.cuh"

using namespace act8;

namespace {

// chunk id -> (row, 8-column chunk); ids of one launch stay below 2^31 (the host cuts larger tensors into row ranges)
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ x, long ldx, uint32_t nchunk, uint32_t total, int C,
                                                   uint8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  if (id >= total) return;                       // total % 4 == 0: a quad leaves as one
  const uint32_t row = id / nchunk, c = id - row * nchunk;
  Raw8<T> r;
  float v[8];
  load_raw(x + (long)row * ldx + 8 * c, C - 8 * (int)c, r);
  widen(r, v);
  const uint32_t b = exp_byte(quad_umax(amax_bits8(r)));
  *reinterpret_cast<uint2*>(codes + ((long)row * nchunk + c) * 8) = codes8(v, b);
  if ((c & 3) == 0) exps[(long)row * (nchunk >> 2) + (c >> 2)] = (uint8_t)b;
}

template <class T>
__global__ __launch_bounds__(256) void unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, uint32_t nchunk,
                                                     uint32_t total, int C, T* __restrict__ out, long ldo) {
  const uint32_t id = blockIdx.x * 256u + threadIdx.x;
  if (id >= total) return;
  const uint32_t row = id / nchunk, c = id - row * nchunk;
  const uint2 q = *reinterpret_cast<const uint2*>(codes + ((long)row * nchunk + c) * 8);
  const float st = step(exps[(long)row * (nchunk >> 2) + (c >> 2)]);
  float v[8];
  values4(q.x, st, v);
  values4(q.y, st, v + 4);
  store8(out + (long)row * ldo + 8 * c, C - 8 * (int)c, v);
}

}  // namespace

extern "C" int aql_act8_pack(const void* x, int dtype, long M, int C, long ldx, uint8_t* codes, uint8_t* exps, hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && C > 0 && C <= (1 << 24) && ldx >= C && (dtype == 0 || dtype == 1), "aql_act8_pack: bad shape M=%ld C=%d ldx=%ld dtype=%d", M, C, ldx, dtype);
  if (M == 0) return AQL_OK;
  AQL_CHECK_ARG(x && codes && exps, "aql_act8_pack: null operand");
  const uint32_t nchunk = (uint32_t)((C + 31) / 32) * 4;
  const long per = (1L << 30) / nchunk;
  for (long r0 = 0; r0 < M; r0 += per) {
    const uint32_t total = (uint32_t)((M - r0 < per ? M - r0 : per) * nchunk);
    uint8_t *qc = codes + r0 * nchunk * 8, *qe = exps + r0 * (nchunk / 4);
    if (dtype == 0)
      hipLaunchKernelGGL(pack_kernel<bf16_t>, dim3((total + 255) / 256), dim3(256), 0, stream, (const bf16_t*)x + r0 * ldx, ldx, nchunk, total, C, qc, qe);
    else
      hipLaunchKernelGGL(pack_kernel<float>, dim3((total + 255) / 256), dim3(256), 0, stream, (const float*)x + r0 * ldx, ldx, nchunk, total, C, qc, qe);
    AQL_CHECK_LAUNCH("aql_act8_pack");
  }
  return AQL_OK;
}

extern "C" int aql_act8_unpack(const uint8_t* codes, const uint8_t* exps, long M, int C, void* out, int dtype, long ldo, hipStream_t stream) {
  AQL_CHECK_ARG(M >= 0 && C > 0 && C <= (1 << 24) && ldo >= C && (dtype == 0 || dtype == 1), "aql_act8_unpack: bad shape M=%ld C=%d ldo=%ld dtype=%d", M, C, ldo, dtype);
  if (M == 0) return AQL_OK;
  AQL_CHECK_ARG(out && codes && exps, "aql_act8_unpack: null operand");
  const uint32_t nchunk = (uint32_t)((C + 31) / 32) * 4;
  const long per = (1L << 30) / nchunk;
  for (long r0 = 0; r0 < M; r0 += per) {
    const uint32_t total = (uint32_t)((M - r0 < per ? M - r0 : per) * nchunk);
    const uint8_t *qc = codes + r0 * nchunk * 8, *qe = exps + r0 * (nchunk / 4);
    if (dtype == 0)
      hipLaunchKernelGGL(unpack_kernel<bf16_t>, dim3((total + 255) / 256), dim3(256), 0, stream, qc, qe, nchunk, total, C, (bf16_t*)out + r0 * ldo, ldo);
    else
      hipLaunchKernelGGL(unpack_kernel<float>, dim3((total + 255) / 256), dim3(256), 0, stream, qc, qe, nchunk, total, C, (float*)out + r0 * ldo, ldo);
    AQL_CHECK_LAUNCH("aql_act8_unpack");
  }
  return AQL_OK;
}
