// Block-scaled fp8: the quantizer of activation rows, and resident weights from row-major codes or f32 values.
#include <algorithm>

#include "fp8.hpp"
#include "kernels.hpp"

// Rows of x in blocks of 128: scale = max(amax / 448, 1e-12), codes x / scale to nearest even. 16 lanes a block, 8 values
// a lane (one or two 16-byte loads), the maximum over the 16 lanes by lane exchanges. Codes past K up to the row's padded
// end are zeros. HBM-bound: 2 bytes in and one out per value of a 16-bit x; 16000 × 4096 values of bf16 on MI355X 40 us, 4.9 TB/s.
namespace {
constexpr int QT = 256;
}
template <int DT>
__global__ __launch_bounds__(QT) void quantize_fp8_kernel(const void *__restrict__ x, int64_t blocks, int k, int kt,
                                                          uint8_t *__restrict__ q, int64_t q_stride, float *__restrict__ scale) {
  const int sub = threadIdx.x & 15;
  const int64_t step = (int64_t)gridDim.x * (QT / 16);
  for (int64_t b = (int64_t)blockIdx.x * (QT / 16) + threadIdx.x / 16; b < blocks; b += step) {
    const int64_t row = (uint32_t)b / (uint32_t)kt;  // (2^32 blocks do not fit the memory)
    const int at = (int)(b - row * kt), col = at * 128 + sub * 8;
    float v[8];
    const bool in = col < k;
    if (in) {
      if constexpr (DT == RK_DTYPE_F32) {
        dt_load_vec<DT, 4>(x, row * k + col, v);
        dt_load_vec<DT, 4>(x, row * k + col + 4, v + 4);
      } else {
        dt_load_vec<DT, 8>(x, row * k + col, v);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[e]));
    const float s = fp8_scale(fp8_max16(amax));
    const Fp8Div div(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = div(v[e]);
    const uintx2 c = {fp8_codes4(v[0], v[1], v[2], v[3]), fp8_codes4(v[4], v[5], v[6], v[7])};
    if (col < q_stride) *(uintx2 *)(q + row * q_stride + col) = c;
    if (sub == 0) scale[b] = s;
  }
}

hipError_t rk_launch_quantize_fp8(const void *x, int dtype, int64_t m, int k, uint8_t *q, int64_t q_stride, float *scale,
                                  hipStream_t st) {
  const int kt = (k + 127) / 128;
  const int64_t blocks = m * kt;
  const unsigned grid = (unsigned)std::min<int64_t>((blocks + 15) / 16, 1 << 16);
  auto kern = dtype == RK_DTYPE_F32 ? quantize_fp8_kernel<RK_DTYPE_F32>
              : dtype == RK_DTYPE_F16 ? quantize_fp8_kernel<RK_DTYPE_F16> : quantize_fp8_kernel<RK_DTYPE_BF16>;
  hipLaunchKernelGGL(kern, dim3(grid), dim3(QT), 0, st, x, blocks, k, kt, q, q_stride, scale);
  return hipGetLastError();
}

// Row-major codes [n, k] into the resident layout (fp8_offset). Row r goes to row (r / 32)·grp_stride + grp_off + r % 32:
// (32, 0) as it is, (64, 0) and (64, 32) the gate and up halves of an expert's first product. A thread per 16 codes.
__global__ __launch_bounds__(256) void fp8_layout_kernel(const uint8_t *__restrict__ codes, int64_t n, int k, int kt, int grp_stride,
                                                         int grp_off, uint8_t *__restrict__ out) {
  const int64_t chunks = k / 16, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * chunks) return;
  const int64_t r = i / chunks, c = i - r * chunks;
  const int64_t to = (r / 32) * grp_stride + grp_off + r % 32;
  *(uintx4 *)(out + fp8_offset(to, c * 16, kt)) = *(const uintx4 *)(codes + r * k + c * 16);
}
hipError_t rk_launch_fp8_layout(const uint8_t *codes, int64_t n, int k, int grp_stride, int grp_off, uint8_t *out, hipStream_t st) {
  const int64_t chunks = n * (k / 16);
  hipLaunchKernelGGL(fp8_layout_kernel, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, st, codes, n, k, (k + 127) / 128,
                     grp_stride, grp_off, out);
  return hipGetLastError();
}

// f32 weights [n, k] to codes in the resident layout and one scale per 128 × 128 block, by the quantizer's rule. A
// workgroup per block, read twice (the second time from the caches): packing is no hot path.
__global__ __launch_bounds__(256) void fp8_pack_kernel(const float *__restrict__ w, int64_t n, int k, int kt, int grp_stride,
                                                       int grp_off, uint8_t *__restrict__ out, float *__restrict__ scale) {
  __shared__ float s_max[4];
  const int64_t r0 = (int64_t)blockIdx.y * 128;
  const int k0 = blockIdx.x * 128;
  const int rows = (int)min<int64_t>(128, n - r0), cols = min(128, k - k0);
  float amax = 0.f;
  for (int i = threadIdx.x; i < rows * cols; i += 256) amax = fmaxf(amax, fabsf(w[(r0 + i / cols) * k + k0 + i % cols]));
  for (int d = 1; d < 64; d *= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = amax;
  __syncthreads();
  const float s = fp8_scale(fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3])));
  if (threadIdx.x == 0) scale[(int64_t)blockIdx.y * kt + blockIdx.x] = s;
  const Fp8Div div(s);
  for (int i = threadIdx.x; i < rows * cols / 4; i += 256) {
    const int r = i * 4 / cols, c = i * 4 % cols;
    const float *p = w + (r0 + r) * k + k0 + c;
    const int64_t row = r0 + r, to = (row / 32) * grp_stride + grp_off + row % 32;
    *(uint32_t *)(out + fp8_offset(to, k0 + c, kt)) = fp8_codes4(div(p[0]), div(p[1]), div(p[2]), div(p[3]));
  }
}
hipError_t rk_launch_fp8_pack(const float *w, int64_t n, int k, int grp_stride, int grp_off, uint8_t *out, float *scale,
                              hipStream_t st) {
  const int kt = (k + 127) / 128;
  hipLaunchKernelGGL(fp8_pack_kernel, dim3(kt, (unsigned)((n + 127) / 128)), dim3(256), 0, st, w, n, k, kt, grp_stride, grp_off,
                     out, scale);
  return hipGetLastError();
}
