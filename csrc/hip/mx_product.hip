// MXFP4 product and linear layer (format and layout: mx.h).
#include "mx_common.h"

namespace gpumon_hip {
namespace mx {
namespace {

// One wave's 16x16x128 step. Operand fragments: lane l holds row l & 15, block l >> 4 of the quad
// (16 bytes), its scale in byte 0; D: lane l holds columns-of-B row l & 15 and rows-of-A 4 (l >> 4) + i.
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c, unsigned sa, unsigned sb) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// 32 x 32 results a wave, operands straight from memory. b's rows take the instruction's A side, so
// that a lane's four sums are neighbours in a row of c. Rows past the end read the last row instead,
// and their sums are not stored.
template <typename T>
__global__ void __launch_bounds__(256) product_direct_kernel(const u32x4* __restrict__ ac, const unsigned* __restrict__ as,
                                                             const u32x4* __restrict__ bc, const unsigned* __restrict__ bs,
                                                             unsigned m, unsigned n, unsigned quads, T* __restrict__ c,
                                                             int64_t stride, Div tiles_n) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const unsigned tm = tiles_n.quot(blockIdx.x), tn = blockIdx.x - tm * tiles_n.d;
  const unsigned m0 = tm * 64 + (wave & 1) * 32, n0 = tn * 64 + (wave >> 1) * 32;
  unsigned rm[2], rn[2];
  for (int f = 0; f < 2; ++f) rm[f] = min(m0 + f * 16 + r, m - 1), rn[f] = min(n0 + f * 16 + r, n - 1);
  f32x4 acc[2][2] = {};
  for (unsigned q = 0; q < quads; ++q) {
    u32x4 a[2], b[2];
    unsigned sa[2], sb[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      a[f] = ac[(static_cast<size_t>(rm[f]) * quads + q) * 4 + g];
      b[f] = bc[(static_cast<size_t>(rn[f]) * quads + q) * 4 + g];
      sa[f] = as[static_cast<size_t>(q) * m + rm[f]] >> (8 * g);
      sb[f] = bs[static_cast<size_t>(q) * n + rn[f]] >> (8 * g);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma16(b[j], a[i], acc[i][j], sb[j], sa[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (unsigned e = 0; e < 4; ++e) {
        const unsigned row = m0 + i * 16 + r, col = n0 + j * 16 + g * 4 + e;
        if (row < m && col < n) c[static_cast<int64_t>(row) * stride + col] = Elem<T>::from_f32(acc[i][j][e]);
      }
}

void check_product(int64_t m, int64_t n, int64_t k, int64_t stride) {
  require(m >= 0 && n >= 0 && k >= 1, "mx: m and n must be >= 0 and k >= 1");
  require(m < (1ll << 31) && n < (1ll << 31) && k <= (1ll << 31) - 256 && m * mx_quads(k) < (1ll << 31) &&
              n * mx_quads(k) < (1ll << 31) && ((m + 63) / 64) * ((n + 63) / 64) < (1ll << 31),
          "mx: a product's sizes are beyond what its grid holds (2^31 quads of a side, 2^31 tiles of 64 x 64)");
  require(stride >= n || m <= 1, "mx: stride must be at least n");
}

size_t round16(size_t b) { return (b + 15) / 16 * 16; }

}  // namespace
}  // namespace mx

using namespace mx;

size_t mx_product_workspace(int, int64_t m, int64_t n, int64_t k) {
  check_product(m, n, k, n);
  return 0;
}

void launch_mx_product(int dev, const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales,
                       int64_t m, int64_t n, int64_t k, void* c, const std::string& dtype, int64_t stride, void*,
                       size_t, void* stream) {
  const Type t = type_of(dtype, "mx_product: dtype must be bf16|f16|f32");
  check_product(m, n, k, stride);
  if (m == 0 || n == 0) return;
  require(a_codes && a_scales && b_codes && b_scales && c, "mx_product: null pointer");
  require(aligned(a_codes, 16) && aligned(b_codes, 16) && aligned(a_scales, 4) && aligned(b_scales, 4) &&
              aligned(c, size_of(t)),
          "mx_product: codes aligned to 16, scales to 4 bytes, the result to its type");
  OnDevice on(dev);
  const unsigned tn = static_cast<unsigned>((n + 63) / 64), tm = static_cast<unsigned>((m + 63) / 64);
  with_type(t, [&](auto e) {
    using T = decltype(e);
    hipLaunchKernelGGL(product_direct_kernel<T>, dim3(tm * tn), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const u32x4*>(a_codes), static_cast<const unsigned*>(a_scales),
                       static_cast<const u32x4*>(b_codes), static_cast<const unsigned*>(b_scales),
                       static_cast<unsigned>(m), static_cast<unsigned>(n), static_cast<unsigned>(mx_quads(k)),
                       static_cast<T*>(c), stride, Div(tn));
  });
  check(hipGetLastError(), "mx_product");
}

size_t mx_linear_workspace(int dev, int64_t m, int64_t n, int64_t k) {
  return round16(static_cast<size_t>(mx_codes_bytes(m, k) + mx_scales_bytes(m, k))) + mx_product_workspace(dev, m, n, k);
}

void launch_mx_linear(int dev, const void* x, const std::string& dtype, int64_t x_stride, const void* w_codes,
                      const void* w_scales, int64_t m, int64_t n, int64_t k, void* y, int64_t y_stride,
                      void* workspace, size_t workspace_bytes, void* stream) {
  require(workspace_bytes >= mx_linear_workspace(dev, m, n, k), "mx_linear: workspace too small");
  require(aligned(workspace, 16), "mx_linear: workspace aligned to 16 bytes");
  auto codes = static_cast<char*>(workspace);
  auto scales = codes + mx_codes_bytes(m, k);
  const size_t used = round16(static_cast<size_t>(mx_codes_bytes(m, k) + mx_scales_bytes(m, k)));
  launch_mx_quantize(dev, x, dtype, m, k, x_stride, false, codes, scales, stream);
  launch_mx_product(dev, codes, scales, w_codes, w_scales, m, n, k, y, dtype, y_stride, codes + used,
                    workspace_bytes - used, stream);
}

}  // namespace gpumon_hip
