// MXFP4 product and linear layer (format and layout: mx.h).
#include "mx_common.h"

namespace gpumon_hip {
namespace mx {
namespace {

typedef __attribute__((address_space(3))) void LdsVoid;
typedef const __attribute__((address_space(1))) void GlobalVoid;

// One wave's 16x16x128 step on one chunk of either side; S picks the quad's byte of the scale words.
// D: lane l holds row l & 15 of b's chunk and rows 4 (l >> 4) + i of a's.
template <int S>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c, unsigned sa, unsigned sb) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, S, (int)sa, S, (int)sb);
}

// s_waitcnt with a vmcnt and, if lgkm0, lgkmcnt(0).
constexpr int wait_imm(int vm, bool lgkm0) { return (vm & 15) | ((vm >> 4) << 14) | (7 << 4) | ((lgkm0 ? 0 : 15) << 8); }

template <int S>
using Int = std::integral_constant<int, S>;

// 2 x 2 waves, FM x FN chunks of 16 x 16 results each.
template <typename T, int FM, int FN>
__global__ void __launch_bounds__(256, FM* FN > 32 ? 1 : 2)
    product_tile_kernel(const char* __restrict__ ac, const char* __restrict__ as, const char* __restrict__ bc,
                        const char* __restrict__ bs, unsigned m, unsigned n, unsigned quads, T* __restrict__ c,
                        int64_t stride, Div tiles_n) {
  constexpr int kChunks = 2 * (FM + FN), kLoads = kChunks / 4, kScaleLoads = kChunks >= 16 ? kChunks / 16 : 1;
  constexpr int kStage = kChunks * 1024, kScales = kChunks * 256;
  __shared__ __attribute__((aligned(16))) char lds[4 * kStage + 2 * kScales];
  const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned tm = tiles_n.quot(blockIdx.x), tn = blockIdx.x - tm * tiles_n.d;
  const unsigned rbm = (m + 15) / 16, rbn = (n + 15) / 16, groups = (quads + 3) / 4;
  const unsigned wm = wave & 1, wn = wave >> 1;

  // chunk `x` of the tile, a's 2 FM first; row blocks past the end read the last one instead, and what
  // comes of them is not stored
  auto row_block = [&](unsigned x) {
    return x < 2 * FM ? min(tm * (2 * FM) + x, rbm - 1) : min(tn * (2 * FN) + x - 2 * FM, rbn - 1);
  };
  const char* src[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const unsigned x = wave * kLoads + i;
    src[i] = (x < 2 * FM ? ac : bc) + static_cast<size_t>(row_block(x)) * quads * 1024;
  }
  const char* ssrc[kScaleLoads];
#pragma unroll
  for (int i = 0; i < kScaleLoads; ++i) {
    const unsigned x = ((wave * kScaleLoads + i) * 4 + (lane >> 4)) % kChunks;
    ssrc[i] = (x < 2 * FM ? as : bs) + static_cast<size_t>(row_block(x)) * groups * 256 + (lane & 15) * 16;
  }
  auto load_stage = [&](unsigned t, int slot) {
    const unsigned q = min(t, quads - 1);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds((GlobalVoid*)(src[i] + static_cast<size_t>(q) * 1024 + lane * 16),
                                       (LdsVoid*)(lds + slot * kStage + (wave * kLoads + i) * 1024), 16, 0, 0);
  };
  auto load_scales = [&](unsigned g) {
    const unsigned q = min(g, groups - 1);
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i)
      __builtin_amdgcn_global_load_lds(
          (GlobalVoid*)(ssrc[i] + static_cast<size_t>(q) * 256),
          (LdsVoid*)(lds + 4 * kStage + (g & 1) * kScales + (wave * kScaleLoads + i) * 1024 % kScales), 16, 0, 0);
  };

  u32x4 fa[2][FM], fb[2][FN];
  unsigned sa[FM], sb[FN], sa2[FM], sb2[FN];
  f32x4 acc[FM][FN] = {};
  auto read_stage = [&](int slot, u32x4* a, u32x4* b) {
    const char* p = lds + slot * kStage + lane * 16;
#pragma unroll
    for (int i = 0; i < FM; ++i) a[i] = *reinterpret_cast<const u32x4*>(p + (wm * FM + i) * 1024);
#pragma unroll
    for (int j = 0; j < FN; ++j) b[j] = *reinterpret_cast<const u32x4*>(p + (2 * FM + wn * FN + j) * 1024);
  };
  auto read_scales = [&](unsigned g, unsigned* a, unsigned* b) {
    const char* p = lds + 4 * kStage + (g & 1) * kScales + lane * 4;
#pragma unroll
    for (int i = 0; i < FM; ++i) a[i] = *reinterpret_cast<const unsigned*>(p + (wm * FM + i) * 256);
#pragma unroll
    for (int j = 0; j < FN; ++j) b[j] = *reinterpret_cast<const unsigned*>(p + (2 * FM + wn * FN + j) * 256);
  };

  load_scales(0);
#pragma unroll
  for (int t = 0; t < 4; ++t) load_stage(t, t);
  __builtin_amdgcn_s_waitcnt(wait_imm(3 * kLoads, false));
  __builtin_amdgcn_s_barrier();
  read_scales(0, sa, sb);
  read_stage(0, fa[0], fb[0]);

  auto body = [&](unsigned g, auto step) {
    constexpr int J = decltype(step)::value;
    const unsigned t = g * 4 + J;
    // stage t + 1 is here, for every wave, and every wave has read stage t
    __builtin_amdgcn_s_waitcnt(wait_imm(2 * kLoads + (J == 1 || J == 2 ? kScaleLoads : 0), true));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (J == 0) load_scales(g + 1);
    load_stage(t + 4, J);
    read_stage((J + 1) & 3, fa[(J + 1) & 1], fb[(J + 1) & 1]);
    if constexpr (J == 3) read_scales(g + 1, sa2, sb2);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        acc[i][j] = mfma16<J>(fb[J & 1][j], fa[J & 1][i], acc[i][j], sb[j], sa[i]);
    if constexpr (J == 3) {
#pragma unroll
      for (int i = 0; i < FM; ++i) sa[i] = sa2[i];
#pragma unroll
      for (int j = 0; j < FN; ++j) sb[j] = sb2[j];
    }
#pragma unroll
    for (int i = 0; i < FM + FN; ++i) {  // one read of LDS, then its share of the matrix instructions
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, FM * FN / (FM + FN), 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const unsigned whole = quads / 4, rest = quads & 3;
  for (unsigned g = 0; g < whole; ++g) {
    body(g, Int<0>{});
    body(g, Int<1>{});
    body(g, Int<2>{});
    body(g, Int<3>{});
  }
  if (rest > 0) body(whole, Int<0>{});
  if (rest > 1) body(whole, Int<1>{});
  if (rest > 2) body(whole, Int<2>{});
  __builtin_amdgcn_s_waitcnt(wait_imm(0, true));  // nothing may arrive after the workgroup's memory is given back

  const unsigned row0 = (tm * 2 + wm) * FM * 16 + (lane & 15), col0 = (tn * 2 + wn) * FN * 16 + (lane >> 4) * 4;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const unsigned row = row0 + i * 16;
    if (row >= m) continue;
    T* out = c + static_cast<int64_t>(row) * stride;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const unsigned col = col0 + j * 16;
      T v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = Elem<T>::from_f32(acc[i][j][e]);
      if (col + 4 <= n) {
        __builtin_memcpy(out + col, v, sizeof(v));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < n) out[col + e] = v[e];
      }
    }
  }
}

// ---- few rows ----------------------------------------------------------------------------------
// x has at most 16 FM rows: the weights' bytes are the work. A workgroup takes R row blocks of b (16 R
// results a row of x), its waves whole groups of quads in turn, straight from memory to registers,
// U groups a wave in flight; the waves' sums meet in LDS in a fixed order. Sources of x: rows
// quantised before, or plain rows that each wave quantises for its own groups.
constexpr int kWaves = 8;

struct QuantizedRows {
  const char* codes;
  const char* scales;
  unsigned quads, groups, row_blocks;
  struct Raw {};
  static constexpr int kLds = 16;
  template <int FM, bool FULL>
  __device__ __forceinline__ void load(unsigned g, unsigned nq, unsigned lane, Raw&, u32x4 (&x)[4][FM], unsigned (&sx)[FM]) const {
#pragma unroll
    for (int f = 0; f < FM; ++f) {
      const unsigned rb = min(static_cast<unsigned>(f), row_blocks - 1);
      sx[f] = *reinterpret_cast<const unsigned*>(scales + (static_cast<size_t>(rb) * groups + g) * 256 + lane * 4);
#pragma unroll
      for (unsigned q = 0; q < 4; ++q)
        if (FULL || q < nq)
          x[q][f] = *reinterpret_cast<const u32x4*>(codes + (static_cast<size_t>(rb) * quads + g * 4 + q) * 1024 + lane * 16);
        else
          x[q][f] = u32x4{0, 0, 0, 0};
    }
  }
  template <int FM>
  __device__ __forceinline__ void finish(const Raw&, unsigned, char*, u32x4 (&)[4][FM], unsigned (&)[FM]) const {}
};

// Up to ROWS plain rows (ROWS <= 16): eight elements a lane of one row after the other, 16 lanes a quad,
// as the quantising kernel does; the codes change lanes in the wave's own piece of LDS. Rows of the
// operand from ROWS on repeat the last one.
template <typename X, int ROWS>
struct PlainRows {
  const X* x;
  int64_t stride;
  unsigned m;
  int k;
  static constexpr int kWords = 8 / Elem<X>::kPerWord;
  struct Raw {
    unsigned w[ROWS][kWords];
  };
  static constexpr int kLds = ROWS * 256 + 64 * ROWS;
  template <int FM, bool FULL>
  __device__ __forceinline__ void load(unsigned g, unsigned, unsigned lane, Raw& raw, u32x4 (&)[4][FM], unsigned (&)[FM]) const {
#pragma unroll
    for (unsigned r = 0; r < ROWS; ++r)
      load8(x + static_cast<int64_t>(min(r, m - 1)) * stride, static_cast<int>(g * 512 + lane * 8), k, raw.w[r]);
  }
  template <int FM>
  __device__ __forceinline__ void finish(const Raw& raw, unsigned lane, char* lds, u32x4 (&x)[4][FM], unsigned (&sx)[FM]) const {
    unsigned* codes = reinterpret_cast<unsigned*>(lds);  // [quad][block][row][4 words]
    unsigned char* scales = reinterpret_cast<unsigned char*>(lds + ROWS * 256);  // [block][row][quad]
    const unsigned quad = lane >> 4, block = (lane >> 2) & 3;
    __builtin_amdgcn_wave_barrier();  // the wave's earlier reads are done in order
#pragma unroll
    for (unsigned r = 0; r < ROWS; ++r) {
      unsigned m = 0;
#pragma unroll
      for (unsigned v : raw.w[r]) m = Elem<X>::amax(m, v);
      m = Elem<X>::amax_f32(m);
      m = max(m, dpp<kXor1>(m));
      m = max(m, dpp<kXor2>(m));
      const unsigned byte = scale_byte(m);
      codes[((lane >> 2) * ROWS + r) * 4 + (lane & 3)] = byte == 255 ? 0u : codes8<X>(raw.w[r], scale_of(byte));
      if ((lane & 3) == 0) scales[(block * ROWS + r) * 4 + quad] = static_cast<unsigned char>(byte);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const unsigned r = min(lane & 15, ROWS - 1u), b = lane >> 4;
#pragma unroll
    for (unsigned q = 0; q < 4; ++q) x[q][0] = *reinterpret_cast<const u32x4*>(codes + ((q * 4 + b) * ROWS + r) * 4);
    sx[0] = *reinterpret_cast<const unsigned*>(scales + (b * ROWS + r) * 4);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
};

template <typename T, typename Source, int FM, int R, int U>
__global__ void __launch_bounds__(64 * kWaves) product_few_rows_kernel(Source source, const char* __restrict__ bc,
                                                                       const char* __restrict__ bs, unsigned m, unsigned n,
                                                                       unsigned quads, T* __restrict__ c, int64_t stride) {
  constexpr int kSums = kWaves * R * FM * 1024;
  constexpr int kLds = kSums > kWaves * Source::kLds ? kSums : kWaves * Source::kLds;
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned rbn = (n + 15) / 16, groups = (quads + 3) / 4, rb0 = blockIdx.x * R;
  f32x4 acc[R][FM] = {};
  auto run = [&](auto count, auto full_groups, unsigned g0) {  // `count` groups, kWaves apart
    constexpr int N = decltype(count)::value;
    constexpr bool FULL = decltype(full_groups)::value != 0;
    typename Source::Raw raw[N];
    u32x4 x[N][4][FM], w[N][R][4];
    unsigned sx[N][FM], sw[N][R];
    const unsigned nq = FULL ? 4 : quads - g0 * 4;
#pragma unroll
    for (int u = 0; u < N; ++u) source.template load<FM, FULL>(g0 + u * kWaves, nq, lane, raw[u], x[u], sx[u]);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const unsigned rb = min(rb0 + r, rbn - 1), g = g0 + u * kWaves;
        sw[u][r] = *reinterpret_cast<const unsigned*>(bs + (static_cast<size_t>(rb) * groups + g) * 256 + lane * 4);
#pragma unroll
        for (unsigned q = 0; q < 4; ++q)
          if (FULL || q < nq)
            w[u][r][q] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4*>(bc + (static_cast<size_t>(rb) * quads + g * 4 + q) * 1024 + lane * 16));
          else
            w[u][r][q] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      source.template finish<FM>(raw[u], lane, lds + wave * Source::kLds, x[u], sx[u]);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int f = 0; f < FM; ++f) {
          acc[r][f] = mfma16<0>(w[u][r][0], x[u][0][f], acc[r][f], sw[u][r], sx[u][f]);
          acc[r][f] = mfma16<1>(w[u][r][1], x[u][1][f], acc[r][f], sw[u][r], sx[u][f]);
          acc[r][f] = mfma16<2>(w[u][r][2], x[u][2][f], acc[r][f], sw[u][r], sx[u][f]);
          acc[r][f] = mfma16<3>(w[u][r][3], x[u][3][f], acc[r][f], sw[u][r], sx[u][f]);
        }
    }
  };
  const unsigned whole = quads / 4;
  unsigned g = wave;
  for (; g + (U - 1) * kWaves < whole; g += U * kWaves) run(Int<U>{}, Int<1>{}, g);
  for (; g < whole; g += kWaves) run(Int<1>{}, Int<1>{}, g);
  if (g < groups) run(Int<1>{}, Int<0>{}, g);

  __syncthreads();
  f32x4* sums = reinterpret_cast<f32x4*>(lds);  // [wave][block][lane]
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int f = 0; f < FM; ++f) sums[((wave * R + r) * FM + f) * 64 + lane] = acc[r][f];
  __syncthreads();
  const float* flat = reinterpret_cast<const float*>(lds);
  // result i of the workgroup: row of x i / (16 R), column i % (16 R), at lane 16 (column % 16 / 4) + row % 16
  for (unsigned i = threadIdx.x; i < 16u * R * min(m, 16u * FM); i += 64 * kWaves) {
    const unsigned row = i / (16 * R), col = i % (16 * R);
    const unsigned at = (((col / 16) * FM + row / 16) * 64 + (col % 16 / 4) * 16 + row % 16) * 4 + col % 4;
    float v = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += flat[w * R * FM * 256 + at];
    if (rb0 * 16 + col < n) c[static_cast<int64_t>(row) * stride + rb0 * 16 + col] = Elem<T>::from_f32(v);
  }
}

template <typename T, int FM, int R, int U, typename Source>
void launch_few_rows(Source source, const void* bc, const void* bs, int64_t m, int64_t n, int64_t k, T* c,
                     int64_t stride, hipStream_t s) {
  hipLaunchKernelGGL((product_few_rows_kernel<T, Source, FM, R, U>), dim3(static_cast<unsigned>((n + 16 * R - 1) / (16 * R))),
                     dim3(64 * kWaves), 0, s, source, static_cast<const char*>(bc), static_cast<const char*>(bs),
                     static_cast<unsigned>(m), static_cast<unsigned>(n), static_cast<unsigned>(mx_quads(k)), c, stride);
}

constexpr int64_t kFusedRows = 16, kFewRows = 64;

void check_product(int64_t m, int64_t n, int64_t k, int64_t stride) {
  require(m >= 0 && n >= 0 && k >= 1, "mx: m and n must be >= 0 and k >= 1");
  require(mx_fits(m, k) && mx_fits(n, k) && ((m + 15) / 16) * ((n + 15) / 16) < (1ll << 28),
          "mx: a product's sizes are beyond its limits (mx.h)");
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
  require(aligned(a_codes, 16) && aligned(b_codes, 16) && aligned(a_scales, 16) && aligned(b_scales, 16) &&
              aligned(c, size_of(t)),
          "mx_product: codes and scales aligned to 16 bytes, the result to its type");
  OnDevice on(dev);
  with_type(t, [&](auto e) {
    using T = decltype(e);
    auto run = [&](auto kernel, int tile_m, int tile_n) {
      const unsigned tn = static_cast<unsigned>((n + tile_n - 1) / tile_n), tm = static_cast<unsigned>((m + tile_m - 1) / tile_m);
      hipLaunchKernelGGL(kernel, dim3(tm * tn), dim3(256), 0, static_cast<hipStream_t>(stream),
                         static_cast<const char*>(a_codes), static_cast<const char*>(a_scales),
                         static_cast<const char*>(b_codes), static_cast<const char*>(b_scales),
                         static_cast<unsigned>(m), static_cast<unsigned>(n), static_cast<unsigned>(mx_quads(k)),
                         static_cast<T*>(c), stride, Div(tn));
    };
    if (m <= kFewRows) {
      const QuantizedRows x{static_cast<const char*>(a_codes), static_cast<const char*>(a_scales),
                            static_cast<unsigned>(mx_quads(k)), static_cast<unsigned>(mx_groups(k)),
                            static_cast<unsigned>(mx_row_blocks(m))};
      auto s = static_cast<hipStream_t>(stream);
      auto out = static_cast<T*>(c);
      if (m <= 16) launch_few_rows<T, 1, 1, 2>(x, b_codes, b_scales, m, n, k, out, stride, s);
      else if (m <= 32) launch_few_rows<T, 2, 2, 2>(x, b_codes, b_scales, m, n, k, out, stride, s);
      else launch_few_rows<T, 4, 2, 2>(x, b_codes, b_scales, m, n, k, out, stride, s);
    } else if (m > 1024 && n > 1024) run(product_tile_kernel<T, 8, 8>, 256, 256);
    else if (m > 64 && n > 64) run(product_tile_kernel<T, 4, 4>, 128, 128);
    else run(product_tile_kernel<T, 2, 2>, 64, 64);
  });
  check(hipGetLastError(), "mx_product");
}

size_t mx_linear_workspace(int dev, int64_t m, int64_t n, int64_t k) {
  check_product(m, n, k, n);
  if (m <= kFusedRows) return 0;
  return round16(static_cast<size_t>(mx_codes_bytes(m, k) + mx_scales_bytes(m, k))) + mx_product_workspace(dev, m, n, k);
}

void launch_mx_linear(int dev, const void* x, const std::string& dtype, int64_t x_stride, const void* w_codes,
                      const void* w_scales, int64_t m, int64_t n, int64_t k, void* y, int64_t y_stride,
                      void* workspace, size_t workspace_bytes, void* stream) {
  const Type t = type_of(dtype, "mx_linear: dtype must be bf16|f16|f32");
  check_product(m, n, k, y_stride);
  require(x_stride >= k || m <= 1, "mx_linear: x_stride must be at least k");
  if (m == 0 || n == 0) return;
  require(x && w_codes && w_scales && y, "mx_linear: null pointer");
  require(aligned(x, size_of(t)) && aligned(y, size_of(t)) && aligned(w_codes, 16) && aligned(w_scales, 16),
          "mx_linear: x and y aligned to their type, codes and scales to 16 bytes");
  if (m <= kFusedRows) {
    OnDevice on(dev);
    auto s = static_cast<hipStream_t>(stream);
    with_type(t, [&](auto e) {
      using T = decltype(e);
      auto px = static_cast<const T*>(x);
      auto out = static_cast<T*>(y);
      const auto rows = static_cast<unsigned>(m);
      const int len = static_cast<int>(k);
      if (m == 1) launch_few_rows<T, 1, 1, 2>(PlainRows<T, 1>{px, x_stride, rows, len}, w_codes, w_scales, m, n, k, out, y_stride, s);
      else if (m <= 4) launch_few_rows<T, 1, 1, 2>(PlainRows<T, 4>{px, x_stride, rows, len}, w_codes, w_scales, m, n, k, out, y_stride, s);
      else if (m <= 8) launch_few_rows<T, 1, 2, 1>(PlainRows<T, 8>{px, x_stride, rows, len}, w_codes, w_scales, m, n, k, out, y_stride, s);
      else launch_few_rows<T, 1, 2, 1>(PlainRows<T, 16>{px, x_stride, rows, len}, w_codes, w_scales, m, n, k, out, y_stride, s);
    });
    check(hipGetLastError(), "mx_linear");
    return;
  }
  require(workspace && workspace_bytes >= mx_linear_workspace(dev, m, n, k), "mx_linear: workspace too small");
  require(aligned(workspace, 16), "mx_linear: workspace aligned to 16 bytes");
  auto codes = static_cast<char*>(workspace);
  auto scales = codes + mx_codes_bytes(m, k);
  const size_t used = round16(static_cast<size_t>(mx_codes_bytes(m, k) + mx_scales_bytes(m, k)));
  launch_mx_quantize(dev, x, dtype, m, k, x_stride, false, codes, scales, stream);
  launch_mx_product(dev, codes, scales, w_codes, w_scales, m, n, k, y, dtype, y_stride, codes + used,
                    workspace_bytes - used, stream);
}

}  // namespace gpumon_hip
