// What the MXFP4 kernels share: element types, the block's scale and codes, argument checks.
#pragma once

#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>
#include <type_traits>

#include "hip_api.h"
#include "mx.h"

namespace gpumon_hip {
namespace mx {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The conversions of gfx950 divide (multiply) by the scale's power of two exactly, round halves to
// even and saturate at 6, for every scale byte 0..254 including 2^-127, and read 255 as NaN; tested
// over all 16-bit inputs under all scales that they can have, and back over all codes times all scales.
__device__ __forceinline__ float scale_of(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }

// Scale byte of a block from the bits of its largest magnitude as an f32 (magnitudes order like their
// bits, and infinities and NaN come out on top): floor(log2) is the exponent field - 127, subnormals
// end at the clamp.
__device__ __forceinline__ unsigned scale_byte(unsigned amax_bits) {
  const unsigned e = amax_bits >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}

template <typename T>
struct Elem;
template <>
struct Elem<__bf16> {
  static constexpr int kPerWord = 2;
  __device__ static unsigned amax(unsigned m, unsigned w) {  // running magnitudes, per half
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                  __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
  }
  __device__ static unsigned amax_f32(unsigned m) { return max(m & 0xffff0000u, m << 16); }
  template <int SEL>
  __device__ static unsigned cvt(unsigned old, const unsigned* w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, w[0]), s, SEL);
  }
  __device__ static __bf16 from_f32(float v) { return static_cast<__bf16>(v); }
};
template <>
struct Elem<_Float16> {
  static constexpr int kPerWord = 2;
  __device__ static unsigned amax(unsigned m, unsigned w) { return Elem<__bf16>::amax(m, w); }
  __device__ static unsigned amax_f32(unsigned m) {
    const unsigned h = max(m >> 16, m & 0xffffu);  // an infinity or NaN converts to one
    return __builtin_bit_cast(unsigned, static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(h))));
  }
  template <int SEL>
  __device__ static unsigned cvt(unsigned old, const unsigned* w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, w[0]), s, SEL);
  }
  __device__ static _Float16 from_f32(float v) { return static_cast<_Float16>(v); }
};
template <>
struct Elem<float> {
  static constexpr int kPerWord = 1;
  __device__ static unsigned amax(unsigned m, unsigned w) { return max(m, w & 0x7fffffffu); }
  __device__ static unsigned amax_f32(unsigned m) { return m; }
  template <int SEL>
  __device__ static unsigned cvt(unsigned old, const unsigned* w, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, __builtin_bit_cast(float, w[0]),
                                                    __builtin_bit_cast(float, w[1]), s, SEL);
  }
  __device__ static float from_f32(float v) { return v; }
};

// Eight elements to one word of codes. `w`: the elements' words (4 of 16-bit types, 8 of f32).
template <typename T>
__device__ __forceinline__ unsigned codes8(const unsigned* w, float s) {
  constexpr int P = 2 / Elem<T>::kPerWord;  // words a pair
  unsigned c = 0;
  c = Elem<T>::template cvt<0>(c, w, s);
  c = Elem<T>::template cvt<1>(c, w + P, s);
  c = Elem<T>::template cvt<2>(c, w + 2 * P, s);
  c = Elem<T>::template cvt<3>(c, w + 3 * P, s);
  return c;
}

// Eight elements of a row from column k0 on as words, zeros from column k on. Rows start where the
// caller's stride puts them, so the 16 bytes need not be aligned. A branch a lane would make the
// compiler wait for each load by itself, so how to load is chosen for a wave: all within the row; up to
// the row's end, reading its last 16 bytes instead and shifting them into place; or a row of fewer.
enum class Reach { whole, end, tiny };
template <typename T>
__device__ __forceinline__ Reach reach(int end, int k) {  // end: past the wave's last column
  return end <= k ? Reach::whole : k >= 16 / static_cast<int>(sizeof(T)) ? Reach::end : Reach::tiny;
}
// v's bytes from `n` on, zeros after them
__device__ __forceinline__ void shift16(unsigned* v, unsigned n) {
  uint64_t lo = v[0] | static_cast<uint64_t>(v[1]) << 32, hi = v[2] | static_cast<uint64_t>(v[3]) << 32;
  const unsigned bits = n % 8 * 8;
  if (n >= 16) hi = 0;
  if (n >= 8) lo = hi, hi = 0;
  lo = lo >> bits | hi << 1 << (63 - bits);
  hi >>= bits;
  v[0] = static_cast<unsigned>(lo), v[1] = static_cast<unsigned>(lo >> 32);
  v[2] = static_cast<unsigned>(hi), v[3] = static_cast<unsigned>(hi >> 32);
}
template <Reach R, typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int k0, int k, unsigned* w) {
  constexpr int kPer = 16 / sizeof(T);  // elements of 16 bytes
#pragma unroll
  for (int h = 0; h < 8 / kPer; ++h) {
    unsigned* v = w + h * 4;
    const int c = k0 + h * kPer;
    if constexpr (R == Reach::whole) {
      __builtin_memcpy(v, row + c, 16);
    } else if constexpr (R == Reach::end) {
      const int from = min(c, k - kPer);
      __builtin_memcpy(v, row + from, 16);
      shift16(v, static_cast<unsigned>(min(c - from, kPer)) * sizeof(T));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = 0;
#pragma unroll
        for (unsigned e = 0; e < 4 / sizeof(T); ++e) {
          const int at = c + i * (4 / static_cast<int>(sizeof(T))) + static_cast<int>(e);
          unsigned bits = 0;
          __builtin_memcpy(&bits, row + min(at, k - 1), sizeof(T));
          v[i] |= (at < k ? bits : 0u) << (e * 8 * sizeof(T));
        }
      }
    }
  }
}
// f(reach) with the reach as a constant
template <typename T, typename F>
__device__ __forceinline__ void with_reach(int end, int k, F f) {
  const Reach r = reach<T>(end, k);
  if (r == Reach::whole) f(std::integral_constant<Reach, Reach::whole>{});
  else if (r == Reach::end) f(std::integral_constant<Reach, Reach::end>{});
  else f(std::integral_constant<Reach, Reach::tiny>{});
}

// Rows that all start on 64 bytes: stores that fill whole lines of the caches.
template <typename T>
__device__ __forceinline__ bool whole_lines(const T* to, int64_t stride) {
  return ((reinterpret_cast<uintptr_t>(to) | static_cast<uintptr_t>(stride) * sizeof(T)) & 63) == 0;
}

// 16 bytes, aligned or not, `past` the caches or through them. Past them saves the cache what is never read
// again there (8192 x 8192 dequantised to bf16 6.2 TB/s, through them 4.8), but a line written in parts by
// several stores goes to memory in parts, where the cache would join them.
template <typename T>
__device__ __forceinline__ void store16(T* to, const T* v, bool past) {
  struct __attribute__((packed, aligned(sizeof(T)))) Out {
    u32x4 q;
  };
  u32x4 q;
  __builtin_memcpy(&q, v, 16);
  if (past) {
    __builtin_nontemporal_store(q, &reinterpret_cast<Out*>(to)->q);
  } else {
    // the compiler would make one plain store of the two
    asm volatile("" ::: "memory");
    reinterpret_cast<Out*>(to)->q = q;
    asm volatile("" ::: "memory");
  }
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v) {  // another lane's v, within rows of 16 lanes
  return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E;

// x / d for x < 2^31 as a multiplication: m = floor(2^(31 + l) / d) + 1 with 2^l >= d errs by less
// than one part in 2^31 of the quotient, so the floor is exact.
struct Div {
  unsigned d, m;
  int s;
  Div() : d(1), m(0), s(0) {}
  explicit Div(unsigned div) : d(div), m(0), s(0) {
    int l = 0;
    while ((1ull << l) < div) ++l;
    m = static_cast<unsigned>((1ull << (31 + l)) / div + 1);
    s = l - 1;
  }
  __device__ __forceinline__ unsigned quot(unsigned x) const {
    return d == 1 ? x : static_cast<unsigned>((static_cast<uint64_t>(x) * m) >> 32) >> s;
  }
};

// Which of `total` pieces of work this workgroup takes in round r; false if none is left for it.
// Workgroups run on the eight XCDs in turn, and each XCD takes a run of neighbours, so that what
// neighbours share meets in one cache.
__device__ __forceinline__ bool turn(unsigned total, unsigned r, unsigned& piece) {
  const unsigned first = r * gridDim.x, place = blockIdx.x / 8;
  const unsigned count = first < total ? min(total - first, gridDim.x) : 0, per = (count + 7) / 8;
  const unsigned p = blockIdx.x % 8 * per + place;
  piece = first + p;
  return place < per && p < count;
}

// A matrix's tiles in the order in which they are taken: bands of H rows of tiles, down each column of a
// band.
template <unsigned H>
struct Tiles {
  unsigned rows, cols, total;
  Div band, last;  // tiles of a band; rows of the last band
  Tiles(unsigned r, unsigned c) : rows(r), cols(c), total(r * c), band(H * c), last((r + H - 1) % H + 1) {}
  __device__ __forceinline__ void at(unsigned piece, unsigned& row, unsigned& col) const {
    const unsigned b = band.quot(piece), in = piece - b * band.d;
    const bool whole = b * H + H <= rows;
    col = whole ? in / H : last.quot(in);
    row = b * H + in - col * (whole ? H : last.d);
    row = __builtin_amdgcn_readfirstlane(row), col = __builtin_amdgcn_readfirstlane(col);
  }
};

// ---- host ------------------------------------------------------------------------------------
// Keeps the calling thread's current device.
class OnDevice {
 public:
  explicit OnDevice(int dev) {
    check(hipGetDevice(&old_), "hipGetDevice");
    if (old_ != dev) check(hipSetDevice(dev), "hipSetDevice");
    dev_ = dev;
  }
  ~OnDevice() {
    if (old_ != dev_) (void)hipSetDevice(old_);
  }

 private:
  int old_ = 0, dev_ = 0;
};

inline void require(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}
inline bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

enum class Type { bf16, f16, f32 };
inline Type type_of(const std::string& s, const char* what) {
  if (s == "bf16") return Type::bf16;
  if (s == "f16") return Type::f16;
  if (s == "f32") return Type::f32;
  throw std::invalid_argument(what);
}
inline int size_of(Type t) { return t == Type::f32 ? 4 : 2; }
template <typename F>
void with_type(Type t, F f) {  // f(T{})
  if (t == Type::bf16) f(__bf16{});
  else if (t == Type::f16) f(_Float16{});
  else f(float{});
}

// A quantised operand; and one in a buffer, codes then scales.
struct Operand {
  const char *codes, *scales;
};
inline Operand operand(const void* codes, const void* scales) {
  return {static_cast<const char*>(codes), static_cast<const char*>(scales)};
}
inline size_t mx_bytes(int64_t rows, int64_t k) {  // a multiple of 256
  return static_cast<size_t>(mx_codes_bytes(rows, k) + mx_scales_bytes(rows, k));
}
struct Quantized {
  char* at;
  int64_t rows, k;
  char* scales() const { return at + mx_codes_bytes(rows, k); }
  Operand operand() const { return {at, scales()}; }
};

// A matrix to quantise both ways: x [rows, k], its results in buffers as above.
struct Source {
  const void* x;
  int64_t stride, rows, k;
  char *along, *down;
};
void check_source(const Source& s, Type t);
void launch_quantize_both(int dev, const Source* sources, int count, Type t, hipStream_t s);  // up to two

// A product c [m, n] = a [m, k] b [n, k]^T.
struct Job {
  Operand a, b;
  int64_t m, n, k;
  void* c;
  int64_t stride;
};

}  // namespace mx
}  // namespace gpumon_hip
