// MXFP4 product and linear layer (format and layout: mx.h).
#include <algorithm>
#include <atomic>
#include <cmath>

#include "mx_common.h"

namespace gpumon_hip {
namespace mx {
namespace {

typedef __attribute__((address_space(3))) void LdsVoid;

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

// Buffers: a uniform base, an offset of 32 bits a lane; past `size` reads give zeros. The whole offset is the
// lane's: an instruction's uniform offset is not counted in its check against `size`.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer(const char* base, unsigned size) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, static_cast<int>(size), 0x00020000);
}
// 16 bytes a lane to LDS, lane after lane.
__device__ __forceinline__ void load_lds(Buffer b, unsigned offset, char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (LdsVoid*)lds, 16, static_cast<int>(offset), 0, 0, 0);
}

// All waves of the workgroup meet, after waits of their own: a barrier that no access to memory crosses,
// but that, unlike __syncthreads, waits for no loads still on their way to LDS.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int S>
using Int = std::integral_constant<int, S>;

// The order of a stage's work in a wave: FM x FN matrix instructions, row after row, and between them,
// evenly, the next stages' loads (kLoad), and the next stage's operands from LDS: b's (kB), a's last TAIL
// rows (kTail), for both of which there are two sets of registers, and a's other rows (kA), each into the
// registers of its row once that row is done.
enum Op { kLoad, kB, kTail, kA };
template <int FM, int FN, int LOADS>
struct Order {
  static constexpr int kTails = FM / 4 > 0 ? FM / 4 : 1, kOps = LOADS + FN + FM;
  Op op[kOps] = {};
  int index[kOps] = {}, before[kOps] = {};  // matrix instructions before it
  constexpr Order() {
    int load = 0, b = 0, tail = 0, a = 0;
    for (int o = 0; o < kOps; ++o) {
      before[o] = (o + 1) * FM * FN / (kOps + 1);
      if (a < FM - kTails && before[o] >= (a + 1) * FN) op[o] = kA, index[o] = a++;
      else if (tail < kTails) op[o] = kTail, index[o] = tail++;
      else if (load < LOADS && load <= b) op[o] = kLoad, index[o] = load++;
      else if (b < FN) op[o] = kB, index[o] = b++;
      else if (load < LOADS) op[o] = kLoad, index[o] = load++;
      else op[o] = kA, before[o] = (a + 1) * FN, index[o] = a++;
    }
  }
};

template <int O, int FM, int FN, int LOADS>
__device__ __forceinline__ void hold() {
  constexpr Order<FM, FN, LOADS> order;
  if constexpr (O < order.kOps) {
    constexpr int before = order.before[O] - (O ? order.before[O ? O - 1 : 0] : 0);
    if constexpr (before > 0) __builtin_amdgcn_sched_group_barrier(0x008, before, 0);
    __builtin_amdgcn_sched_group_barrier(order.op[O] == kLoad ? 0x010 : 0x100, 1, 0);
    hold<O + 1, FM, FN, LOADS>();
  } else {
    __builtin_amdgcn_sched_group_barrier(0x008, FM * FN - order.before[order.kOps - 1], 0);
  }
}

// WM x WN waves, FM x FN chunks of 16 x 16 results each: sums of 128 elements a matrix instruction in f32,
// scales applied by it, rounded once at the end. The stages (a quad of every chunk of the tile) go
// through LDS in four slots, loaded three stages ahead, without a break from one tile to the next; a
// stage's operands are read into registers while the one before multiplies, so that the matrix
// instructions wait for nothing but the barrier (Order). b's rows take the instruction's A side: a lane's
// four sums are neighbours in a row of c.
//
// The larger the tile the less each element is read: 256 x 256 results need 32 KiB a stage for 64 matrix
// instructions a SIMD. Eight waves of 128 x 64, since four of 128 x 128, which read a third less from LDS,
// were no faster (8192^3 236 to 254 us, these 240 to 261 in the same run). What bounds large products is the
// power their operands' bits take: for seconds on end 8192^3 takes 223 us on random ones, 1379 to 1393 W of the
// card's 1400 at 1692 MHz, and 157 on zeros, 1100 W at 2384 MHz; over runs and cards 212 to 261 and 157 to 174.
// Matrix instructions alone, on random registers, come to 7.10 PFLOP/s, and 6.49 in the 32x32x64 form. About
// 10 us of a launch are its first loads and last stores (one tile a compute unit, fitted over k). Smaller
// tiles are for fewer results, so that every compute unit has one (kTiles has what each takes).
//
// One launch takes up to two products, the second's tiles after the first's.
// SPLIT: the tiles' columns are taken `parts` times, each time with `per` of k's groups of quads, and each
// part's sums go to a matrix of its own.
struct Product {
  const char *ac, *as, *bc, *bs;
  void* c;
  int64_t stride;
  unsigned m, n, quads, per;
  Div part_cols;
  Tiles<8> tiles;
};
struct Products {
  Product p[2];
};
template <typename T, int FM, int FN, int WM, int WN, int RESIDENT, bool SPLIT = false>
__global__ void __launch_bounds__(64 * WM * WN, RESIDENT * WM * WN / 4) product_tile_kernel(Products products) {
  constexpr int TM = FM * WM, TN = FN * WN, kChunks = TM + TN, kLoads = kChunks / (WM * WN);
  constexpr int kScaleLoads = kChunks >= 4 * WM * WN ? kChunks / (4 * WM * WN) : 1;
  constexpr int kStage = kChunks * 1024, kScales = kChunks * 256;
  // results leave through LDS in pieces of 16 rows x up to 128 bytes, kParts times 16 bytes a row
  constexpr int kPiece = 8 / static_cast<int>(sizeof(T)) < FN ? 8 / static_cast<int>(sizeof(T)) : FN;
  constexpr int kParts = kPiece * static_cast<int>(sizeof(T)), kOut = 256 * kParts;
  __shared__ __attribute__((aligned(16))) char lds[4 * kStage + 2 * kScales + WM * WN * kOut];
  const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned wm = wave % WM, wn = wave / WM;

  Buffer src[kLoads], ssrc[kScaleLoads];
  unsigned soff[kScaleLoads];  // four chunks' scales a load, 16 lanes each; TM is a multiple of 4
  // Where the loads come from: chunk x of a tile, a's TM first. Row blocks past the end read the last one
  // instead, and what comes of them is not stored. Past the last tile, and past the last quad, zeros come
  // without a read (load_lds): four steps at a time are taken, and scales there are zeros too.
  auto aim = [&](bool any, const Product& p, unsigned tm, unsigned tn) {
    const unsigned rbm = (p.m + 15) / 16, rbn = (p.n + 15) / 16, quads = p.quads, all_groups = (quads + 3) / 4;
    unsigned g0 = 0;
    if constexpr (SPLIT) {
      const unsigned part = p.part_cols.quot(tn);
      tn -= part * p.part_cols.d;
      g0 = part * p.per;
    }
    auto row_block = [&](unsigned x) {
      return x < TM ? min(tm * TM + x, rbm - 1) : min(tn * TN + x - TM, rbn - 1);
    };
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const unsigned x = wave * kLoads + i;
      src[i] = buffer((x < TM ? p.ac : p.bc) + (static_cast<size_t>(row_block(x)) * quads + g0 * 4) * 1024,
                      any ? (quads - g0 * 4) * 1024 : 0);
    }
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
      const unsigned x = (wave * kScaleLoads + i) * 4 % kChunks, first = row_block(x);
      ssrc[i] = buffer((x < TM ? p.as : p.bs) + (static_cast<size_t>(first) * all_groups + g0) * 256,
                       any ? ((row_block(x + 3) - first + 1) * all_groups - g0) * 256 : 0);
      soff[i] = (row_block(x + (lane >> 4)) - first) * all_groups * 256 + (lane & 15) * 16;
    }
  };
  auto load_chunk = [&](int i, unsigned at, int slot) {
    load_lds(src[i], lane * 16 + at, lds + slot * kStage + (wave * kLoads + i) * 1024);
  };
  auto load_scales = [&](unsigned g, unsigned half) {
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i)
      load_lds(ssrc[i], soff[i] + g * 256, lds + 4 * kStage + half * kScales + (wave * kScaleLoads + i) * 1024 % kScales);
  };

  constexpr Order<FM, FN, kLoads> order;
  constexpr int kTails = order.kTails, kHead = FM - kTails;
  u32x4 fa[kHead], ft[2][kTails], fb[2][FN];
  unsigned sa[FM], sb[FN];
  f32x4 acc[FM][FN];
  auto read_a = [&](int x, int slot) {
    return *reinterpret_cast<const u32x4*>(lds + slot * kStage + lane * 16 + (wm * FM + x) * 1024);
  };
  auto read_b = [&](int x, int slot) {
    return *reinterpret_cast<const u32x4*>(lds + slot * kStage + lane * 16 + (TM + wn * FN + x) * 1024);
  };
  auto read_scales = [&](unsigned half) {
    const char* p = lds + 4 * kStage + half * kScales + lane * 4;
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[i] = *reinterpret_cast<const unsigned*>(p + (wm * FM + i) * 256);
#pragma unroll
    for (int j = 0; j < FN; ++j) sb[j] = *reinterpret_cast<const unsigned*>(p + (TM + wn * FN + j) * 256);
  };

  // the tile of round r: which product's, and where
  auto tile_of = [&](unsigned r, unsigned& which, unsigned& row, unsigned& col) {
    unsigned piece;
    const unsigned first = products.p[0].tiles.total;
    const bool any = turn(first + products.p[1].tiles.total, r, piece);
    which = piece < first || !any ? 0 : 1;
    products.p[which].tiles.at(piece - (which ? first : 0), row, col);
    return any;
  };
  unsigned which = 0, tm = 0, tn = 0, round = 0;
  if (!tile_of(0, which, tm, tn)) return;
  aim(true, products.p[which], tm, tn);
  load_scales(0, 0);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_chunk(i, t * 1024, t);
  __builtin_amdgcn_s_waitcnt(wait_imm(3 * kLoads, false));
  meet();
  read_scales(0);
#pragma unroll
  for (int x = 0; x < kHead; ++x) fa[x] = read_a(x, 0);
#pragma unroll
  for (int x = 0; x < kTails; ++x) ft[0][x] = read_a(kHead + x, 0);
#pragma unroll
  for (int x = 0; x < FN; ++x) fb[0][x] = read_b(x, 0);

  unsigned half = 0;     // of the scales' two places, the one in use
  auto body = [&](unsigned g, unsigned groups, auto step) {
    constexpr int J = decltype(step)::value;
    // stage g * 4 + J + 1 is here, for every wave, and every wave has read the one before it
    constexpr int kAfter = 2 * kLoads + (J == 1 || J == 2 ? kScaleLoads : 0);
    __builtin_amdgcn_s_waitcnt(wait_imm(kAfter, true));
    meet();
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kNow = J & 1, kNext = kNow ^ 1, kSlot = (J + 1) & 3;
    const bool last = g + 1 == groups;  // then the next tile's loads
    const unsigned at = last ? J * 1024 : (g * 4 + J + 4) * 1024;
    auto multiply = [&](int from, int to) {
#pragma unroll
      for (int x = from; x < to; ++x) {
        const int i = x / FN, j = i % 2 ? FN - 1 - x % FN : x % FN;  // to and fro: each keeps an operand of the last
        acc[i][j] = mfma16<J>(fb[kNow][j], i < kHead ? fa[i] : ft[kNow][i - kHead], acc[i][j], sb[j], sa[i]);
      }
    };
    if constexpr (J == 0) load_scales(last ? 0 : g + 1, half ^ 1);
#pragma unroll
    for (int o = 0; o < order.kOps; ++o) {
      multiply(o ? order.before[o - 1] : 0, order.before[o]);
      const int x = order.index[o];
      if (order.op[o] == kLoad) load_chunk(x, at, J);
      else if (order.op[o] == kB) fb[kNext][x] = read_b(x, kSlot);
      else if (order.op[o] == kTail) ft[kNext][x] = read_a(kHead + x, kSlot);
      else fa[x] = read_a(x, kSlot);
    }
    multiply(order.before[order.kOps - 1], FM * FN);
    // and the scheduler is held to it
    if constexpr (J == 0) __builtin_amdgcn_sched_group_barrier(0x010, kScaleLoads, 0);
    hold<0, FM, FN, kLoads>();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (J == 3) {
      half ^= 1;
      read_scales(half);
    }
  };

  for (;;) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    unsigned next = 0, next_m = 0, next_n = 0;
    const bool more = tile_of(round + 1, next, next_m, next_n);
    const Product& p = products.p[which];
    unsigned groups = (p.quads + 3) / 4, col = tn, part = 0;
    if constexpr (SPLIT) {
      part = p.part_cols.quot(tn);
      col -= part * p.part_cols.d;
      groups = min(p.per, groups - part * p.per);
    }
#pragma unroll 1
    for (unsigned g = 0; g < groups; ++g) {
      if (g + 1 == groups) aim(more, products.p[next], next_m, next_n);
      body(g, groups, Int<0>{});
      body(g, groups, Int<1>{});
      body(g, groups, Int<2>{});
      body(g, groups, Int<3>{});
    }

    unsigned l = lane;
    asm volatile("" : "+v"(l));  // what follows from the lane is computed here, not kept through the loop above
    const unsigned row0 = (tm * WM + wm) * FM * 16, col0 = (col * WN + wn) * FN * 16, r = l & 15, q = l >> 4;
    const unsigned m = p.m, n = p.n;
    const int64_t stride = p.stride;
    T* out = static_cast<T*>(p.c) + static_cast<size_t>(part) * m * n + static_cast<int64_t>(row0) * stride + col0;
    char* piece = lds + 4 * kStage + 2 * kScales + wave * kOut;
    auto leave = [&](auto store) {
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int h = 0; h < FN; h += kPiece) {
          // the 16-byte parts' places in a row are mixed by the row: neither writes nor reads meet in a bank
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (unsigned j = 0; j < kPiece; ++j) {
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = Elem<T>::from_f32(acc[i][h + j][e]);
            const unsigned at = (j * 4 + q) * sizeof(v);  // in the row
            __builtin_memcpy(__builtin_assume_aligned(piece + r * (16 * kParts) + ((at / 16) ^ (r % kParts)) * 16 + at % 16, sizeof(v)), v, sizeof(v));
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (unsigned o = 0; o < kParts / 4; ++o) {
            const unsigned row = o * (64 / kParts) + l / kParts, part = l % kParts;
            T v[16 / sizeof(T)];
            __builtin_memcpy(v, __builtin_assume_aligned(piece + row * (16 * kParts) + (part ^ (row % kParts)) * 16, 16), 16);
            store(i * 16 + row, h * 16 + part * (16 / sizeof(T)), v);
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    };
    // A store instruction leaves up to four pieces of a row; past the caches where they are whole lines
    // (8192 x 8064 x 512 to bf16 35 us, through them 38 to 39; 8192 x 8016 71 and 49; 8192 x 8001 102 and 55).
    const bool past = __builtin_amdgcn_readfirstlane(whole_lines(out, stride));
    if (__builtin_amdgcn_readfirstlane(row0 + FM * 16 <= m && col0 + FN * 16 <= n)) {
      leave([&](unsigned row, unsigned col, const T* v) {
        store16(out + static_cast<int64_t>(row) * stride + col, v, past);
      });
    } else {
      leave([&](unsigned row, unsigned col, const T* v) {
        if (row0 + row >= m) return;
#pragma unroll
        for (unsigned e = 0; e < 16 / sizeof(T); ++e)
          if (col0 + col + e < n) out[static_cast<int64_t>(row) * stride + col + e] = v[e];
      });
    }
    if (!more) break;
    which = next, tm = next_m, tn = next_n, ++round;
  }
  __builtin_amdgcn_s_waitcnt(wait_imm(0, true));  // no load may arrive after the workgroup's memory is given back
}

// c = the parts' sums, added up in their order (no atomics: the same result every time); four columns a
// thread. 206 x 491 results of 4 parts: 5.0 us, next to 6.4 for the parts.
template <typename T>
__global__ void __launch_bounds__(256) product_sum_kernel(const float* __restrict__ sums, unsigned parts, unsigned m,
                                                          unsigned n, T* __restrict__ c, int64_t stride, Div quarters) {
  const unsigned i = blockIdx.x * 256 + threadIdx.x, row = quarters.quot(i), col = (i - row * quarters.d) * 4;
  if (row >= m) return;
  const size_t at = static_cast<size_t>(row) * n + col, step = static_cast<size_t>(m) * n;
  T* out = c + static_cast<int64_t>(row) * stride + col;
  if (col + 4 <= n) {
    f32x4 v = {0, 0, 0, 0};
    for (unsigned p = 0; p < parts; ++p) {
      f32x4 x;
      __builtin_memcpy(&x, sums + p * step + at, 16);
      v += x;
    }
    T o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = Elem<T>::from_f32(v[e]);
    __builtin_memcpy(out, o, sizeof(o));
  } else {
    for (unsigned e = 0; col + e < n; ++e) {
      float v = 0;
      for (unsigned p = 0; p < parts; ++p) v += sums[p * step + at + e];
      out[e] = Elem<T>::from_f32(v);
    }
  }
}

// ---- few rows ----------------------------------------------------------------------------------
// x has at most 16 FM rows: the weights' bytes are the work (8192 x 8192 weights, 36 MB: a row 7.2 us,
// 5.0 TB/s, 64 rows, whose codes each workgroup reads too, 11.8; a row on 28672 x 8192 5.7 TB/s). A workgroup
// takes R row blocks of b (16 R
// results a row of x), its waves whole groups of quads in turn, straight from memory to registers,
// U groups a wave in flight; the waves' sums meet in LDS in a fixed order. Sources of x: rows
// quantised before, or plain rows that each wave quantises for its own groups.
struct QuantizedRows {
  const char* codes;
  const char* scales;
  unsigned quads, groups, row_blocks;
  struct Raw {};
  static constexpr bool kFirst = false;
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

// Up to ROWS plain rows: eight elements a lane of one row after the other, 16 lanes a quad,
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
  static constexpr bool kFirst = true;
  static constexpr int kLds = ROWS * 256 + 64 * ROWS;
  template <int FM, bool FULL>
  __device__ __forceinline__ void load(unsigned g, unsigned, unsigned lane, Raw& raw, u32x4 (&)[4][FM], unsigned (&)[FM]) const {
    with_reach<X>(static_cast<int>(g * 512 + 512), k, [&](auto how) {
#pragma unroll
      for (unsigned r = 0; r < ROWS; ++r)
        load8<decltype(how)::value>(x + static_cast<int64_t>(min(r, m - 1)) * stride, static_cast<int>(g * 512 + lane * 8), k,
                                    raw.w[r]);
    });
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

template <typename T, typename Source, int FM, int R, int U, int kWaves>
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
    auto load_x = [&](int u) { source.template load<FM, FULL>(g0 + u * kWaves, nq, lane, raw[u], x[u], sx[u]); };
    // Loads come back in order. Plain rows come first, to be quantised while the weights are on their way;
    // quantised ones, which are closer, after the weights: after their own group's if there are more than
    // 16, so that it multiplies while the next one's are on their way (8192 x 8192 weights: 32 rows 11.4 ->
    // 10.8 us, 64 rows 14.1 -> 13.0, but 16 rows 9.8 -> 10.1).
    constexpr bool kOwn = !Source::kFirst && FM > 1;
    if constexpr (Source::kFirst) {
#pragma unroll
      for (int u = 0; u < N; ++u) load_x(u);
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
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
      if constexpr (kOwn) {
        load_x(u);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (!Source::kFirst && !kOwn) {
#pragma unroll
      for (int u = 0; u < N; ++u) load_x(u);
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
void few_rows(Source source, const Operand& b, int64_t m, int64_t n, int64_t k, T* c, int64_t stride,
              hipStream_t s) {
  auto run = [&](auto kernel, int waves) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n + 16 * R - 1) / (16 * R))), dim3(64 * waves), 0, s, source,
                       b.codes, b.scales, static_cast<unsigned>(m), static_cast<unsigned>(n),
                       static_cast<unsigned>(mx_quads(k)), c, stride);
  };
  // no more waves than groups of quads
  if (mx_groups(k) <= 4) run(product_few_rows_kernel<T, Source, FM, R, 1, 4>, 4);
  else run(product_few_rows_kernel<T, Source, FM, R, U, 8>, 8);
}

// Compute units, asked for once a device (a multiple of eight: whole XCDs).
int compute_units(int dev) {
  static std::atomic<int> known[64];
  if (dev < 0 || dev >= 64) return device_cu_count(dev);
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    n = std::max(8, device_cu_count(dev) / 8 * 8);
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

constexpr int64_t kFewRows = 64;
constexpr int kComputeUnits = 256;  // what the choices between kernels are made for

// What the tile kernels take, in us, measured on MI355X (products of 2048 and 8192 elements along k, 128 to
// 2048 tiles): a stage (a quad of k) with at most half, or at most one, tile a compute unit; once some have
// two; a stage for each tile a compute unit where there are many; and what does not depend on k, alone
// and for each tile a compute unit.
struct TileCost {
  int m, n;
  bool whole_rounds;  // one tile a compute unit at a time
  double half, one, two, each, fixed, fixed_each;
};
constexpr TileCost kTiles[] = {
    {256, 256, true, 0.62, 0.81, 0, 0.82, 6, 5},   {256, 128, true, 0.35, 0.43, 0, 0.46, 8, 1.5},
    {128, 128, false, 0.22, 0.24, 0.37, 0.24, 6, 1}, {64, 128, false, 0.16, 0.19, 0.28, 0.15, 5.3, 0.5},
    {64, 64, false, 0.13, 0.13, 0.195, 0.098, 4.8, 0.5},
};
struct Plan {
  // tiles as in kTiles, then the most rows of the few-rows kernel, x2 with two row blocks of b a workgroup
  enum Shape { k256, k256x128, k128, k64x128, k64, kFew16, kFew32, kFew32x2, kFew64, kFew64x2 } shape;
  unsigned parts, per;  // of k, and groups of quads a part
  double us;
};
// `whole`: k in one piece. Every tile kernel then adds up a result's k in the same order.
Plan plan_tiles(const Job* jobs, int count, bool whole) {
  Plan best{Plan::k64, 1, 0, 1e30};
  const int64_t groups = count == 1 ? mx_groups(jobs[0].k) : 0;
  for (int shape = 0; shape < 5; ++shape) {
    const TileCost& c = kTiles[shape];
    int64_t total = 0;
    double stages = 0, longest = 0;
    for (int i = 0; i < count; ++i) {
      const int64_t t = (jobs[i].m + c.m - 1) / c.m * ((jobs[i].n + c.n - 1) / c.n);
      const double q = static_cast<double>(mx_groups(jobs[i].k)) * 4;
      total += t;
      stages += q * static_cast<double>(t);
      longest = std::max(longest, q);
    }
    stages /= static_cast<double>(total);
    auto us = [&](int64_t tiles, double len) {
      const double x = static_cast<double>(tiles) / kComputeUnits, rounds = std::ceil(x);
      const double stage = x <= 0.5 ? c.half : x <= 1 ? c.one : c.whole_rounds ? c.each * rounds : std::max(c.two, c.each * x);
      return c.fixed + c.fixed_each * (c.whole_rounds ? rounds : x) + len * stage;
    };
    const double one = us(total, total <= kComputeUnits ? longest : stages);
    if (one < best.us) best = {static_cast<Plan::Shape>(shape), 1, static_cast<unsigned>(groups), one};
    if (shape != Plan::k64 || whole || total >= kComputeUnits) continue;
    // k in parts: their sums, written and read, and a launch more
    for (int64_t parts = 2; parts <= 8 && parts * 2 <= groups; ++parts) {
      const int64_t per = (groups + parts - 1) / parts, some = (groups + per - 1) / per;
      const double t = us(total * some, static_cast<double>(per) * 4) + 3 + static_cast<double>(some * jobs[0].m * jobs[0].n) * 8 / 4e6;
      if (t < best.us) best = {Plan::k64, static_cast<unsigned>(some), static_cast<unsigned>(per), t};
    }
  }
  return best;
}
Plan plan(const Job& j) {
  const int64_t small = (j.m + 63) / 64 * ((j.n + 63) / 64);
  // few rows: the weights stream by (from the same measurements, 3.5 us and 5 TB/s, less with more rows)
  const bool narrow = j.n <= 16 * kComputeUnits;  // a row block a workgroup fills the chip better than two
  if (j.m <= 32 || (j.m <= kFewRows && small < 192))
    return {j.m <= 16   ? Plan::kFew16
            : j.m <= 32 ? narrow ? Plan::kFew32 : Plan::kFew32x2
            : narrow    ? Plan::kFew64
                        : Plan::kFew64x2, 1, static_cast<unsigned>(mx_groups(j.k)),
            3.5 + static_cast<double>(j.n) * static_cast<double>(mx_quads(j.k)) * 68 * (1 + static_cast<double>(j.m) / 64) / 5e6};
  return plan_tiles(&j, 1, false);
}
// Whether two products should take less in one launch, k whole, than one after the other.
bool together(const Job* jobs) { return plan_tiles(jobs, 2, true).us <= plan(jobs[0]).us + plan(jobs[1]).us; }

std::string name_of(const Plan& p) {
  const char* names[] = {"256x256", "256x128", "128x128", "64x128", "64x64", "few16", "few32", "few32x2", "few64", "few64x2"};
  return p.parts > 1 ? "64x64/" + std::to_string(p.parts) : names[p.shape];
}

void check_product(int64_t m, int64_t n, int64_t k, int64_t stride) {
  require(m >= 0 && n >= 0 && k >= 1, "mx: m and n must be >= 0 and k >= 1");
  require(mx_fits(m, k) && mx_fits(n, k) && ((m + 15) / 16) * ((n + 15) / 16) < (1ll << 28),
          "mx: a product's sizes are beyond its limits (mx.h)");
  require(stride >= n || m <= 1, "mx: stride must be at least n");
}

// Whether a linear layer's rows are quantised by the workgroups that multiply them, each for itself, or
// once by a launch before. The launch costs 2 to 3 us; on the way, each workgroup reads and quantises all of
// x: 400 KB of it a compute unit, over its workgroups one after the other, take about as long. In us, on the
// way and with the launch: bf16, 8 rows, 8192 x 8192 weights 9.5 and 11.5, 4096 x 28672 16.5 and 16.8, 28672 x
// 8192 25.0 and 25.6; f32, 4096 x 28672, 2 rows 14.7 and 16.9, 5 rows 20.2 and 16.9. Where it is wrong by most:
// two f32 rows on 28672 x 8192, which it takes on the way, 28.9 and 25.2.
enum class Way { launch, one, four, eight, eight_x2 };  // the launch before, or the most rows on the way
Way way_of(int64_t m, int64_t n, int64_t k, int size) {
  const int64_t blocks = (n + 15) / 16;
  // row blocks in hand at once: two workgroups a compute unit for up to four rows, else one of one or two
  const int64_t at_once = m > 4 && blocks <= kComputeUnits ? kComputeUnits : 2 * kComputeUnits;
  if (m > 8 || m * k * size * ((blocks + at_once - 1) / at_once) > 400000) return Way::launch;
  return m == 1 ? Way::one : m <= 4 ? Way::four : n <= 16 * kComputeUnits ? Way::eight : Way::eight_x2;
}

}  // namespace
}  // namespace mx

using namespace mx;

namespace mx {
namespace {

size_t workspace_of(const Plan& p, const Job& j) {
  return p.parts > 1 ? static_cast<size_t>(p.parts) * j.m * j.n * 4 : 0;
}

void check_job(const Job& j, Type t) {
  check_product(j.m, j.n, j.k, j.stride);
  if (j.m == 0 || j.n == 0) return;
  require(j.a.codes && j.a.scales && j.b.codes && j.b.scales && j.c, "mx_product: null pointer");
  require(aligned(j.a.codes, 16) && aligned(j.b.codes, 16) && aligned(j.a.scales, 16) && aligned(j.b.scales, 16) &&
              aligned(j.c, size_of(t)),
          "mx_product: codes and scales aligned to 16 bytes, the result to its type");
}

template <typename T, int FM, int FN, int WM, int WN, int RESIDENT, bool SPLIT = false>
void run_tiles(int dev, const Job* jobs, int count, const Plan& plan, hipStream_t s) {
  auto product = [&](const Job& j, bool any) {
    const unsigned rows = static_cast<unsigned>((j.m + 16 * FM * WM - 1) / (16 * FM * WM));
    const unsigned cols = static_cast<unsigned>((j.n + 16 * FN * WN - 1) / (16 * FN * WN));
    Tiles<8> tiles(rows, cols * plan.parts);
    if (!any) tiles.total = 0;
    return Product{j.a.codes, j.a.scales, j.b.codes, j.b.scales, j.c, j.stride, static_cast<unsigned>(j.m),
                   static_cast<unsigned>(j.n), static_cast<unsigned>(mx_quads(j.k)), plan.per, Div(cols), tiles};
  };
  const Products products{{product(jobs[0], true), product(jobs[count - 1], count > 1)}};
  const unsigned total = products.p[0].tiles.total + products.p[1].tiles.total;
  const unsigned grid = std::min((total + 7) / 8 * 8, static_cast<unsigned>(compute_units(dev) * RESIDENT));
  hipLaunchKernelGGL((product_tile_kernel<T, FM, FN, WM, WN, RESIDENT, SPLIT>), dim3(grid), dim3(64 * WM * WN), 0, s,
                     products);
}

// One product, or two in one launch.
void run_jobs(int dev, Job* jobs, int count, const Plan& p, Type t, void* workspace, hipStream_t s) {
  with_type(t, [&](auto e) {
    using T = decltype(e);
    Job& j = jobs[0];
    auto rows = [&] {
      return QuantizedRows{j.a.codes, j.a.scales, static_cast<unsigned>(mx_quads(j.k)),
                           static_cast<unsigned>(mx_groups(j.k)), static_cast<unsigned>(mx_row_blocks(j.m))};
    };
    switch (p.shape) {
      case Plan::kFew16: few_rows<T, 1, 1, 2>(rows(), j.b, j.m, j.n, j.k, static_cast<T*>(j.c), j.stride, s); break;
      case Plan::kFew32: few_rows<T, 2, 1, 2>(rows(), j.b, j.m, j.n, j.k, static_cast<T*>(j.c), j.stride, s); break;
      case Plan::kFew32x2: few_rows<T, 2, 2, 2>(rows(), j.b, j.m, j.n, j.k, static_cast<T*>(j.c), j.stride, s); break;
      case Plan::kFew64: few_rows<T, 4, 1, 1>(rows(), j.b, j.m, j.n, j.k, static_cast<T*>(j.c), j.stride, s); break;
      case Plan::kFew64x2: few_rows<T, 4, 2, 2>(rows(), j.b, j.m, j.n, j.k, static_cast<T*>(j.c), j.stride, s); break;
      case Plan::k256: run_tiles<T, 8, 4, 2, 4, 1>(dev, jobs, count, p, s); break;
      case Plan::k256x128: run_tiles<T, 4, 4, 4, 2, 1>(dev, jobs, count, p, s); break;
      case Plan::k128: run_tiles<T, 4, 4, 2, 2, 2>(dev, jobs, count, p, s); break;
      case Plan::k64x128: run_tiles<T, 2, 4, 2, 2, 2>(dev, jobs, count, p, s); break;
      case Plan::k64:
        if (p.parts == 1) {
          run_tiles<T, 2, 2, 2, 2, 3>(dev, jobs, count, p, s);
        } else {
          auto out = static_cast<T*>(j.c);
          const int64_t stride = j.stride;
          j.c = workspace, j.stride = j.n;
          run_tiles<float, 2, 2, 2, 2, 3, true>(dev, jobs, 1, p, s);
          const unsigned quarters = static_cast<unsigned>((j.n + 3) / 4);
          hipLaunchKernelGGL(product_sum_kernel<T>, dim3(static_cast<unsigned>((j.m * quarters + 255) / 256)), dim3(256), 0,
                             s, static_cast<const float*>(workspace), p.parts, static_cast<unsigned>(j.m),
                             static_cast<unsigned>(j.n), out, stride, Div(quarters));
        }
        break;
    }
  });
}

}  // namespace

// One product, or two of one result type in one launch (neither empty). `whole`: k in one piece, as two
// always have it.
void launch_products(int dev, const Job* jobs, int count, bool whole, Type t, void* workspace, size_t workspace_bytes,
                     hipStream_t s) {
  for (int i = 0; i < count; ++i) check_job(jobs[i], t);
  if (jobs[0].m == 0 || jobs[0].n == 0) return;
  const Plan p = count == 2 || whole ? plan_tiles(jobs, count, true) : plan(jobs[0]);
  const size_t need = workspace_of(p, jobs[0]);
  require(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
          "mx_product: needs a workspace of mx_product_workspace bytes, aligned to 16");
  OnDevice on(dev);
  Job todo[2] = {jobs[0], jobs[count - 1]};
  run_jobs(dev, todo, count, p, t, workspace, s);
  check(hipGetLastError(), "mx_product");
}

}  // namespace mx

size_t mx_product_workspace(int64_t m, int64_t n, int64_t k) {
  check_product(m, n, k, n);
  const Job j{{}, {}, m, n, k, nullptr, n};
  return workspace_of(plan(j), j);
}

std::string mx_product_kernel(int64_t m, int64_t n, int64_t k) {
  check_product(m, n, k, n);
  return name_of(plan(Job{{}, {}, m, n, k, nullptr, n}));
}

void launch_mx_product(int dev, const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales,
                       int64_t m, int64_t n, int64_t k, void* c, const std::string& dtype, int64_t stride,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const Type t = type_of(dtype, "mx_product: dtype must be bf16|f16|f32");
  const Job j{operand(a_codes, a_scales), operand(b_codes, b_scales), m, n, k, c, stride};
  launch_products(dev, &j, 1, false, t, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

size_t mx_linear_workspace(int64_t m, int64_t n, int64_t k, const std::string& dtype) {
  check_product(m, n, k, n);
  if (way_of(m, n, k, size_of(type_of(dtype, "mx_linear: dtype must be bf16|f16|f32"))) != Way::launch) return 0;
  return mx_bytes(m, k) + mx_product_workspace(m, n, k);
}

std::string mx_linear_kernel(int64_t m, int64_t n, int64_t k, const std::string& dtype) {
  check_product(m, n, k, n);
  const char* names[] = {"", "way1", "way4", "way8", "way8x2"};
  const Way way = way_of(m, n, k, size_of(type_of(dtype, "mx_linear: dtype must be bf16|f16|f32")));
  return way == Way::launch ? mx_product_kernel(m, n, k) : names[static_cast<int>(way)];
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
  const Way way = way_of(m, n, k, size_of(t));
  if (way != Way::launch) {
    OnDevice on(dev);
    auto s = static_cast<hipStream_t>(stream);
    const Operand w = operand(w_codes, w_scales);
    with_type(t, [&](auto e) {
      using T = decltype(e);
      auto px = static_cast<const T*>(x);
      auto out = static_cast<T*>(y);
      const auto rows = static_cast<unsigned>(m);
      const int len = static_cast<int>(k);
      if (way == Way::one) few_rows<T, 1, 1, 2>(PlainRows<T, 1>{px, x_stride, rows, len}, w, m, n, k, out, y_stride, s);
      else if (way == Way::four) few_rows<T, 1, 1, 2>(PlainRows<T, 4>{px, x_stride, rows, len}, w, m, n, k, out, y_stride, s);
      else if (way == Way::eight) few_rows<T, 1, 1, 1>(PlainRows<T, 8>{px, x_stride, rows, len}, w, m, n, k, out, y_stride, s);
      else few_rows<T, 1, 2, 1>(PlainRows<T, 8>{px, x_stride, rows, len}, w, m, n, k, out, y_stride, s);
    });
    check(hipGetLastError(), "mx_linear");
    return;
  }
  require(workspace && workspace_bytes >= mx_linear_workspace(m, n, k, dtype), "mx_linear: workspace too small");
  require(aligned(workspace, 16), "mx_linear: workspace aligned to 16 bytes");
  auto codes = static_cast<char*>(workspace);
  auto scales = codes + mx_codes_bytes(m, k);
  launch_mx_quantize(dev, x, dtype, m, k, x_stride, false, codes, scales, stream);
  launch_mx_product(dev, codes, scales, w_codes, w_scales, m, n, k, y, dtype, y_stride, codes + mx_bytes(m, k),
                    workspace_bytes - mx_bytes(m, k), stream);
}

// ---- training step -------------------------------------------------------------------------------
// saved: x and w down their columns (rows k, along m and along n). Workspaces: what else is quantised,
// then the products'.
size_t mx_linear_train_saved(int64_t m, int64_t n, int64_t k) {
  check_product(m, n, k, n);
  return mx_bytes(k, m) + mx_bytes(k, n);
}
size_t mx_linear_train_workspace(int64_t m, int64_t n, int64_t k) {
  return mx_bytes(m, k) + mx_bytes(n, k) + mx_product_workspace(m, n, k);
}

void launch_mx_linear_train(int dev, const void* x, const std::string& dtype, int64_t x_stride, const void* w,
                            const std::string& w_dtype, int64_t w_stride, int64_t m, int64_t n, int64_t k, void* y,
                            int64_t y_stride, void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes,
                            void* stream) {
  const Type t = type_of(dtype, "mx_linear_train: dtype must be bf16|f16|f32");
  require(m >= 1 && n >= 1, "mx_linear_train: m and n must be >= 1");
  check_product(m, n, k, y_stride);
  require(saved && saved_bytes >= mx_linear_train_saved(m, n, k) && aligned(saved, 16) && workspace &&
              workspace_bytes >= mx_linear_train_workspace(m, n, k) && aligned(workspace, 16),
          "mx_linear_train: saved and workspace of their sizes, aligned to 16 bytes");
  auto kept = static_cast<char*>(saved), ws = static_cast<char*>(workspace);
  const Quantized xq{ws, m, k}, wq{ws + mx_bytes(m, k), n, k}, xt{kept, k, m}, wt{kept + mx_bytes(k, m), k, n};
  const Source sources[2] = {{x, x_stride, m, k, xq.at, xt.at}, {w, w_stride, n, k, wq.at, wt.at}};
  const Job j{xq.operand(), wq.operand(), m, n, k, y, y_stride};
  check_job(j, t);
  auto s = static_cast<hipStream_t>(stream);
  const Type tw = type_of(w_dtype, "mx_linear_train: w_dtype must be bf16|f16|f32");
  check_source(sources[0], t);
  check_source(sources[1], tw);
  if (t == tw) {
    launch_quantize_both(dev, sources, 2, t, s);
  } else {
    launch_quantize_both(dev, sources, 1, t, s);
    launch_quantize_both(dev, sources + 1, 1, tw, s);
  }
  const size_t used = static_cast<size_t>(mx_bytes(m, k) + mx_bytes(n, k));
  launch_products(dev, &j, 1, false, t, ws + used, workspace_bytes - used, s);
}

size_t mx_linear_grad_workspace(int64_t m, int64_t n, int64_t k) {
  check_product(m, n, k, n);
  return mx_bytes(m, n) + mx_bytes(n, m) + std::max(mx_product_workspace(m, k, n), mx_product_workspace(n, k, m));
}

std::string mx_linear_grad_kernel(int64_t m, int64_t n, int64_t k) {
  check_product(m, n, k, n);
  require(m >= 1 && n >= 1, "mx_linear_grad: m and n must be >= 1");
  const Job jobs[2] = {{{}, {}, m, k, n, nullptr, k}, {{}, {}, n, k, m, nullptr, k}};
  return together(jobs) ? name_of(plan_tiles(jobs, 2, true)) : "";
}

void launch_mx_linear_grad(int dev, const void* dy, const std::string& dtype, int64_t dy_stride, const void* saved,
                           int64_t m, int64_t n, int64_t k, void* dx, int64_t dx_stride, void* dw,
                           const std::string& w_dtype, int64_t dw_stride, void* workspace, size_t workspace_bytes,
                           void* stream) {
  const Type t = type_of(dtype, "mx_linear_grad: dtype must be bf16|f16|f32");
  const Type tw = type_of(w_dtype, "mx_linear_grad: w_dtype must be bf16|f16|f32");
  require(m >= 1 && n >= 1, "mx_linear_grad: m and n must be >= 1");
  check_product(m, k, n, dx ? dx_stride : k);
  check_product(n, k, m, dw ? dw_stride : k);
  require(saved && aligned(saved, 16) && workspace && workspace_bytes >= mx_linear_grad_workspace(m, n, k) &&
              aligned(workspace, 16),
          "mx_linear_grad: saved and workspace of their sizes, aligned to 16 bytes");
  auto kept = static_cast<char*>(const_cast<void*>(saved)), ws = static_cast<char*>(workspace);
  const Quantized along{ws, m, n}, down{ws + mx_bytes(m, n), n, m}, xt{kept, k, m}, wt{kept + mx_bytes(k, m), k, n};
  const Source source{dy, dy_stride, m, n, along.at, down.at};
  check_source(source, t);
  const Job jobs[2] = {{along.operand(), wt.operand(), m, k, n, dx, dx_stride}, {down.operand(), xt.operand(), n, k, m, dw, dw_stride}};
  if (dx) check_job(jobs[0], t);
  if (dw) check_job(jobs[1], tw);
  auto s = static_cast<hipStream_t>(stream);
  const size_t used = static_cast<size_t>(mx_bytes(m, n) + mx_bytes(n, m));
  // What is chosen for both holds for one alone too: a gradient's bits do not depend on what else is asked for.
  // It costs one alone that would have taken fewer stages up to 4 us (dx of 20 rows on 4096 x 4096 8.3 -> 12.3).
  const bool both = t == tw && together(jobs);
  auto products = [&](const Job* j, int count, Type type) {
    launch_products(dev, j, count, both, type, ws + used, workspace_bytes - used, s);
  };
  if (dx && dw) launch_quantize_both(dev, &source, 1, t, s);
  else if (dx) launch_mx_quantize(dev, dy, dtype, m, n, dy_stride, false, along.at, along.scales(), stream);
  else if (dw) launch_mx_quantize(dev, dy, dtype, m, n, dy_stride, true, down.at, down.scales(), stream);
  if (dx && dw && both) {
    products(jobs, 2, t);
  } else {
    if (dx) products(jobs, 1, t);
    if (dw) products(jobs + 1, 1, tw);
  }
}

}  // namespace gpumon_hip
