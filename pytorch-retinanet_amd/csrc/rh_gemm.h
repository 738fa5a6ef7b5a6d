// Matrix-product core of the classifier loss (gfx950): C[m][n] = sum_k A(m,k) B(n,k) on the matrix
// units, operands staged to LDS by direct loads through a ring of four stages.
//
// An operand comes in one of two layouts, so that the loss's three products need no transposed
// copies:   kRows  element (i,k) at  base + i*ld + k   (the sum runs along a row)
//           kCols  element (i,k) at  base + k*ld + i   (the sum runs down a column)
// Both are staged as they lie in memory.  A kRows tile holds 64 bytes of k per row and its 16-byte
// fragments are read as they are; a kCols tile is read with the transposing LDS load.
//
// float operands are taken apart into three bfloat16 numbers, x = x0 + x1 + x2, each the nearest to what
// is left: |x1| <= 2^-9 |x|, |x2| <= 2^-18 |x|, exact but for what lies below bfloat16's range.  Of the nine
// products of two of them the six of 2^-18 and up are summed, smallest first; the rest is below 2^-26 of
// the product, a quarter of what one float32 rounding of it would be.  Six bfloat16 instructions do what
// eight of float32 (32x32x2) do at a quarter of their time each.
//
// What this library lays out itself (the features, P) it lays out in panels of 64 bytes of columns, the
// rows of a panel one after the other: the tiles of either layout are then runs of whole kilobytes.
//
// Every global read goes through a buffer descriptor whose record count ends at the operand's last
// valid element: what a tile reaches beyond it reads as zero and touches no memory.
#pragma once
#include "rh_common.h"

namespace rh {
namespace gemm {

#define RH_LDS __attribute__((address_space(3)))

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

enum Layout { kRows = 0, kCols = 1 };
constexpr bool kPlain = false, kPanels = true;

// 64 bytes of k per tile step: 32 values, two halves (kk) of the matrix instructions' depth each.  A panel
// has as many columns.
constexpr int kStepBytes = 64;
constexpr int kStepK = 32;
constexpr int kRing = 4;

template <typename T>
struct TypeOf;
template <>
struct TypeOf<float> {
  typedef __bf16 Part;      // what the matrix units are given
  static constexpr int kParts = 3, kTerms = 6;
  static constexpr unsigned kOrderA = 0x010120, kOrderB = 0x001102;      // term t: parts (nibble t) of a and b
  static __device__ __forceinline__ float to_float(float v) { return v; }
  static __device__ __forceinline__ float from_float(float v) { return v; }
};
template <>
struct TypeOf<__bf16> {
  typedef __bf16 Part;
  static constexpr int kParts = 1, kTerms = 1;
  static constexpr unsigned kOrderA = 0, kOrderB = 0;
  static __device__ __forceinline__ f32x16 mma(const u32x4 a, const u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 from_float(float v) { return (__bf16)v; }
};
template <>
struct TypeOf<_Float16> {
  typedef _Float16 Part;
  static constexpr int kParts = 1, kTerms = 1;
  static constexpr unsigned kOrderA = 0, kOrderB = 0;
  static __device__ __forceinline__ f32x16 mma(const u32x4 a, const u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from_float(float v) { return (_Float16)v; }
};

// A lane of the lower half of the wave has four values of each of two groups of eight, x of the first
// and y of the second (as 8 bytes), its partner 32 lanes on the other four: afterwards the lower lane
// has the first group whole, the upper one the second.
__device__ __forceinline__ u32x4 whole_group(const unsigned long long x, const unsigned long long y) {
  const auto lo = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)y, false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap((unsigned)(x >> 32), (unsigned)(y >> 32), false, false);
  return u32x4{lo[0], hi[0], lo[1], hi[1]};
}

template <typename T>
struct Vec4 {
  T v[4];
} __attribute__((aligned(4 * sizeof(T))));

// Workgroups of neighbouring numbers land on different XCDs: number `id` of `total` -> the tile
// number that gives each of the eight XCDs a contiguous run of tiles.
__device__ __forceinline__ int xcd_run(const int id, const int total) {
  const int per = total >> 3, rest = total & 7, x = id & 7, at = id >> 3;
  return x * per + min(x, rest) + at;
}

constexpr unsigned kMostBytes = 0xffffff00u;
constexpr int kNowhere = (int)0xffffff80u;      // an offset no descriptor reaches: reads as zero

// One operand's descriptor: `bytes` readable from base on.
__device__ __forceinline__ u32x4 make_rsrc(const char* base, const long long bytes) {
  const unsigned long long at = (unsigned long long)base;
  const unsigned low = (unsigned)bytes, high = (unsigned)((unsigned long long)bytes >> 32);
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((unsigned)at);
  r[1] = __builtin_amdgcn_readfirstlane((unsigned)(at >> 32));      // 47 bits of address, no stride
  r[2] = __builtin_amdgcn_readfirstlane(high ? kMostBytes : min(low, kMostBytes));
  r[3] = 0x00020000u;
  return r;
}

// 16 bytes per lane from the buffer to LDS, lane after lane from `lds` on.  Written out, because
// the compiler waits for every such load of its own before any LDS read; here stage_wait() does.
template <int kAt>
__device__ __forceinline__ void load_to_lds(const u32x4 rsrc, const unsigned lds, const int offset) {
  [[maybe_unused]] unsigned m0;      // an output, so that the compiler keeps nothing of its own there
  asm volatile("s_add_u32 m0, %1, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
               : "={m0}"(m0)
               : "s"(lds), "v"(offset), "s"(rsrc), "n"(kAt)
               : "memory", "scc");
}
// All but this wave's latest kLeft loads have landed and its LDS reads have returned; then every wave's.
template <int kLeft>
__device__ __forceinline__ void stage_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
}

template <int k>
struct Int {
  static constexpr int value = k;
};
template <int kN, int kI = 0, typename F>
__device__ __forceinline__ void each(const F f) {      // f(Int<0>) .. f(Int<kN - 1>)
  if constexpr (kI < kN) {
    f(Int<kI>());
    each<kN, kI + 1>(f);
  }
}

// Moves one stage of an operand's tile (kR rows or columns of the result, kStepBytes of k) to LDS.  The
// steps go through k once for every term, through the part of the operand that kOrder names for it.
template <Layout kL, bool kPaneled, int kR, int kThreads, int kTerms, unsigned kOrder>
struct Loader {
  static constexpr int kOps = kR * kStepBytes / (kThreads * 16);
  static constexpr int kRowBytes = kL == kRows ? kStepBytes : kR * 2;
  static constexpr int kChunks = kRowBytes / 16;             // 16-byte chunks of a staged row
  static constexpr int kRowsPerOp = kThreads / kChunks;      // staged rows one pass of all threads covers
  int offset[kOps];       // this lane's byte offsets from the tile's first element
  const char* base;       // of the coming step
  long long left;         // bytes readable from base on
  long long step;         // bytes from one step to the next
  const char* origin;
  long long bytes, part;
  int steps, at, term;

  static __device__ __forceinline__ int row_of(const int i) { return i * kRowsPerOp + (int)threadIdx.x / kChunks; }
  static __device__ __forceinline__ int chunk_of(const int i) {
    const int row = row_of(i), at = (int)threadIdx.x % kChunks;
    return kL == kRows ? at ^ ((row >> 2) & 3) : at ^ ((row & 3) << 2);    // kCols: 32-byte blocks, block ^ 2*(k & 3)
  }
  __device__ __forceinline__ void to_term() {
    const long long off = (kOrder >> (4 * term) & 15) * part;
    base = origin + off;
    left = bytes;
    at = 0;
  }
  // from: first element of the tile at k = 0; stride: bytes from row to row, or from panel to panel;
  // readable: bytes from `from` on, in each part; parts: bytes from part to part; n: steps of a term.
  __device__ __forceinline__ void init(const void* from, long long stride, long long readable, long long parts,
                                       int n) {
    origin = (const char*)from;
    bytes = readable;
    part = parts;
    steps = n;
    term = 0;
    to_term();
    if (kPaneled) step = kL == kRows ? stride : kStepK * kStepBytes;
    else step = kL == kRows ? kStepBytes : kStepK * stride;
#pragma unroll
    for (int i = 0; i < kOps; ++i) {
      const int row = row_of(i), chunk = chunk_of(i);
      if (!kPaneled) offset[i] = (int)(row * stride) + chunk * 16;
      else if (kL == kRows) offset[i] = row * kStepBytes + chunk * 16;
      else offset[i] = (int)((chunk >> 2) * stride) + row * kStepBytes + (chunk & 3) * 16;
    }
  }
  // A step's loads: plan() works out the descriptor of the coming one, begin() makes it the one that
  // load() takes.  A step that is not `there` reads zeros and touches no memory.  limit: bytes (kRows) or
  // values (kCols) of its k that belong to the operand, the others read as zero.
  u32x4 rsrc, coming;
  unsigned to;
  int limit;
  __device__ __forceinline__ void plan(const bool there) {
    coming = make_rsrc(base, there ? left : 0);
    // a lane instruction may have written these registers: a memory instruction that takes them has to
    // stay five cycles behind, which nobody else sees to for the written-out ones
    asm volatile("s_nop 4" : "+s"(coming));
    base += step;
    left -= step;
    if (kTerms > 1 && ++at == steps) {
      ++term;
      to_term();
    }
  }
  __device__ __forceinline__ void begin(const unsigned stage, const int k_limit) {
    rsrc = coming;
    to = stage;
    limit = k_limit;
  }
  template <bool kTail, int i>
  __device__ __forceinline__ void load() const {
    const bool in = !kTail || (kL == kRows ? chunk_of(i) * 16 < limit : row_of(i) < limit);
    load_to_lds<i * kThreads * 16>(rsrc, to, in ? offset[i] : kNowhere);
  }
};

// Reads the matrix instructions' fragments of one wave from a staged tile.  `first`: the wave's
// first row / column of the tile (a multiple of 32); fragment f covers 32 from first + 32 f on.
template <Layout kL, int kR, int kF>
struct Fragments {
  static constexpr int kRowBytes = kR * 2;      // kCols only
  static constexpr int kAddr = kL == kRows ? 2 : kF;
  int addr[kAddr];
  __device__ __forceinline__ void init(const int first) {
    const int l = (int)threadIdx.x & 63;
    if (kL == kRows) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
        addr[kk] = (first + (l & 31)) * kStepBytes + (((2 * kk + (l >> 5)) ^ ((l >> 2) & 3)) << 4);
    } else {
      const int q = (l >> 2) & 3;
#pragma unroll
      for (int f = 0; f < kAddr; ++f)
        addr[f] = (8 * (l >> 5) + q) * kRowBytes + (((first / 32 + f) ^ q) << 6) + ((l >> 4) & 1) * 32 +
                  (l & 3) * 8;
    }
  }
  __device__ __forceinline__ u32x4 read(const RH_LDS char* stage, const int f, const int kk) const {
    if constexpr (kL == kRows) {
      return *(const RH_LDS u32x4*)(stage + addr[kk] + f * 32 * kStepBytes);
    } else {
      union {
        bf16x4 h[2];
        u32x4 u;
      } r;
      const RH_LDS char* p = stage + addr[f] + kk * 16 * kRowBytes;
      r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((RH_LDS bf16x4*)p);
      r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((RH_LDS bf16x4*)(p + 4 * kRowBytes));
      return r.u;
    }
  }
};

// A workgroup's tile: kWM x kWN waves, each kFM x kFN fragments of 32 x 32.
template <int kWM_, int kWN_, int kFM_, int kFN_>
struct Shape {
  static constexpr int kWM = kWM_, kWN = kWN_, kFM = kFM_, kFN = kFN_;
  static constexpr int kBM = kWM * kFM * 32, kBN = kWN * kFN * 32;
  static constexpr int kThreads = kWM * kWN * 64;
  static constexpr int kStage = (kBM + kBN) * kStepBytes;
  static constexpr int kLdsBytes = kRing * kStage;
};

// acc[i][j][r]: result row m = 32 i + lane % 32 and column n = 32 j + 8 (r / 4) + 4 (lane / 32) + r % 4
// of the wave's part: a lane owns rows, four neighbouring columns at a time.
template <typename T, Layout kLA, bool kPA, Layout kLB, bool kPB, typename S>
struct Tile {
  typedef TypeOf<T> Type;
  typedef Loader<kLA, kPA, S::kBM, S::kThreads, Type::kTerms, Type::kOrderA> LoaderA;
  typedef Loader<kLB, kPB, S::kBN, S::kThreads, Type::kTerms, Type::kOrderB> LoaderB;
  f32x16 acc[S::kFM][S::kFN];

  // a / b: first elements of the tile's operands at the first k; lda, ldb: bytes from row to row or from
  // panel to panel; *_bytes: readable from there; *_part: bytes from one part of the numbers to the next
  // (float); steps: k steps (of kStepK values); a_limit, b_limit: how much of the last one is the operand's
  // (kCols: values; plain kRows: bytes of a row).
  //
  // Fragments are read one half step ahead of the instructions that take them, and the loads of a
  // stage are spread over the step that frees its place in the ring, nearly three steps before it is
  // read.  8192 x 4096 x 16384 in bfloat16, uniform values: two stages of twice the depth, their loads in one
  // burst, 1.04-1.10 PFLOP/s; this 1.12-1.16 (1.6-1.7 on zeros, where the clock stays at 2.4 GHz; here it is below 1.8).
  __device__ __forceinline__ void run(const void* a, long long lda, long long a_bytes, long long a_part,
                                      const void* b, long long ldb, long long b_bytes, long long b_part,
                                      const int steps_of_k, RH_LDS char* lds, const int a_limit = kStepBytes,
                                      const int b_limit = kStepBytes) {
    LoaderA la;
    LoaderB lb;
    Fragments<kLA, S::kBM, S::kFM> fa;
    Fragments<kLB, S::kBN, S::kFN> fb;
    const int steps = steps_of_k * Type::kTerms;
    constexpr int kOffB = S::kBM * kStepBytes;
    const int wave = (int)threadIdx.x >> 6;
    la.init(a, lda, a_bytes, a_part, steps_of_k);
    lb.init(b, ldb, b_bytes, b_part, steps_of_k);
    fa.init((wave / S::kWN) * S::kFM * 32);
    fb.init((wave % S::kWN) * S::kFN * 32);
#pragma unroll
    for (int i = 0; i < S::kFM; ++i)
#pragma unroll
      for (int j = 0; j < S::kFN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    if (steps <= 0) return;
    // where k ends inside the last step: the rows of a plain kRows operand do, and kCols ones (panels are
    // padded in k along the row)
    constexpr bool kTailA = kLA == kCols, kTailB = kLB == kCols || !kPB;
    constexpr int kFull = kStepBytes;      // more than either kind of limit needs
    constexpr int kOpsA = LoaderA::kOps;
    constexpr int kOpsB = LoaderB::kOps;
    static_assert(kOpsA == kOpsB, "both operands' tiles are of one size");
    // where this wave's loads of a stage go
    const unsigned to = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds + wave * 1024);
    auto plan = [&](const int s) {
      la.plan(s < steps);
      lb.plan(s < steps);
    };
    int last = steps_of_k - 1;      // the step that ends the running term
    auto begin = [&](const int s) {      // step s's loads, to its place in the ring
      const unsigned stage = to + (s & (kRing - 1)) * S::kStage;
      la.begin(stage, s == last ? a_limit : kFull);
      lb.begin(stage + kOffB, s == last ? b_limit : kFull);
      if (Type::kTerms > 1 && s == last) last += steps_of_k;
    };
    auto load_a = [&](auto i) { la.template load<kTailA, decltype(i)::value>(); };
    auto load_b = [&](auto i) { lb.template load<kTailB, decltype(i)::value>(); };
#pragma unroll
    for (int s = 0; s < kRing; ++s) {
      plan(s);
      begin(s);
      each<kOpsA>(load_a);
      if (s < kRing - 1) each<kOpsB>(load_b);      // the last one's follow in the loop
    }
    stage_wait<(kRing - 1) * (kOpsA + kOpsB) - kOpsB>();
    u32x4 x[2][S::kFM], y[2][S::kFN];
    constexpr int kSlots = S::kFM * S::kFN, kFragments = S::kFM + S::kFN;
    // Fragment f of a quarter, in the order the products take them: y0 x0 y1 .. yn x1 .. xm.
    auto read = [&](const int to, const RH_LDS char* stage, const int kk, const int f) {
      if (f == 0) y[to][0] = fb.read(stage + kOffB, 0, kk);
      else if (f == 1) x[to][0] = fa.read(stage, 0, kk);
      else if (f <= S::kFN) y[to][f - 1] = fb.read(stage + kOffB, f - 1, kk);
      else x[to][f - S::kFN] = fa.read(stage, f - S::kFN, kk);
    };
    // A half step's products, with what comes next issued between them: while one instruction runs on
    // the matrix unit (32 cycles) the wave has time for about seven others.
    auto half_step = [&](auto from, const RH_LDS char* stage, auto kk, auto load, auto beside) {
      constexpr int kFrom = decltype(from)::value;
      each<kSlots>([&](auto slot) {
        constexpr int t = decltype(slot)::value;
        acc[t / S::kFN][t % S::kFN] =
            TypeOf<typename Type::Part>::mma(y[kFrom][t % S::kFN], x[kFrom][t / S::kFN], acc[t / S::kFN][t % S::kFN]);
        if constexpr (t < kFragments) read(kFrom ^ 1, stage, decltype(kk)::value, t);
        if constexpr (t * kOpsA % kSlots == 0) load(Int<t * kOpsA / kSlots>());
        else if constexpr (t == kSlots / 2 + 1) beside();
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    static_assert(kSlots >= kFragments && kSlots % kOpsA == 0, "a fragment, and at most one load, a product");
#pragma unroll
    for (int f = 0; f < kFragments; ++f) read(0, lds, 0, f);
    for (int s = 0; s < steps; ++s) {
      const RH_LDS char* const here = lds + (s & (kRing - 1)) * S::kStage;
      const RH_LDS char* const next = lds + ((s + 1) & (kRing - 1)) * S::kStage;
      half_step(Int<0>(), here, Int<1>(), load_b, [&] { plan(s + kRing); });
      stage_wait<(kRing - 2) * (kOpsA + kOpsB)>();      // step s is read out, step s + 1 has landed
      begin(s + kRing);
      half_step(Int<1>(), next, Int<0>(), load_a, [] {});
    }
    stage_wait<0>();      // LDS is the caller's again
  }
};

}  // namespace gemm
}  // namespace rh
