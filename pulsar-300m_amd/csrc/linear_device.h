// Device side of the products with epilogues, shared by their kernels: operand staging, matrix
// core fragments, tile placement, epilogues.
#pragma once

#include <type_traits>

#include "linear.h"

namespace pulsar {

namespace {

constexpr int kXcds = 8;  // consecutive workgroups go to the 8 XCDs in turn

// Operand chunks that lie outside a matrix (past the last k, outside a group, rows an index
// does not name) are loaded from here: both factors of a product past the end are then zero,
// whatever the memory beside the matrix holds.
__device__ __attribute__((aligned(16))) const uint4 kZeroChunk = {0u, 0u, 0u, 0u};

// The LDS address of shared memory, and 16 bytes per lane from global memory straight to it
// (load_lds16 with the address in hand: a wave's lanes land 16 bytes apart).
__device__ __forceinline__ uint32_t lds_address(const void* shared) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_vptr) const_cast<void*>(shared)));
}
__device__ __forceinline__ void load_lds16_at(const void* g, uint32_t lds) {
  // one wait state between the M0 write and the load that reads it
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(g)
               : "memory", "m0");
}

// A workgroup of WR x WC waves owns a tile of BM = 16 RT WR rows and BN = 16 CT WC columns;
// wave (wr, wc) computes RT x CT matrix-core tiles of 16 x 16.
// WPS: workgroups that share a CU.
template <int RT_, int CT_, int WR_, int WC_, int WPS_>
struct LinShape {
  static constexpr int RT = RT_, CT = CT_, WR = WR_, WC = WC_, WPS = WPS_;
  static constexpr int kThreads = 64 * WR * WC;
  static constexpr int BM = 16 * RT * WR, BN = 16 * CT * WC;
  static constexpr bool kShared = kThreads == 512;  // one workgroup a CU
};

// How a fragment's lane index i (0..15) of tile t maps to the row of the operand's LDS tile.
//   PLAIN: 16 t + i.
//   WIDE (bf16, k contiguous): tiles in pairs, 32 (t / 2) + 8 (i / 4) + 4 (t % 2) + i % 4, so
//     that a lane ends with 8 consecutive columns of C in the pair's accumulators.
//   BLOCK (fp32, k strided): B = 4 or 2 tiles share each LDS read, 16 B (t / B) + B i + t % B.
enum Map { PLAIN, WIDE, BLOCK };

// Stages one operand's tile of R rows x 128 bytes of k (64 bf16 or 32 fp32) in LDS. Operands
// come in whole chunks of 16 bytes, aligned (others are copied so first).
//   KC (k contiguous in memory): LDS [R][8] chunks of 16 bytes; chunk c of row r sits at
//     c ^ key(r), which spreads the 16 rows a fragment read takes over the banks.
//   otherwise (rows of R contiguous elements per k): LDS [k][R]. bf16 tiles are read through
//     the LDS transpose load, 4 k rows x 32 bytes per 16 lanes, 32 lanes at once: 32-byte
//     pairs of chunks sit at pair ^ pair_key(k), which puts those 8 rows (k .. k + 3 and k + 8
//     .. k + 11) on different banks of the 64. ROWS: k row r is stored row
//     k_rows[r].
__device__ __forceinline__ int pair_key(int k) { return (k & 3) | ((k >> 3 & 1) << 2); }
template <typename T, int R, bool KC, Map MAP, int THREADS, bool ROWS = false>
struct Operand {
  static constexpr int EV = 16 / (int)sizeof(T), BK = 128 / (int)sizeof(T);
  static constexpr int kChunks = R * 8, NCH = kChunks / THREADS;
  static_assert(kChunks % THREADS == 0, "whole chunks per thread");
  static_assert(KC ? (THREADS / 8) % 16 == 0 : sizeof(T) == 4 || ((THREADS * EV / R) % 16 == 0 && R >= 128),
                "one swizzle key per thread, eight pairs a row");

  const T* base[KC ? NCH : 1];
  int64_t ld;             // !KC: elements from k to k + 1
  const int32_t* k_rows;  // ROWS: stored row of each k
  int64_t k_nrows;
  uint32_t ok;            // KC: rows that exist
  int off;                // KC: first k of this thread's chunks; else: its first k row
  bool valid;             // !KC: this thread's chunk columns lie inside the matrix
  int index;              // ROWS: the lane's row of the step to be loaded next

  __device__ __forceinline__ static int key(int r) {
    if constexpr (MAP == WIDE) return (r & 3) | ((r >> 3 & 1) << 2);
    return r & 7;
  }
  // KC: row(local) -> pointer to the stored row, or nullptr
  template <typename F>
  __device__ __forceinline__ void init_kc(F&& row) {
    const int r0 = (int)threadIdx.x >> 3;
    off = (((int)threadIdx.x & 7) ^ key(r0)) * EV;
    ok = 0;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      base[i] = row(r0 + i * (THREADS / 8));
      ok |= (base[i] ? 1u : 0u) << i;
    }
  }
  // !KC: col(local) -> stored column of the first element, and the columns' end in `lim`
  template <typename F>
  __device__ __forceinline__ void init_nc(const T* p, int64_t ld_, const int32_t* rows,
                                          int64_t nrows, F&& col) {
    const int c = (int)threadIdx.x % (R / EV);
    off = (int)threadIdx.x / (R / EV);
    int lc = c;
    if constexpr (sizeof(T) == 2) lc = (((c >> 1) ^ pair_key(off)) << 1) | (c & 1);
    int lim;
    const int g = col(lc * EV, lim);
    valid = g < lim;
    base[0] = p + (valid ? g : 0);
    ld = ld_;
    k_rows = rows;
    k_nrows = nrows;
  }
  // Reads the row indices of step k0, a lane each, one step ahead of the loads that use them.
  __device__ __forceinline__ void prefetch(int k0, int K) {
    if constexpr (ROWS) {
      static_assert(BK <= 64, "a lane per k");
      const int k = k0 + ((int)threadIdx.x & 63);
      index = k < K ? k_rows[k] : -1;
    }
  }
  // Loads chunk i of k step k0 of a matrix with K k's, zeros for what it does not have.
  __device__ __forceinline__ void fetch(int i, int k0, int K, uint32_t lds) const {
    const T* p;
    bool in;
    if constexpr (KC) {
      const int k = k0 + off;
      in = (ok >> i & 1) && k < K;
      p = base[i] + k;
    } else {
      const int k = k0 + off + i * (THREADS * EV / R);
      in = valid && k < K;
      if constexpr (ROWS) {
        // a row index outside the matrix, negative ones too, is past its rows as an unsigned one;
        // strides fit 32 bits
        const uint32_t r = (uint32_t)__shfl(index, off + i * (THREADS * EV / R), 64);
        in = in && r < (uint64_t)k_nrows;
        p = base[0] + (uint64_t)r * (uint32_t)ld;
      } else {
        p = base[0] + (int64_t)k * ld;
      }
    }
    const uint32_t w = __builtin_amdgcn_readfirstlane((int)threadIdx.x & ~63);
    load_lds16_at(in ? (const void*)p : (const void*)&kZeroChunk, lds + (w + i * THREADS) * 16);
  }
};

// Local row of lane index i of tile t.
template <Map MAP, int BW>
__device__ __forceinline__ constexpr int map_row(int t, int i) {
  if (MAP == WIDE) return 32 * (t / 2) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
  if (MAP == BLOCK) return 16 * BW * (t / BW) + BW * i + t % BW;
  return 16 * t + i;
}

template <typename T>
struct Frag;
template <>
struct Frag<bf16> { typedef lin_bf16x8 type; };
template <>
struct Frag<float> { typedef lin_f32x4 type; };

// Reads the fragments of a wave's tiles, whose rows start at row0 of the staged tile: of half s of
// a step, the lane's 8 bf16 k's 32 s + 8 (lane / 16) .., or its 4 fp32 k's 16 s + 4 (lane / 16) ...
// The lane's part of the LDS addresses is computed once; tiles and halves differ by constants.
template <typename T, int R, bool KC, Map MAP, int BW, int NT>
struct Reader {
  static constexpr int kTiles = MAP == BLOCK ? BW : 1;  // of one read_at
  static constexpr int NV = KC ? 2 : sizeof(T) == 2 ? NT : 1;
  static_assert(KC || sizeof(T) == 4 || NT <= 8, "a tile's pair differs from its first's in three bits");
  int off[NV];  // bytes
  __device__ __forceinline__ explicit Reader(int row0) {
    const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
    if constexpr (KC) {
      const int r = row0 + map_row<MAP, BW>(0, i16);  // row0 % 16 == 0 (WIDE: 32)
      const int key = MAP == WIDE ? (i16 & 3) | ((i16 >> 2 & 1) << 2) : i16 & 7;
#pragma unroll
      for (int s = 0; s < 2; ++s) off[s] = r * 128 + ((4 * s + kq) ^ key) * 16;
    } else if constexpr (sizeof(T) == 2) {
      // lane j of a 16-lane group addresses k row j / 4, columns 4 (j % 4) ..; it receives
      // column j of the 4 rows
      const int k = 8 * kq + (i16 >> 2), c = 4 * (i16 & 3);
#pragma unroll
      for (int u = 0; u < NT; ++u)
        off[u] = k * (R * 2) + (((row0 >> 4) + u) ^ pair_key(k)) * 32 + c * 2;
    } else {
      off[0] = (4 * kq * R + row0 + BW * i16) * 4;
    }
  }
  __device__ __forceinline__ void read(const uint4* lds, int s, typename Frag<T>::type* f) const {
#pragma unroll
    for (int t = 0; t < NT; t += MAP == BLOCK ? BW : 1) read_at(lds, s, t, f + t);
  }
  // Tile t (BLOCK: the BW tiles from it).
  __device__ __forceinline__ void read_at(const uint4* lds, int s, int t,
                                          typename Frag<T>::type* f) const {
    const char* l = reinterpret_cast<const char*>(lds);
    if constexpr (KC) {
      const int d = map_row<MAP, BW>(t, 0) * 128;
      *f = *reinterpret_cast<const typename Frag<T>::type*>(l + off[s] + d);
    } else if constexpr (sizeof(T) == 2) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4* lds_s4;
      const char* p = l + off[t] + 32 * s * (R * 2);
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 4 * (R * 2)));
      *f = __builtin_bit_cast(lin_bf16x8,
                                __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* p = l + off[0] + ((16 * s + j) * R + 16 * t) * 4;
        if constexpr (BW == 4) {
          const lin_f32x4 v = *reinterpret_cast<const lin_f32x4*>(p);
#pragma unroll
          for (int b = 0; b < 4; ++b) f[b][j] = v[b];
        } else {
          const float2 v = *reinterpret_cast<const float2*>(p);
          f[0][j] = v.x;
          f[1][j] = v.y;
        }
      }
    }
  }
};

__device__ __forceinline__ lin_f32x4 mma(lin_bf16x8 a, lin_bf16x8 b, lin_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ lin_f32x4 mma(lin_f32x4 a, lin_f32x4 b, lin_f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// fp32 products on the bf16 matrix cores, which are 16 times as fast as the fp32 ones: x = h + m + l
// exactly, 8 significant bits each by rounding to the nearest, and a b = the six products down
// to m m and h l. What is left out, m l, l m and l l, is at most 2^-24 of |a b| (|m| <= 2^-8,
// |l| <= 2^-17 of the largest power of two in |x|), half a step of fp32. Each kept product is
// exact in fp32 and summed in fp32. An infinite x, or one that rounds to infinity, gives m = NaN:
// results that are not finite are computed again by the fp32 products. (Below 2^-110 l is a
// subnormal bf16.)
struct Split {
  lin_bf16x8 h, m, l;
  __device__ __forceinline__ explicit Split(const float (&x)[8]) {
    // two values an instruction where there is one
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    auto round2 = [](f2 v) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2)); };
    auto rest = [](f2 v, uint32_t r) {
      return f2{v[0] - __uint_as_float(r << 16), v[1] - __uint_as_float(r & 0xffff0000u)};
    };
    uint32_t w[3][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f2 v = {x[2 * q], x[2 * q + 1]};
      w[0][q] = round2(v);
      const f2 r = rest(v, w[0][q]);
      w[1][q] = round2(r);
      w[2][q] = round2(rest(r, w[1][q]));
    }
    __builtin_memcpy(&h, w[0], 16);
    __builtin_memcpy(&m, w[1], 16);
    __builtin_memcpy(&l, w[2], 16);
  }
};
__device__ __forceinline__ lin_f32x4 mma(const Split& a, const Split& b, lin_f32x4 c) {
  c = mma(a.l, b.h, c);
  c = mma(a.h, b.l, c);
  c = mma(a.m, b.m, c);
  c = mma(a.m, b.h, c);
  c = mma(a.h, b.m, c);
  return mma(a.h, b.h, c);
}

// Reads a wave's fp32 tiles for them: the lane's 8 k's 8 (lane / 16) .. of a whole step.
template <int R, bool KC, int BW>
struct SplitReader {
  static constexpr int kTiles = KC ? 1 : BW;
  int off[2];  // bytes
  __device__ __forceinline__ explicit SplitReader(int row0) {
    const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
#pragma unroll
    for (int s = 0; s < 2; ++s)
      off[s] = KC ? (row0 + i16) * 128 + ((2 * kq + s) ^ (i16 & 7)) * 16 : (8 * kq * R + row0 + BW * i16) * 4;
  }
  // Tile t (!KC: the BW tiles from it).
  __device__ __forceinline__ void read(const uint4* lds, int t, float (*f)[8]) const {
    const char* l = reinterpret_cast<const char*>(lds);
    if constexpr (KC) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        *reinterpret_cast<lin_f32x4*>(&f[0][4 * s]) = *reinterpret_cast<const lin_f32x4*>(l + off[s] + t * 2048);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float* p = reinterpret_cast<const float*>(l + off[0] + (j * R + 16 * t) * 4);
        float v[BW];
        __builtin_memcpy(v, __builtin_assume_aligned(p, 4 * BW), sizeof(v));
#pragma unroll
        for (int b = 0; b < BW; ++b) f[b][j] = v[b];
      }
    }
  }
};

// Their main loop. A step's values wait in registers: while they are split and multiplied, the next
// step's are read over them from the other LDS buffer, and the step after next is loaded into
// the buffer they came from. extra(i, a, b) as pipe_loop's.
template <typename SH, typename OA, typename OB, typename RA, typename RB, typename EX>
__device__ __forceinline__ void split_loop(OA& oa, OB& ob, int K, uint4* sA, uint4* sB,
                                           lin_f32x4 (&acc)[SH::RT][SH::CT], const RA& ra, RB&& rb,
                                           EX&& extra) {
  constexpr int RT = SH::RT, CT = SH::CT, BK = OA::BK, LA = OA::NCH, LB = OB::NCH, AT = RA::kTiles;
  const int steps = (K + BK - 1) / BK;
  if (steps == 0) return;
  const uint32_t da = lds_address(sA), db = lds_address(sB);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    oa.prefetch(p * BK, K);
    ob.prefetch(p * BK, K);
#pragma unroll
    for (int c = 0; c < LA; ++c) oa.fetch(c, p * BK, K, da + p * OA::kChunks * 16);
#pragma unroll
    for (int c = 0; c < LB; ++c) ob.fetch(c, p * BK, K, db + p * OB::kChunks * 16);
  }
  oa.prefetch(2 * BK, K);
  ob.prefetch(2 * BK, K);
  wait_vmcnt<LA + LB>();
  lds_barrier();
  float xa[RT][8], xb[CT][8];
  rb(sB, xb);
#pragma unroll
  for (int i = 0; i < RT; i += AT) ra.read(sA, i, xa + i);
#pragma unroll 1
  for (int st = 0; st < steps; ++st) {
    const int x = st & 1, y = x ^ 1, k0 = (st + 2) * BK;
    wait_vmcnt<0>();
    lds_barrier();  // step st is in registers everywhere, step st + 1 in buffer y
    static_assert(CT == 4, "as many as there are initialisers");
    Split b[CT] = {Split(xb[0]), Split(xb[1]), Split(xb[2]), Split(xb[3])};
    rb(sB + y * OB::kChunks, xb);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const Split a(xa[i]);
      if (i % AT == AT - 1) ra.read(sA + y * OA::kChunks, i - (AT - 1), xa + i - (AT - 1));
#pragma unroll
      for (int c = i * LA / RT; c < (i + 1) * LA / RT; ++c) oa.fetch(c, k0, K, da + x * (OA::kChunks * 16));
#pragma unroll
      for (int c = i * LB / RT; c < (i + 1) * LB / RT; ++c) ob.fetch(c, k0, K, db + x * (OB::kChunks * 16));
#pragma unroll
      for (int j = 0; j < CT; ++j) acc[i][j] = mma(b[j], a, acc[i][j]);
      extra(i, a, b);
    }
    oa.prefetch(k0 + BK, K);
    ob.prefetch(k0 + BK, K);
  }
  wait_vmcnt<0>();  // the loads past the end: their buffers are used again
}

// Whether any of the workgroup's sums is not finite.
template <int RT, int CT>
__device__ __forceinline__ bool any_not_finite(const lin_f32x4 (&acc)[RT][CT]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(acc[i][j][e], 0.f, s);
  return __syncthreads_or(s != s);
}
template <int N, int M>
__device__ __forceinline__ void clear(lin_f32x4 (&acc)[N][M]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < M; ++j) acc[i][j] = lin_f32x4{0.f, 0.f, 0.f, 0.f};
}

// The main loop: acc += A tile . B tile^T over K, B as the matrix core's first operand, so that a
// lane ends with 4 consecutive n of its own m.
//
// A step is 128 bytes of k in two halves. While a half is multiplied, the next one's fragments
// are read from LDS: B's into a second set of registers, those of A's row tile i into its own
// as soon as its products are issued (the last tile alternates with a spare, so that its read
// need not wait for the half's end). After a step's first half nobody needs its buffer any
// more: one barrier there frees it for the loads of the step after next, which are issued
// between the second half's products and have a step and a half to arrive, and makes the next
// step's buffer, loaded by then, visible. extra(i, fa, fb): more products with row tile i.
template <typename T, typename SH, typename OA, typename OB, typename RA, typename RB, typename EX>
__device__ __forceinline__ void pipe_loop(OA& oa, OB& ob, int K, uint4* sA, uint4* sB,
                                          lin_f32x4 (&acc)[SH::RT][SH::CT], const RA& ra, RB&& rb,
                                          EX&& extra) {
  constexpr int RT = SH::RT, CT = SH::CT, BK = OA::BK, LA = OA::NCH, LB = OB::NCH;
  constexpr int AT = RA::kTiles;  // tiles one read of A yields
  typedef typename Frag<T>::type F;
  const int steps = (K + BK - 1) / BK;
  if (steps == 0) return;
  const uint32_t da = lds_address(sA), db = lds_address(sB);
  F fa[RT], spare[AT], fb0[CT], fb1[CT];
  // one half: products of (fa, with the last tiles in `last`) and fb; reads half s of (la, lb) into
  // (fa, with the last tiles in `next_last`) and nb
  auto half = [&](F(&fb)[CT], F(&nb)[CT], F* last, F* next_last, const uint4* la, const uint4* lb,
                  int s, auto&& load) {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (i == 0) {
        rb(lb, s, nb);
        ra.read_at(la, s, RT - AT, next_last);
      } else if (i % AT == 0) {
        ra.read_at(la, s, i - AT, fa + i - AT);
      }
      load(i);
      const F& f = i < RT - AT ? fa[i] : last[i - (RT - AT)];
#pragma unroll
      for (int j = 0; j < CT; ++j) acc[i][j] = mma(fb[j], f, acc[i][j]);
      extra(i, f, fb);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // steps past the end load zero chunks and are never multiplied: the loop has one form
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    oa.prefetch(p * BK, K);
    ob.prefetch(p * BK, K);
#pragma unroll
    for (int c = 0; c < LA; ++c) oa.fetch(c, p * BK, K, da + p * OA::kChunks * 16);
#pragma unroll
    for (int c = 0; c < LB; ++c) ob.fetch(c, p * BK, K, db + p * OB::kChunks * 16);
  }
  oa.prefetch(2 * BK, K);
  ob.prefetch(2 * BK, K);
  wait_vmcnt<LA + LB>();
  lds_barrier();
  rb(sB, 0, fb0);
#pragma unroll
  for (int i = 0; i < RT; i += AT) ra.read_at(sA, 0, i, fa + i);
#pragma unroll 1
  for (int st = 0; st < steps; ++st) {
    const int x = st & 1, y = x ^ 1, k0 = (st + 2) * BK;
    half(fb0, fb1, fa + RT - AT, spare, sA + x * OA::kChunks, sB + x * OB::kChunks, 1, [](int) {});
    wait_vmcnt<0>();
    lds_barrier();
    half(fb1, fb0, spare, fa + RT - AT, sA + y * OA::kChunks, sB + y * OB::kChunks, 0, [&](int i) {
#pragma unroll
      for (int c = i * LA / RT; c < (i + 1) * LA / RT; ++c)
        oa.fetch(c, k0, K, da + x * (OA::kChunks * 16));
#pragma unroll
      for (int c = i * LB / RT; c < (i + 1) * LB / RT; ++c)
        ob.fetch(c, k0, K, db + x * (OB::kChunks * 16));
    });
    oa.prefetch(k0 + BK, K);
    ob.prefetch(k0 + BK, K);
  }
  wait_vmcnt<0>();  // the loads past the end: their buffers are used again
}

// Rows [r0, r1) of group g, kept inside the matrix whatever the offsets hold; group `groups` is
// the rows past the last one.
__device__ __forceinline__ void group_span(const LinearArgs& a, int g, int& r0, int& r1) {
  if (!a.offsets) {
    r0 = 0;
    r1 = g == 0 ? a.rows : 0;
    return;
  }
  r0 = min(max(a.offsets[g], 0), a.rows);
  r1 = g < a.groups ? min(max(a.offsets[g + 1], 0), a.rows) : a.rows;
}

// Finds the row tiles of a launch, counted group by group, 64 groups at a time, one per lane. The
// last of them are the rows of no group. With fewer than 64 groups (the usual case) the offsets
// are looked at once.
template <int BM>
struct RowTiles {
  const LinearArgs& a;
  int total;             // at most the launch's bound
  int s0, s1, nt, incl;  // this lane's group of the 64 looked at: rows, tiles, tiles up to it
  __device__ __forceinline__ explicit RowTiles(const LinearArgs& args) : a(args) {
    int64_t all = 0;
    for (int g0 = 0; g0 <= a.groups; g0 += 64) all += look(g0);
    total = (int)min(all, (int64_t)a.max_tiles);
  }
  __device__ __forceinline__ int look(int g0) {
    const int lane = (int)threadIdx.x & 63;
    s0 = s1 = 0;
    if (g0 + lane <= a.groups) group_span(a, g0 + lane, s0, s1);
    nt = s1 > s0 ? (s1 - s0 + BM - 1) / BM : 0;
    incl = nt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(incl, d, 64);
      if (lane >= d) incl += v;
    }
    return __builtin_amdgcn_readlane(incl, 63);
  }
  // Row tile t: its group, first row and the group's end. false: there is none.
  __device__ __forceinline__ bool find(int t, int& group, int& r0, int& r1) {
    int64_t before = 0;
    for (int g0 = 0; g0 <= a.groups; g0 += 64) {
      const int all = a.groups < 64 ? __builtin_amdgcn_readlane(incl, 63) : look(g0);
      if (t < before + all) {
        // the first lane whose inclusive count passes t
        const int src = (int)__builtin_popcountll(__ballot(before + incl <= t));
        group = g0 + src;
        r1 = __builtin_amdgcn_readlane(s1, src);
        r0 = __builtin_amdgcn_readlane(s0, src) +
             (int)(t - before - __builtin_amdgcn_readlane(incl - nt, src)) * BM;
        return true;
      }
      before += all;
    }
    return false;
  }
};

// Tiles in the order that shares operands through one L2: the launch's tiles are cut into 8
// contiguous ranges, one per XCD (workgroup L runs on XCD L % 8), and run in bands of kBand
// rows of tiles, rows fastest: the 32 CUs of an XCD then work on about 8 x 4 tiles.
constexpr int kBand = 8;
__device__ __forceinline__ void band_tile(int item, int band_rows, int tiles_r, int tiles_c, int& tr,
                                          int& tc) {
  const int band = item / (band_rows * tiles_c), in = item - band * band_rows * tiles_c;
  const int rows = min(band_rows, tiles_r - band * band_rows);
  tr = band * band_rows + in % rows;
  tc = in / rows;
}
// This workgroup's tile; false: it has none.
__device__ __forceinline__ bool place_tile(int tiles_r, int tiles_c, int& tr, int& tc) {
  const int total = tiles_r * tiles_c, xcd = (int)blockIdx.x % kXcds, slot = (int)blockIdx.x / kXcds;
  const int per = (total + kXcds - 1) / kXcds, item = xcd * per + slot;
  if (slot >= per || item >= total) return false;
  band_tile(item, kBand, tiles_r, tiles_c, tr, tc);
  return true;
}

// The same where the last tiles of an XCD's range, those past whole rounds of its CUs, may be shared:
// `parts` workgroups a tile.
constexpr int kXcdCus = 32;
__host__ __device__ inline int shared_parts(int rest) { return rest * 4 <= kXcdCus ? 4 : rest * 2 <= kXcdCus ? 2 : 1; }
// Workgroups for a range of `count` tiles.
__host__ __device__ inline int shared_slots(int count) {
  const int rest = count % kXcdCus;
  return count - rest + rest * shared_parts(rest);
}
__device__ __forceinline__ bool place_shared(int tiles_r, int tiles_c, int& tr, int& tc, int& part,
                                             int& parts) {
  const int total = tiles_r * tiles_c, xcd = (int)blockIdx.x % kXcds, slot = (int)blockIdx.x / kXcds;
  const int per = (total + kXcds - 1) / kXcds, first = xcd * per, count = min(per, total - first);
  if (count <= 0) return false;
  const int whole = count / kXcdCus * kXcdCus, rest = count - whole;
  int item = slot;
  part = 0;
  parts = 1;
  if (slot >= whole) {
    parts = shared_parts(rest);
    item = whole + (slot - whole) / parts;
    part = (slot - whole) % parts;
  }
  if (item >= count) return false;
  band_tile(first + item, kBand, tiles_r, tiles_c, tr, tc);
  return true;
}

// Weight-gradient tiles: group by group, the largest groups first (up to 64 groups), so that the
// long sums start early and the short ones fill up behind them; a group's tiles go to the XCDs
// in runs of an eighth of them, so that every XCD gets its share of every group.
__host__ __device__ inline int wgrad_run(int tiles_of_group) {
  return tiles_of_group < kXcds ? 1 : tiles_of_group / kXcds;
}
__device__ __forceinline__ bool place_wgrad(const LinearArgs& a, int& group, int& split, int& mt, int& nt) {
  const int per_split = a.tiles_m * a.tiles_n, per = per_split * a.splits, c = wgrad_run(per);
  const int xcd = (int)blockIdx.x % kXcds, slot = (int)blockIdx.x / kXcds;
  const int64_t q = (int64_t)(slot / c) * (kXcds * c) + xcd * c + slot % c;
  if (q >= (int64_t)a.groups * per) return false;
  group = (int)(q / per);
  const int in = (int)(q % per);
  if (a.offsets && a.groups <= 64) {
    const int lane = (int)threadIdx.x & 63;
    int r0 = 0, r1 = 0;
    if (lane < a.groups) group_span(a, lane, r0, r1);
    const int size = lane < a.groups ? max(r1 - r0, 0) : -1;
    int rank = 0;
    for (int j = 0; j < a.groups; ++j) {
      const int o = __builtin_amdgcn_readlane(size, j);
      rank += o > size || (o == size && j < lane);
    }
    group = (int)__builtin_ctzll(__ballot(lane < a.groups && rank == group));
  }
  split = in / per_split;
  band_tile(in % per_split, 4, a.tiles_m, a.tiles_n, mt, nt);
  return true;
}

// W consecutive elements, whole or up to n of them.
template <int W>
__device__ __forceinline__ void store_run(float* p, const float* v, int n) {
  if (n >= W) {
    __builtin_memcpy(p, v, 4 * W);
  } else {
#pragma unroll
    for (int q = 0; q < W; ++q)
      if (q < n) p[q] = v[q];
  }
}
template <int W>
__device__ __forceinline__ void store_run(bf16* p, const float* v, int n) {
  if (n >= W) {
    uint32_t w[W / 2];
#pragma unroll
    for (int q = 0; q < W / 2; ++q)
      w[q] = (uint32_t)f2bf(v[2 * q]).u | ((uint32_t)f2bf(v[2 * q + 1]).u << 16);
    __builtin_memcpy(p, w, 2 * W);
  } else {
#pragma unroll
    for (int q = 0; q < W; ++q)
      if (q < n) p[q] = f2bf(v[q]);
  }
}
template <int W, typename T>
__device__ __forceinline__ void load_run(const T* p, float* v, int n) {
  if (n >= W) {
    T t[W];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = to_f(t[q]);
  } else {
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = q < n ? to_f(p[q]) : 0.f;
  }
}

template <typename T, bool KC>
constexpr Map out_map() {
  return KC ? (sizeof(T) == 2 ? WIDE : PLAIN) : (sizeof(T) == 2 ? PLAIN : BLOCK);
}

// bf16 results leave the matrix core's layout in registers: of a pair of column tiles, lane group
// kq (16 lanes, a row each) ends with 8 consecutive columns, 16 bytes to store, 64 bytes a row
// beside the other groups. WIDE tiles come that way; of PLAIN ones group kq holds columns 4 kq
// .. of both tiles, and exchanging the odd groups of the first with the even ones of the second
// leaves tile kq % 2, columns 8 (kq / 2) ...
template <Map MAP>
__device__ __forceinline__ int run_col(int kq) { return MAP == WIDE ? 8 * kq : 16 * (kq & 1) + 8 * (kq >> 1); }
template <Map MAP>
__device__ __forceinline__ void take_run(const lin_f32x4& x, const lin_f32x4& y, float (&v)[8]) {
  static_assert(MAP != BLOCK, "bf16 tiles");
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (MAP == WIDE) {
      v[e] = x[e];
      v[4 + e] = y[e];
    } else {
      const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[e]), __float_as_uint(y[e]),
                                                      false, false);
      v[e] = __uint_as_float(s[0]);
      v[4 + e] = __uint_as_float(s[1]);
    }
  }
}

// fp32 results, and those of the erf activation (280 instructions a run: unrolled over the
// accumulators they take longer to fetch than the products to run), leave through LDS, a row tile
// at a time in memory of the wave's own: matrix-core order in, whole rows of C out, 8 columns a
// lane, in a short loop. A row's 16-byte chunks sit at chunk ^ row, so that the 16 rows of a
// column are on different banks. 256 x 256 tiles: 10 us this way, 5 from registers.
struct Slab {
  static constexpr int CT = 4, kFloats = 16 * 16 * CT;
  float* l;
  __device__ __forceinline__ lin_f32x4& chunk(int row, int c) const {
    return reinterpret_cast<lin_f32x4*>(l)[row * 4 * CT + (c ^ row)];
  }
  // Writes a row tile's accumulators, columns in order; tiles beyond NCT are the second set of a
  // pair, 16 NCT columns on.
  template <Map MAP, int BW, int NCT>
  __device__ __forceinline__ void write(const lin_f32x4 (&acc)[CT]) const {
    const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
#pragma unroll
    for (int j = 0; j < CT; ++j) {
      const int set = 4 * NCT * (j / NCT), u = j % NCT;
      if constexpr (MAP == BLOCK) {
        // element e of tiles u .. u + BW - 1: columns 16 u + BW (4 kq + e) ..
        if (u % BW) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BW == 4) {
            chunk(i16, set + 4 * u + 4 * kq + e) = lin_f32x4{acc[j][e], acc[j + 1][e], acc[j + 2][e], acc[j + 3][e]};
          } else {
            float* p = reinterpret_cast<float*>(&chunk(i16, set + 4 * u + 2 * kq + e / 2)) + 2 * (e & 1);
            p[0] = acc[j][e];
            p[1] = acc[j + 1][e];
          }
        }
      } else if constexpr (MAP == WIDE) {
        chunk(i16, set + 8 * (u / 2) + 2 * kq + (u & 1)) = acc[j];
      } else {
        chunk(i16, set + 4 * u + kq) = acc[j];
      }
    }
  }
  __device__ __forceinline__ void read8(int row, int c, float (&v)[8]) const {
    const lin_f32x4 x = chunk(row, c), y = chunk(row, c + 1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = x[q];
      v[4 + q] = y[q];
    }
  }
};
// Between a wave's own writes and reads of LDS.
__device__ __forceinline__ void lds_settle() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The bias of 8 columns, of both halves for a pair.
template <bool PAIR>
__device__ __forceinline__ void load_bias(const LinearArgs& a, int group, bool none, int col, int f,
                                          float (&bias)[2][8]) {
  const int n = f - col;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int q = 0; q < 8; ++q) bias[h][q] = 0.f;
  if (!a.bias || none || n <= 0) return;
#pragma unroll
  for (int h = 0; h < (PAIR ? 2 : 1); ++h) {
    const int64_t o = (int64_t)group * a.N + col + h * f;
    if (a.bias_dtype == PULSAR_F32)
      load_run<8>(reinterpret_cast<const float*>(a.bias) + o, bias[h], n);
    else
      load_run<8>(reinterpret_cast<const bf16*>(a.bias) + o, bias[h], n);
  }
}

// 8 columns of row r from their sums v (and u, a pair's second half): bias, activation and
// residual in fp32. Leaves the pre-activation values in `pre` (and u), the results in v.
template <typename T, bool PAIR>
__device__ __forceinline__ void finish_values(const LinearArgs& a, int act, int64_t r, int col, int f,
                                              float (&v)[8], float (&u)[8], float (&pre)[8],
                                              const float (&bias)[2][8]) {
  if (a.bias) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      v[q] += bias[0][q];
      if constexpr (PAIR) u[q] += bias[1][q];
    }
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) pre[q] = v[q];
  if constexpr (PAIR) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = v[q] * fast_sigmoid(v[q]) * u[q];
  } else {
    act_values(act, v);
  }
  if (a.residual) {
    float x[8];
    load_run<8>(reinterpret_cast<const T*>(a.residual) + r * a.ldr + col, x, f - col);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += x[q];
  }
}
// 8 partial sums of row r from column col on, of split blockIdx.y.
__device__ __forceinline__ void store_part(const LinearArgs& a, int64_t r, int col, int f, const float (&v)[8]) {
  store_run<8>(a.part + ((int64_t)blockIdx.y * a.rows + r) * a.N + col, v, f - col);
}
// The same, stored with one rounding, or the sums of one of the splits (SPLIT).
template <typename T, bool PAIR, bool SPLIT>
__device__ __forceinline__ void finish_run(const LinearArgs& a, int act, int64_t r, int col, int f,
                                           float (&v)[8], float (&u)[8], const float (&bias)[2][8]) {
  if (SPLIT && a.part) {
    store_part(a, r, col, f, v);
    if constexpr (PAIR) store_part(a, r, f + col, 2 * f, u);
    return;
  }
  float pre[8];
  finish_values<T, PAIR>(a, act, r, col, f, v, u, pre, bias);
  const int n = f - col;
  if (a.pre) {
    T* o = reinterpret_cast<T*>(a.pre) + r * a.ldpre + col;
    store_run<8>(o, pre, n);
    if constexpr (PAIR) store_run<8>(o + f, u, n);
  }
  store_run<8>(reinterpret_cast<T*>(a.C) + r * a.ldc + col, v, n);
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] = (uint32_t)f2bf(v[2 * q]).u | ((uint32_t)f2bf(v[2 * q + 1]).u << 16);
  return uint4{w[0], w[1], w[2], w[3]};
}

// Stores two runs of a lane, as bf16, of columns c0 .. and 32 further on, in the wave's layout (row
// i16, column run by lane group). Rows 0 - 7 give their second run for rows 8 - 15's first, so
// that a store covers 8 rows by 128 bytes, whole cache lines, and not 16 by 64. With two waves
// on a SIMD an instruction for each of a lane's 128 results is half a us of a tile: addresses
// are one 64-bit addition a store, bounds are only looked at in tiles that have any.
template <Map MAP>
struct PairStore {
  bf16* p;
  int64_t ld;
  int left, n;  // rows and columns inside from this lane's first
  bool whole;   // of the wave's tile
  __device__ __forceinline__ PairStore(bf16* m, int64_t ld_, int rows, int r0, int r1, int c0, int f) : ld(ld_) {
    const int lane = (int)threadIdx.x & 63, i16 = lane & 15;
    const int r = r0 + (i16 & 7), c = c0 + run_col<MAP>(lane >> 4) + (i16 >= 8 ? 32 : 0);
    p = m + r * ld + c;
    left = r1 - r;
    n = f - c;
    whole = r1 - r0 >= rows && f - c0 >= 64;
  }
  __device__ __forceinline__ void operator()(int i, const uint4& x, const uint4& y) const {
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
    uint32_t w[2][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // lanes 8 - 15 of each 16: the other half's (row rotation by 8, written to banks 2 and 3)
      w[0][q] = (uint32_t)__builtin_amdgcn_update_dpp((int)xs[q], (int)ys[q], 0x128, 0xf, 0xc, false);
      w[1][q] = (uint32_t)__builtin_amdgcn_update_dpp((int)ys[q], (int)xs[q], 0x128, 0xf, 0x3, false);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16* o = p + (16 * i + 8 * h) * ld;
      if (whole || (16 * i + 8 * h < left && n >= 8)) {
        __builtin_memcpy(o, w[h], 16);
      } else if (16 * i + 8 * h < left) {
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (q < n) o[q].u = (uint16_t)(w[h][q >> 1] >> (16 * (q & 1)));
      }
    }
  }
};

// The bias of the wave's columns as the epilogue will want them: of bf16 results runs of 8, from
// column c0; of fp32 ones the lane's 8 of a slab row.
template <typename T, Map MAP, bool PAIR>
struct EpilogueBias {
  static constexpr int NCT = PAIR ? Slab::CT / 2 : Slab::CT;
  static constexpr int N = sizeof(T) == 2 ? NCT / 2 : 1;
  float b[N][2][8], slab[2][8];
  __device__ __forceinline__ EpilogueBias(const LinearArgs& a, int group, bool none, int c0, int f) {
    const int lane = (int)threadIdx.x & 63;
    const bool via_slab = sizeof(T) == 4 || a.act == PULSAR_ACT_GELU;
    const int lc = c0 + lane % (NCT * 2) * 8;
    load_bias<PAIR>(a, group, none || !via_slab, lc, f, slab);
#pragma unroll
    for (int p = 0; p < N; ++p) load_bias<PAIR>(a, group, none || via_slab, c0 + 32 * p + run_col<MAP>(lane >> 4), f, b[p]);
  }
};

// Epilogue of a product's tile. The wave's accumulators start at row r0 and output column c0; of
// `f` output columns and rows below r1 only those inside are stored. PAIR: the second half of the
// CT tiles are the up-projection twins of the first.
template <typename T, Map MAP, int BW, bool PAIR, bool SPLIT, int RT>
__device__ __forceinline__ void rows_epilogue(const LinearArgs& a, lin_f32x4 (&acc)[RT][Slab::CT],
                                              Slab slab, const EpilogueBias<T, MAP, PAIR>& bias,
                                              bool none, int r0, int r1, int c0, int f) {
  constexpr int NCT = PAIR ? Slab::CT / 2 : Slab::CT;
  const int lane = (int)threadIdx.x & 63, act = none ? PULSAR_ACT_NONE : a.act;
  if constexpr (sizeof(T) == 2 && !PAIR) {
    if (SPLIT && a.part) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float v[8];
          take_run<MAP>(acc[i][2 * p], acc[i][2 * p + 1], v);
          const int r = r0 + 16 * i + (lane & 15), col = c0 + 32 * p + run_col<MAP>(lane >> 4);
          if (r < r1 && col < f) store_part(a, r, col, f, v);
        }
      return;
    }
    const PairStore<MAP> out(reinterpret_cast<bf16*>(a.C), a.ldc, 16 * RT, r0, r1, c0, f);
    if (act == PULSAR_ACT_NONE && !a.bias && !a.residual && !a.pre) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float v[2][8];
#pragma unroll
        for (int p = 0; p < 2; ++p) take_run<MAP>(acc[i][2 * p], acc[i][2 * p + 1], v[p]);
        out(i, pack8(v[0]), pack8(v[1]));
      }
      return;
    }
    if (act != PULSAR_ACT_GELU) {
      const PairStore<MAP> kept(reinterpret_cast<bf16*>(a.pre), a.ldpre, 16 * RT, r0, r1, c0, f);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        // the residual's rows past the end: the last one's
        const int64_t r = min(r0 + 16 * i + (lane & 15), r1 - 1);
        uint4 o[2], k[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          float v[8], u[8], pre[8];
          take_run<MAP>(acc[i][2 * p], acc[i][2 * p + 1], v);
          finish_values<T, PAIR>(a, act, r, c0 + 32 * p + run_col<MAP>(lane >> 4), f, v, u, pre, bias.b[p]);
          o[p] = pack8(v);
          k[p] = pack8(pre);
        }
        if (a.pre) kept(i, k[0], k[1]);
        out(i, o[0], o[1]);
      }
      return;
    }
  } else if constexpr (sizeof(T) == 2) {
    const int col = c0 + run_col<MAP>(lane >> 4);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float v[8], u[8];
      take_run<MAP>(acc[i][0], acc[i][1], v);
      take_run<MAP>(acc[i][2], acc[i][3], u);
      const int64_t r = r0 + 16 * i + (lane & 15);
      if (r < r1 && col < f) finish_run<T, PAIR, SPLIT>(a, act, r, col, f, v, u, bias.b[0]);
    }
    return;
  }
  constexpr int LPR = NCT * 2, RPI = 64 / LPR;  // lanes a row, rows a pass
  const int lc = lane % LPR, lr = lane / LPR, col = c0 + 8 * lc;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    slab.write<MAP, BW, NCT>(acc[i]);
    lds_settle();
#pragma unroll 1
    for (int p = lr; p < 16; p += RPI) {
      const int64_t r = r0 + 16 * i + p;
      if (r >= r1 || col >= f) continue;
      float v[8], u[8] = {};
      slab.read8(p, 2 * lc, v);
      if constexpr (PAIR) slab.read8(p, 4 * NCT + 2 * lc, u);
      finish_run<T, PAIR, SPLIT>(a, act, r, col, f, v, u, bias.slab);
    }
    lds_settle();  // read before the next rows overwrite
  }
}

// Epilogue of a weight gradient's tile: into C, or a split's partial sums. `sums`: this wave holds
// the column sums of SIDE's operand.
template <typename T, Map MAP, int BWR, int BWC, int SIDE, int RT, int CT, int NS>
__device__ __forceinline__ void wgrad_epilogue(const LinearArgs& a, lin_f32x4 (&acc)[RT][CT],
                                               lin_f32x4 (&sum)[NS], Slab slab, bool sums,
                                               int group, int split, int m0, int n0) {
  const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
  const int64_t pg = (int64_t)split * a.groups + group;  // a split's partial results
  auto store = [&](int64_t m, int col, const float (&v)[8]) {
    if (m >= a.M || col >= a.N) return;
    if (a.splits > 1)
      store_run<8>(a.part + (pg * a.M + m) * a.N + col, v, a.N - col);
    else
      store_run<8>(reinterpret_cast<T*>(a.C) + group * a.c_group + m * a.ldc + col, v, a.N - col);
  };
  if constexpr (sizeof(T) == 2) {
    const PairStore<MAP> out(reinterpret_cast<bf16*>(a.C) + group * a.c_group, a.ldc, 16 * RT, m0, a.M, n0, a.N);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float v[2][8];
#pragma unroll
      for (int p = 0; p < 2; ++p) take_run<MAP>(acc[i][2 * p], acc[i][2 * p + 1], v[p]);
      if (a.splits > 1) {
#pragma unroll
        for (int p = 0; p < 2; ++p) store(m0 + 16 * i + i16, n0 + 32 * p + run_col<MAP>(kq), v[p]);
      } else {
        out(i, pack8(v[0]), pack8(v[1]));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      slab.write<MAP, BWC, CT>(acc[i]);
      lds_settle();
#pragma unroll 1
      for (int p = lane / 8; p < 16; p += 8) {
        float v[8];
        slab.read8(p, lane % 8 * 2, v);
        store(m0 + map_row<MAP, BWR>(i, p), n0 + lane % 8 * 8, v);
      }
      lds_settle();
    }
  }
  // SIDE 1: lane i16 holds row map_row(i, i16) of A in every element; SIDE 2: element e of lane
  // group kq holds row 4 kq + e of B's tile
  if constexpr (SIDE == 1) {
    if (sums && kq == 0) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int m = m0 + map_row<MAP, BWR>(i, i16);
        if (m >= a.M) continue;
        if (a.splits > 1)
          a.part_db[pg * a.M + m] = sum[i][0];
        else
          reinterpret_cast<T*>(a.db)[(int64_t)group * a.M + m] = from_f<T>(sum[i][0]);
      }
    }
  }
  if constexpr (SIDE == 2) {
    if (sums && i16 == 0) {
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = n0 + map_row<MAP, BWC>(j, 4 * kq + e);
          if (c >= a.N) continue;
          if (a.splits > 1)
            a.part_db[pg * a.N + c] = sum[j][e];
          else
            reinterpret_cast<T*>(a.db)[(int64_t)group * a.N + c] = from_f<T>(sum[j][e]);
        }
    }
  }
}

}  // namespace

}  // namespace pulsar
