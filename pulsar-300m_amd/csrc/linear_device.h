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
//     the LDS transpose load, 4 k rows x 32 bytes per 16 lanes: 32-byte pairs of chunks sit
//     at pair ^ (k & 3), which puts the 4 rows on different banks. ROWS: k row r is stored row
//     k_rows[r].
template <typename T, int R, bool KC, Map MAP, int THREADS, bool ROWS = false>
struct Operand {
  static constexpr int EV = 16 / (int)sizeof(T), BK = 128 / (int)sizeof(T);
  static constexpr int kChunks = R * 8, NCH = kChunks / THREADS;
  static_assert(kChunks % THREADS == 0, "whole chunks per thread");
  static_assert(KC ? (THREADS / 8) % 16 == 0 : (THREADS * EV / R) % 4 == 0, "one swizzle key per thread");

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
    if constexpr (sizeof(T) == 2) lc = (((c >> 1) ^ (off & 3)) << 1) | (c & 1);
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
template <typename T, int R, bool KC, Map MAP, int BW>
struct Reader {
  static constexpr int kTiles = MAP == BLOCK ? BW : 1;  // of one read_at
  static constexpr int NV = KC ? 2 : sizeof(T) == 2 ? 4 : 1;
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
      for (int u = 0; u < 4; ++u)
        off[u] = k * (R * 2) + (((row0 >> 4) + u) ^ (k & 3)) * 32 + c * 2;
    } else {
      off[0] = (4 * kq * R + row0 + BW * i16) * 4;
    }
  }
  template <int NT>
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
      const char* p = l + off[t & 3] + 32 * s * (R * 2) + (t >> 2) * 128;
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

// The number of row tiles of the launch, counted group by group (64 at a time, one per lane), at
// most the launch's bound.
template <int BM>
__device__ __forceinline__ int count_tiles(const LinearArgs& a) {
  const int lane = (int)threadIdx.x & 63;
  int64_t all = 0;
  for (int g0 = 0; g0 <= a.groups; g0 += 64) {
    int s0 = 0, s1 = 0;
    if (g0 + lane <= a.groups) group_span(a, g0 + lane, s0, s1);
    int nt = s1 > s0 ? (s1 - s0 + BM - 1) / BM : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) nt += __shfl_xor(nt, d, 64);
    all += nt;
  }
  return (int)min(all, (int64_t)a.max_tiles);
}

// Row tile t: its group, first row and the group's end. false: there is none.
template <int BM>
__device__ __forceinline__ bool find_tile(const LinearArgs& a, int t, int& group, int& r0, int& r1) {
  const int lane = (int)threadIdx.x & 63;
  int64_t before = 0;
  for (int g0 = 0; g0 <= a.groups; g0 += 64) {
    int s0 = 0, s1 = 0;
    if (g0 + lane <= a.groups) group_span(a, g0 + lane, s0, s1);
    const int nt = s1 > s0 ? (s1 - s0 + BM - 1) / BM : 0;
    int incl = nt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(incl, d, 64);
      if (lane >= d) incl += v;
    }
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (t < before + total) {
      // the first lane whose inclusive count passes t
      const int src = (int)__builtin_popcountll(__ballot(before + incl <= t));
      group = g0 + src;
      r1 = __builtin_amdgcn_readlane(s1, src);
      r0 = __builtin_amdgcn_readlane(s0, src) +
           (int)(t - before - __builtin_amdgcn_readlane(incl - nt, src)) * BM;
      return true;
    }
    before += total;
  }
  return false;
}

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
__device__ __forceinline__ bool place_tile(int tiles_r, int tiles_c, int& tr, int& tc) {
  const int total = tiles_r * tiles_c;
  const int L = (int)blockIdx.x, xcd = L % kXcds, slot = L / kXcds;
  const int per = (total + kXcds - 1) / kXcds;
  const int item = xcd * per + slot;
  if (slot >= per || item >= total) return false;
  band_tile(item, kBand, tiles_r, tiles_c, tr, tc);
  return true;
}

// The tile of this workgroup: column block tc, rows r0 .. of group `group`, whose end is r1.
template <int BM>
__device__ __forceinline__ bool locate_tile(const LinearArgs& a, int tiles_c, int& tc, int& group,
                                            int& r0, int& r1) {
  int tr;
  if (a.groups < 64) {  // one look at the offsets (their loads are the start of every chain here)
    const int lane = (int)threadIdx.x & 63;
    int s0 = 0, s1 = 0;
    if (lane <= a.groups) group_span(a, lane, s0, s1);
    const int nt = s1 > s0 ? (s1 - s0 + BM - 1) / BM : 0;
    int incl = nt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(incl, d, 64);
      if (lane >= d) incl += v;
    }
    const int tiles_r = min(__builtin_amdgcn_readlane(incl, 63), a.max_tiles);
    if (!place_tile(tiles_r, tiles_c, tr, tc)) return false;
    group = (int)__builtin_popcountll(__ballot(incl <= tr));
    r1 = __builtin_amdgcn_readlane(s1, group);
    r0 = __builtin_amdgcn_readlane(s0, group) +
         (tr - __builtin_amdgcn_readlane(incl - nt, group)) * BM;
    return true;
  }
  return place_tile(count_tiles<BM>(a), tiles_c, tr, tc) && find_tile<BM>(a, tr, group, r0, r1);
}

// Weight-gradient tiles: group by group, the largest groups first (up to 64 groups), so that the
// long sums start early and the short ones fill up behind them; a group's tiles go to the XCDs
// in runs of an eighth of them, so that every XCD gets its share of every group.
__device__ __forceinline__ int wgrad_run(int tiles_of_group) { return max(1, tiles_of_group / kXcds); }
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

// Accumulators leave through LDS, two row tiles (32 rows) at a time in memory of the wave's own:
// matrix-core order in, whole rows of C out, 8 columns a lane. Columns are read back in order,
// so stores are 16 bytes and cover cache lines, and the epilogue is a short loop (unrolled
// over the registers it was 15,000 instructions, which took longer to fetch than the tile's
// products to run). Rows are 4 floats apart from a multiple of the banks.
template <int CT>
struct Slab {
  static constexpr int kCols = 16 * CT, kStride = kCols + 4, kFloats = 32 * kStride;
};

// Writes one row tile of accumulators: LDS row i16, columns in order.
template <Map MAP, int BW, int NCT, int CT>
__device__ __forceinline__ void slab_write_tile(float* slab, const lin_f32x4 (&acc)[CT]) {
  const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    // tiles beyond NCT are the second set of a pair, 16 NCT columns on
    const int u = j % NCT;
    float* p = slab + i16 * Slab<CT>::kStride + j / NCT * 16 * NCT;
    if constexpr (MAP == BLOCK) {
      // element e of tile u: column 16 BW (u / BW) + BW (4 kq + e) + u % BW
      if (u % BW) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int b = 0; b < BW; ++b) p[16 * u + BW * (4 * kq + e) + b] = acc[j + b][e];
    } else {
      // 4 consecutive columns
      *reinterpret_cast<lin_f32x4*>(p + map_row<MAP, BW>(u, 0) + (MAP == WIDE ? 8 : 4) * kq) = acc[j];
    }
  }
}

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
// residual in fp32, one rounding per output.
template <typename T, bool PAIR>
__device__ __forceinline__ void finish_run(const LinearArgs& a, int act, int64_t r, int col, int f,
                                           float (&v)[8], float (&u)[8], const float (&bias)[2][8]) {
  const int n = f - col;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    v[q] += bias[0][q];
    if constexpr (PAIR) u[q] += bias[1][q];
  }
  if (a.pre) {
    T* pre = reinterpret_cast<T*>(a.pre) + r * a.ldpre + col;
    store_run<8>(pre, v, n);
    if constexpr (PAIR) store_run<8>(pre + f, u, n);
  }
  if constexpr (PAIR) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = v[q] * fast_sigmoid(v[q]) * u[q];
  } else if (act != PULSAR_ACT_NONE) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = act_value(act, v[q]);
  }
  if (a.residual) {
    float x[8];
    load_run<8>(reinterpret_cast<const T*>(a.residual) + r * a.ldr + col, x, n);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += x[q];
  }
  store_run<8>(reinterpret_cast<T*>(a.C) + r * a.ldc + col, v, n);
}

// Epilogue of a product's tile. The wave's accumulators start at row r0 and output column c0; of `f` output columns and rows
// below r1 only those inside are stored. PAIR: the second half of the CT tiles are the
// up-projection twins of the first.
template <typename T, Map MAP, int BW, bool PAIR, int RT, int CT>
__device__ __forceinline__ void rows_epilogue(const LinearArgs& a, lin_f32x4 (&acc)[RT][CT],
                                              float* slab, int group, bool none, int r0, int r1,
                                              int c0, int f) {
  constexpr int NCT = PAIR ? CT / 2 : CT, LPR = NCT * 2, RPI = 64 / LPR;  // lanes a row, rows a pass
  static_assert(64 % LPR == 0, "whole rows per pass");
  const int lane = (int)threadIdx.x & 63, lc = (lane % LPR) * 8, lr = lane / LPR;
  const int col = c0 + lc, n = f - col;
  float bias[2][8];
  load_bias<PAIR>(a, group, none, col, f, bias);
  const int act = none ? PULSAR_ACT_NONE : a.act;
#pragma unroll
  for (int i = 0; i < RT; i += 2) {
    slab_write_tile<MAP, BW, NCT>(slab, acc[i]);
    slab_write_tile<MAP, BW, NCT>(slab + 16 * Slab<CT>::kStride, acc[i + 1]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
    for (int p = lr; p < 32; p += RPI) {
      const int64_t r = r0 + 16 * i + p;
      if (r >= r1 || n <= 0) continue;
      float v[8], u[8];
      const float* l = slab + p * Slab<CT>::kStride + lc;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        v[q] = l[q];
        u[q] = PAIR ? l[16 * NCT + q] : 0.f;
      }
      finish_run<T, PAIR>(a, act, r, col, f, v, u, bias);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next rows overwrite
  }
}

// Epilogue of a weight gradient's tile: into C, or a split's partial sums. `sums`: this wave holds
// the column sums of SIDE's operand.
template <typename T, Map MAP, int BWR, int BWC, int SIDE, int RT, int CT, int NS>
__device__ __forceinline__ void wgrad_epilogue(const LinearArgs& a, lin_f32x4 (&acc)[RT][CT],
                                               lin_f32x4 (&sum)[NS], float* slab, bool sums,
                                               int group, int split, int m0, int n0) {
  const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
  constexpr int LPR = CT * 2, RPI = 64 / LPR;
  const int lc = (lane % LPR) * 8, lr = lane / LPR, col = n0 + lc, n = a.N - col;
  const int64_t pg = (int64_t)split * a.groups + group;  // a split's partial results
#pragma unroll
  for (int i = 0; i < RT; i += 2) {
    slab_write_tile<MAP, BWC, CT>(slab, acc[i]);
    slab_write_tile<MAP, BWC, CT>(slab + 16 * Slab<CT>::kStride, acc[i + 1]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
    for (int p = lr; p < 32; p += RPI) {
      const int64_t m = m0 + (p < 16 ? map_row<MAP, BWR>(i, p) : map_row<MAP, BWR>(i + 1, p - 16));
      if (m >= a.M || n <= 0) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = slab[p * Slab<CT>::kStride + lc + q];
      if (a.splits > 1)
        store_run<8>(a.part + (pg * a.M + m) * a.N + col, v, n);
      else
        store_run<8>(reinterpret_cast<T*>(a.C) + group * a.c_group + m * a.ldc + col, v, n);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
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
