// Dense and ragged (grouped by expert) products with bias, activation and residual in the
// epilogue, and their gradients: fused_linear_* and grouped_linear_* of the op surface.
#include <algorithm>
#include <type_traits>

#include "linear.h"

namespace pulsar {

namespace {

constexpr int kXcds = 8;  // consecutive workgroups go to the 8 XCDs in turn

// Operand chunks that lie outside a matrix (past the last k, outside a group, rows an index
// does not name) are loaded from here: both factors of a product past the end are then zero,
// whatever the memory beside the matrix holds.
__device__ __attribute__((aligned(16))) const uint4 kZeroChunk = {0u, 0u, 0u, 0u};

// A workgroup of WR x WC waves owns a tile of BM = 16 RT WR rows and BN = 16 CT WC columns;
// wave (wr, wc) computes RT x CT matrix-core tiles of 16 x 16.
template <int RT_, int CT_, int WR_, int WC_>
struct LinShape {
  static constexpr int RT = RT_, CT = CT_, WR = WR_, WC = WC_;
  static constexpr int kThreads = 64 * WR * WC;
  static constexpr int BM = 16 * RT * WR, BN = 16 * CT * WC;
};

// How a fragment's lane index i (0..15) of tile t maps to the row of the operand's LDS tile.
//   PLAIN: 16 t + i.
//   WIDE (bf16, k contiguous): tiles in pairs, 32 (t / 2) + 8 (i / 4) + 4 (t % 2) + i % 4, so
//     that a lane ends with 8 consecutive columns of C in the pair's accumulators.
//   BLOCK (fp32, k strided): B = 4 or 2 tiles share each LDS read, 16 B (t / B) + B i + t % B.
enum Map { PLAIN, WIDE, BLOCK };

// Stages one operand's tile of R rows x 128 bytes of k (64 bf16 or 32 fp32) in LDS.
//   KC (k contiguous in memory): LDS [R][8] chunks of 16 bytes; chunk c of row r sits at
//     c ^ key(r), which spreads the 16 rows a fragment read takes over the banks.
//   otherwise (rows of R contiguous elements per k): LDS [k][R]. bf16 tiles are read through
//     the LDS transpose load, 4 k rows x 32 bytes per 16 lanes: 32-byte pairs of chunks sit
//     at pair ^ (k & 3), which puts the 4 rows on different banks.
template <typename T, int R, bool KC, Map MAP, int THREADS>
struct Operand {
  static constexpr int EV = 16 / (int)sizeof(T), BK = 128 / (int)sizeof(T);
  static constexpr int kChunks = R * 8, NCH = kChunks / THREADS;
  static_assert(kChunks % THREADS == 0, "whole chunks per thread");
  static_assert(KC ? (THREADS / 8) % 16 == 0 : (THREADS * EV / R) % 4 == 0, "one swizzle key per thread");

  const T* base[KC ? NCH : 1];
  int64_t ld;             // !KC: elements from k to k + 1
  const int32_t* k_rows;  // !KC: stored row of each k (nullptr: k itself)
  int64_t k_nrows;
  uint32_t ok;            // KC: rows that exist
  int off;                // KC: first k of this thread's chunks; else: its first k row
  int valid;              // !KC: elements of this thread's chunk columns inside the matrix

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
    valid = min(max(lim - g, 0), EV);
    base[0] = p + (valid > 0 ? g : 0);
    ld = ld_;
    k_rows = rows;
    k_nrows = nrows;
  }
  // Address and number of elements of chunk i at k step k0 of a matrix with K k's.
  __device__ __forceinline__ const T* chunk(int i, int k0, int K, int& n) const {
    if constexpr (KC) {
      const int k = k0 + off;
      n = (ok >> i & 1) ? min(max(K - k, 0), EV) : 0;
      return base[i] + k;
    } else {
      const int k = k0 + off + i * (THREADS * EV / R);
      n = k < K ? valid : 0;
      int64_t r = k;
      if (k_rows) {
        r = k < K ? k_rows[k] : 0;
        if (r < 0 || r >= k_nrows) n = 0;
      }
      return base[0] + r * ld;
    }
  }
  // Direct loads: 16-byte aligned chunks, each whole or absent.
  __device__ __forceinline__ void fetch(int k0, int K, uint4* lds) const {
    const int w = (int)threadIdx.x & ~63;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      int n;
      const T* p = chunk(i, k0, K, n);
      load_lds16(n > 0 ? (const void*)p : (const void*)&kZeroChunk, lds + w + i * THREADS);
    }
  }
  // Any alignment: through registers, the partial chunk of a row's end element by element.
  __device__ __forceinline__ void load(int k0, int K, uint4 (&r)[NCH]) const {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      int n;
      const T* p = chunk(i, k0, K, n);
      r[i] = uint4{0u, 0u, 0u, 0u};
      if (n == EV) {
        __builtin_memcpy(&r[i], p, 16);
      } else if (n > 0) {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          if (e >= n) continue;
          if constexpr (sizeof(T) == 2)
            w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e & 1));
          else
            w[e] = reinterpret_cast<const uint32_t*>(p)[e];
        }
        r[i] = uint4{w[0], w[1], w[2], w[3]};
      }
    }
  }
  __device__ __forceinline__ void store(const uint4 (&r)[NCH], uint4* lds) const {
#pragma unroll
    for (int i = 0; i < NCH; ++i) lds[threadIdx.x + i * THREADS] = r[i];
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

// Fragments of NT tiles whose rows start at `row0` of the staged tile, k half s: of bf16 the
// lane's 8 k's 32 s + 8 (lane / 16) .., of fp32 its 4 k's 16 s + 4 (lane / 16) ...
template <typename T, int R, bool KC, Map MAP, int BW, int NT>
__device__ __forceinline__ void read_frags(const uint4* lds, int row0, int s,
                                           typename Frag<T>::type* f) {
  const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
  if constexpr (KC) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = row0 + map_row<MAP, BW>(t, i16);
      const int key = MAP == WIDE ? (r & 3) | ((r >> 3 & 1) << 2) : r & 7;
      f[t] = __builtin_bit_cast(typename Frag<T>::type, lds[r * 8 + ((4 * s + kq) ^ key)]);
    }
  } else if constexpr (sizeof(T) == 2) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4* lds_s4;
    // lane j of a 16-lane group addresses k row j / 4, columns 4 (j % 4) ..; it receives
    // column j of the 4 rows
    const int k = 32 * s + 8 * kq + (i16 >> 2);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int col = row0 + 16 * t + 4 * (i16 & 3);  // first of 4
      const int chunk = (((col >> 4) ^ (k & 3)) << 1) | (col >> 3 & 1);
      const char* p = reinterpret_cast<const char*>(lds) + k * (R * 2) + chunk * 16 + (col & 4) * 2;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 4 * (R * 2)));
      f[t] = __builtin_bit_cast(lin_bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  } else {
    const float* l = reinterpret_cast<const float*>(lds);
#pragma unroll
    for (int t = 0; t < NT; t += BW)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float* p = l + (16 * s + 4 * kq + j) * R + row0 + 16 * t + BW * i16;
        if constexpr (BW == 4) {
          const lin_f32x4 v = *reinterpret_cast<const lin_f32x4*>(p);
#pragma unroll
          for (int b = 0; b < 4; ++b) f[t + b][j] = v[b];
        } else {
          const float2 v = *reinterpret_cast<const float2*>(p);
          f[t][j] = v.x;
          f[t + 1][j] = v.y;
        }
      }
  }
}

__device__ __forceinline__ lin_f32x4 mma(lin_bf16x8 a, lin_bf16x8 b, lin_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ lin_f32x4 mma(lin_f32x4 a, lin_f32x4 b, lin_f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// The main loop: acc += A tile . B tile^T over K. B goes in as the matrix core's first operand,
// so that a lane ends with 4 consecutive n of its own m. VEC: direct global-to-LDS loads one
// step ahead in two buffers; otherwise through registers.
template <typename T, bool VEC, typename SH, typename OA, typename OB, typename F>
__device__ __forceinline__ void main_loop(const OA& oa, const OB& ob, int K, uint4* sA, uint4* sB,
                                          F&& compute) {
  constexpr int BK = OA::BK;
  const int steps = (K + BK - 1) / BK;
  if (steps == 0) return;
  if constexpr (VEC) {
    oa.fetch(0, K, sA);
    ob.fetch(0, K, sB);
    wait_vmcnt<0>();
    lds_barrier();
    for (int kt = 0; kt < steps; ++kt) {
      const int b = kt & 1;
      if (kt + 1 < steps) {
        oa.fetch((kt + 1) * BK, K, sA + (b ^ 1) * OA::kChunks);
        ob.fetch((kt + 1) * BK, K, sB + (b ^ 1) * OB::kChunks);
      }
      compute(sA + b * OA::kChunks, sB + b * OB::kChunks);
      wait_vmcnt<0>();
      lds_barrier();
    }
  } else {
    uint4 ra[OA::NCH], rb[OB::NCH];
    oa.load(0, K, ra);
    ob.load(0, K, rb);
    oa.store(ra, sA);
    ob.store(rb, sB);
    __syncthreads();
    for (int kt = 0; kt < steps; ++kt) {
      const int b = kt & 1;
      if (kt + 1 < steps) {
        oa.load((kt + 1) * BK, K, ra);
        ob.load((kt + 1) * BK, K, rb);
      }
      compute(sA + b * OA::kChunks, sB + b * OB::kChunks);
      if (kt + 1 < steps) {
        oa.store(ra, sA + (b ^ 1) * OA::kChunks);
        ob.store(rb, sB + (b ^ 1) * OB::kChunks);
      }
      __syncthreads();
    }
  }
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

// Row tile t of the launch, tiles counted group by group: its group and first row. 64 groups at a
// time, one per lane. Returns the number of row tiles (t < 0: only that).
template <int BM>
__device__ __forceinline__ int find_tile(const LinearArgs& a, int t, int& group, int& r0, int& r1) {
  const int lane = (int)threadIdx.x & 63;
  int before = 0;
  for (int g0 = 0; g0 <= a.groups; g0 += 64) {
    const int g = g0 + lane;
    int s0 = 0, s1 = 0;
    if (g <= a.groups) group_span(a, g, s0, s1);
    const int nt = s1 > s0 ? (s1 - s0 + BM - 1) / BM : 0;
    int incl = nt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(incl, d, 64);
      if (lane >= d) incl += v;
    }
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (t >= before && t < before + total) {
      // the first lane whose inclusive count passes t
      const int src = (int)__builtin_popcountll(__ballot(before + incl <= t));
      const int first = __builtin_amdgcn_readlane(incl - nt, src);
      group = g0 + src;
      r1 = __builtin_amdgcn_readlane(s1, src);
      r0 = __builtin_amdgcn_readlane(s0, src) + (t - before - first) * BM;
      return 0;
    }
    before += total;
  }
  return before;
}

// Tiles in the order that shares operands through one L2: the launch's tiles are cut into 8
// contiguous ranges, one per XCD (workgroup L runs on XCD L % 8), and run in bands of kBand
// rows of tiles, rows fastest: the 32 CUs of an XCD then work on about 8 x 4 tiles.
constexpr int kBand = 8;
__device__ __forceinline__ bool place_tile(int tiles_r, int tiles_c, int& tr, int& tc) {
  const int total = tiles_r * tiles_c;
  const int L = (int)blockIdx.x, xcd = L % kXcds, slot = L / kXcds;
  const int per = (total + kXcds - 1) / kXcds;
  const int item = xcd * per + slot;
  if (slot >= per || item >= total) return false;
  const int band = item / (kBand * tiles_c), in = item - band * kBand * tiles_c;
  const int rows = min(kBand, tiles_r - band * kBand);
  tr = band * kBand + in % rows;
  tc = in / rows;
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

// The n of C that a lane holds, in runs of W consecutive ones: run g, element q is element e of
// tile t.
template <Map MAP, int BW>
struct Runs {
  static constexpr int W = MAP == WIDE ? 8 : MAP == BLOCK ? BW : 4;
  __device__ __forceinline__ static constexpr int tile(int g, int q) {
    return MAP == WIDE ? 2 * g + (q >> 2) : MAP == BLOCK ? BW * (g / 4) + q : g;
  }
  __device__ __forceinline__ static constexpr int elem(int g, int q) {
    return MAP == WIDE ? q & 3 : MAP == BLOCK ? g % 4 : q;
  }
  __device__ __forceinline__ static int col(int g, int kq) {
    return MAP == WIDE ? 32 * g + 8 * kq
         : MAP == BLOCK ? 16 * BW * (g / 4) + BW * (4 * kq + g % 4)
                        : 16 * g + 4 * kq;
  }
};

template <typename T, bool KC>
constexpr Map out_map() {
  return KC ? (sizeof(T) == 2 ? WIDE : PLAIN) : (sizeof(T) == 2 ? PLAIN : BLOCK);
}

// Products over ragged rows: C[i][n] = epi(sum_k A[row(i)][k] B_group[n][k]). PAIR (SwiGLU): a
// tile's columns are BN / 2 gate columns and their up-projection twins N / 2 further on.
template <typename T, bool BKC, bool PAIR, bool VEC, typename SH>
__global__ void __launch_bounds__(SH::kThreads, 2) linear_rows_kernel(LinearArgs a) {
  constexpr int RT = SH::RT, CT = SH::CT, BM = SH::BM, BN = SH::BN;
  constexpr Map MAP = out_map<T, BKC>();
  constexpr int NCT = PAIR ? CT / 2 : CT;  // tiles of output columns per wave
  constexpr int BW = NCT >= 4 ? 4 : 2;
  static_assert(MAP == PLAIN || NCT % (MAP == WIDE ? 2 : BW) == 0, "whole runs per wave");
  typedef Operand<T, BM, true, PLAIN, SH::kThreads> OA;
  typedef Operand<T, BN, BKC, MAP, SH::kThreads> OB;
  __shared__ uint4 sA[2 * OA::kChunks], sB[2 * OB::kChunks];

  const int f = PAIR ? a.N / 2 : a.N;          // output columns
  constexpr int OBN = PAIR ? BN / 2 : BN;      // output columns of a tile
  const int tiles_c = (f + OBN - 1) / OBN;
  int group = 0, r0 = 0, r1 = 0, tr, tc;
  const int tiles_r = find_tile<BM>(a, -1, group, r0, r1);
  if (!place_tile(tiles_r, tiles_c, tr, tc)) return;
  find_tile<BM>(a, tr, group, r0, r1);
  const int n0 = tc * OBN;
  const bool none = group >= a.groups;  // rows of no group: zeros
  const int K = none ? 0 : a.K;

  const T* A = reinterpret_cast<const T*>(a.A);
  const T* B = reinterpret_cast<const T*>(a.B) + (none ? 0 : group) * a.b_group;
  OA oa;
  oa.init_kc([&](int r) -> const T* {
    int64_t i = min(r0 + r, r1 - 1);
    if (a.a_rows) {
      i = none ? 0 : a.a_rows[i];
      if (i < 0 || i >= a.a_nrows) return nullptr;
    }
    return A + i * a.lda;
  });
  OB ob;
  if constexpr (BKC) {
    ob.init_kc([&](int c) -> const T* {
      const int64_t n = PAIR ? (c < OBN ? min(n0 + c, f - 1) : f + min(n0 + c - OBN, f - 1))
                             : min(n0 + c, f - 1);
      return B + n * a.ldb;
    });
  } else {
    ob.init_nc(B, a.ldb, nullptr, 0, [&](int c, int& lim) {
      const bool up = PAIR && c >= OBN;
      lim = up ? a.N : f;
      return up ? f + n0 + c - OBN : n0 + c;
    });
  }

  const int lane = (int)threadIdx.x & 63, wv = (int)threadIdx.x >> 6;
  const int wr = wv / SH::WC, wc = wv % SH::WC;
  const int i16 = lane & 15, kq = lane >> 4;
  const int row_w = wr * RT * 16, col_w = wc * NCT * 16;
  lin_f32x4 acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = lin_f32x4{0.f, 0.f, 0.f, 0.f};

  main_loop<T, VEC, SH>(oa, ob, K, sA, sB, [&](const uint4* la, const uint4* lb) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename Frag<T>::type fa[RT], fb[CT];
      read_frags<T, BM, true, PLAIN, 1, RT>(la, row_w, s, fa);
      read_frags<T, BN, BKC, MAP, BW, NCT>(lb, col_w, s, fb);
      if constexpr (PAIR) read_frags<T, BN, BKC, MAP, BW, NCT>(lb, OBN + col_w, s, fb + NCT);
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
    }
  });

  // epilogue in fp32, one rounding per output
  typedef Runs<MAP, BW> RN;
  constexpr int W = RN::W, NG = NCT * 4 / W;
  T* C = reinterpret_cast<T*>(a.C);
  T* pre = reinterpret_cast<T*>(a.pre);
  const T* res = reinterpret_cast<const T*>(a.residual);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int col = n0 + col_w + RN::col(g, kq), n = f - col;
    if (n <= 0) continue;
    float bias[2][W];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < W; ++q) bias[h][q] = 0.f;
    if (a.bias && !none) {
#pragma unroll
      for (int h = 0; h < (PAIR ? 2 : 1); ++h) {
        const int64_t o = (int64_t)group * a.N + col + h * f;
        if (a.bias_dtype == PULSAR_F32)
          load_run<W>(reinterpret_cast<const float*>(a.bias) + o, bias[h], n);
        else
          load_run<W>(reinterpret_cast<const bf16*>(a.bias) + o, bias[h], n);
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t r = r0 + row_w + 16 * i + i16;
      if (r >= r1) continue;
      float v[W], u[W];
#pragma unroll
      for (int q = 0; q < W; ++q) {
        v[q] = acc[i][RN::tile(g, q)][RN::elem(g, q)] + bias[0][q];
        u[q] = PAIR ? acc[i][(PAIR ? NCT : 0) + RN::tile(g, q)][RN::elem(g, q)] + bias[1][q] : 0.f;
      }
      if (pre) {
        store_run<W>(pre + r * a.ldpre + col, v, n);
        if constexpr (PAIR) store_run<W>(pre + r * a.ldpre + f + col, u, n);
      }
      if constexpr (PAIR) {
#pragma unroll
        for (int q = 0; q < W; ++q) v[q] = v[q] * sigmoidf_(v[q]) * u[q];
      } else if (a.act != PULSAR_ACT_NONE && !none) {
#pragma unroll
        for (int q = 0; q < W; ++q) v[q] = act_value(a.act, v[q]);
      }
      if (res) {
        float x[W];
        load_run<W>(res + r * a.ldr + col, x, n);
#pragma unroll
        for (int q = 0; q < W; ++q) v[q] += x[q];
      }
      store_run<W>(C + r * a.ldc + col, v, n);
    }
  }
}

// Weight gradient: C_group[m][n] = sum over the group's rows r of A[r][m] B[r][n], rows through
// the optional indices. SIDE: the operand whose column sums (the bias gradient) are taken
// along, by one more product with ones in the tiles at 0 of the other dimension (0 none, 1 A,
// 2 B).
template <typename T, bool VEC, int SIDE, typename SH>
__global__ void __launch_bounds__(SH::kThreads, 2) linear_wgrad_kernel(LinearArgs a) {
  constexpr int RT = SH::RT, CT = SH::CT, BM = SH::BM, BN = SH::BN;
  constexpr Map MAP = out_map<T, false>();
  constexpr int BWR = RT >= 4 ? 4 : 2, BWC = CT >= 4 ? 4 : 2;
  typedef Operand<T, BM, false, MAP, SH::kThreads> OA;
  typedef Operand<T, BN, false, MAP, SH::kThreads> OB;
  __shared__ uint4 sA[2 * OA::kChunks], sB[2 * OB::kChunks];

  // (group, split, row of tiles) are the rows of the launch's tiles
  int tr, tc;
  if (!place_tile(a.groups * a.splits * a.tiles_m, a.tiles_n, tr, tc)) return;
  const int mt = tr % a.tiles_m, gs = tr / a.tiles_m, split = gs % a.splits, group = gs / a.splits;
  int r0, r1;
  group_span(a, group, r0, r1);
  r1 = max(r0, r1);
  if (a.splits > 1) {
    const int per = ((r1 - r0 + a.splits - 1) / a.splits + OA::BK - 1) / OA::BK * OA::BK;
    r0 = min(r0 + split * per, r1);
    r1 = min(r0 + per, r1);
  }
  const int m0 = mt * BM, n0 = tc * BN;
  OA oa;
  OB ob;
  // without an index the stored rows start at r0; with one the index does
  oa.init_nc(reinterpret_cast<const T*>(a.A) + (a.a_rows ? 0 : r0 * a.lda), a.lda,
             a.a_rows ? a.a_rows + r0 : nullptr, a.a_nrows, [&](int c, int& lim) {
               lim = a.M;
               return m0 + c;
             });
  ob.init_nc(reinterpret_cast<const T*>(a.B) + (a.b_rows ? 0 : r0 * a.ldb), a.ldb,
             a.b_rows ? a.b_rows + r0 : nullptr, a.b_nrows, [&](int c, int& lim) {
               lim = a.N;
               return n0 + c;
             });

  const int lane = (int)threadIdx.x & 63, wv = (int)threadIdx.x >> 6;
  const int wr = wv / SH::WC, wc = wv % SH::WC;
  const int i16 = lane & 15, kq = lane >> 4;
  const int row_w = wr * RT * 16, col_w = wc * CT * 16;
  lin_f32x4 acc[RT][CT], sum[SIDE == 1 ? RT : CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = lin_f32x4{0.f, 0.f, 0.f, 0.f};
  typename Frag<T>::type ones;
#pragma unroll
  for (int e = 0; e < OA::EV; ++e) ones[e] = 1.f;
  const bool sums = SIDE == 1 ? tc == 0 && wc == 0 : SIDE == 2 ? mt == 0 && wr == 0 : false;
  if constexpr (SIDE != 0) {
#pragma unroll
    for (int i = 0; i < (SIDE == 1 ? RT : CT); ++i) sum[i] = lin_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  main_loop<T, VEC, SH>(oa, ob, r1 - r0, sA, sB, [&](const uint4* la, const uint4* lb) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename Frag<T>::type fa[RT], fb[CT];
      read_frags<T, BM, false, MAP, BWR, RT>(la, row_w, s, fa);
      read_frags<T, BN, false, MAP, BWC, CT>(lb, col_w, s, fb);
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
      if constexpr (SIDE == 1) {
        if (sums)
#pragma unroll
          for (int i = 0; i < RT; ++i) sum[i] = mma(ones, fa[i], sum[i]);
      }
      if constexpr (SIDE == 2) {
        if (sums)
#pragma unroll
          for (int j = 0; j < CT; ++j) sum[j] = mma(fb[j], ones, sum[j]);
      }
    }
  });

  typedef Runs<MAP, BWC> RN;
  constexpr int W = RN::W, NG = CT * 4 / W;
  const int64_t pg = (int64_t)split * a.groups + group;  // a split's partial results
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int col = n0 + col_w + RN::col(g, kq), n = a.N - col;
    if (n <= 0) continue;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t m = m0 + row_w + map_row<MAP, BWR>(i, i16);
      if (m >= a.M) continue;
      float v[W];
#pragma unroll
      for (int q = 0; q < W; ++q) v[q] = acc[i][RN::tile(g, q)][RN::elem(g, q)];
      if (a.splits > 1)
        store_run<W>(a.part + (pg * a.M + m) * a.N + col, v, n);
      else
        store_run<W>(reinterpret_cast<T*>(a.C) + group * a.c_group + m * a.ldc + col, v, n);
    }
    if constexpr (SIDE == 2) {
      if (sums && i16 == 0) {
        float v[W];
#pragma unroll
        for (int q = 0; q < W; ++q) v[q] = sum[RN::tile(g, q)][RN::elem(g, q)];
        if (a.splits > 1)
          store_run<W>(a.part_db + pg * a.N + col, v, n);
        else
          store_run<W>(reinterpret_cast<T*>(a.db) + (int64_t)group * a.N + col, v, n);
      }
    }
  }
  if constexpr (SIDE == 1) {
    if (sums && kq == 0) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int m = m0 + row_w + map_row<MAP, BWR>(i, i16);
        if (m >= a.M) continue;
        if (a.splits > 1)
          a.part_db[pg * a.M + m] = sum[i][0];
        else
          reinterpret_cast<T*>(a.db)[(int64_t)group * a.M + m] = from_f<T>(sum[i][0]);
      }
    }
  }
}

// Sums of a weight gradient's splits, in order; `count` elements of one split's partials, the
// first `n_c` of them C's (contiguous), the rest db's.
template <typename T>
__global__ void __launch_bounds__(256) linear_merge_kernel(const float* part, const float* part_db,
                                                           T* C, T* db, int64_t n_c, int64_t n_db,
                                                           int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const bool is_db = i >= (n_c + 3) / 4 * 4;
  const int64_t k = is_db ? i - (n_c + 3) / 4 * 4 : i, cnt = is_db ? n_db : n_c;
  if (k >= cnt) return;
  const float* p = (is_db ? part_db : part) + k;
  const int n = (int)min(cnt - k, (int64_t)4);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int sp = 0; sp < splits; ++sp) {
    float v[4];
    load_run<4>(p + sp * cnt, v, n);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += v[e];
  }
  store_run<4>((is_db ? db : C) + k, s, n);
}

// dpre = act'(pre) dy over [rows][N]; SwiGLU: pre [rows][2 f], dy [rows][f]. W elements a
// thread, 16 bytes where the rows allow it.
template <typename T, int W>
__global__ void __launch_bounds__(256) linear_act_grad_kernel(const T* pre, const T* dy, T* dpre,
                                                              int64_t rows, int f, int act) {
  const int per = (f + W - 1) / W;
  const int64_t total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * W, n = f - c;
    float g[W], d[W], o[W];
    load_run<W>(dy + r * f + c, d, n);
    if (act == PULSAR_ACT_SWIGLU) {
      float u[W], ou[W];
      load_run<W>(pre + r * 2 * f + c, g, n);
      load_run<W>(pre + r * 2 * f + f + c, u, n);
#pragma unroll
      for (int q = 0; q < W; ++q) {
        ou[q] = d[q] * g[q] * sigmoidf_(g[q]);
        o[q] = d[q] * u[q] * act_slope(PULSAR_ACT_SILU, g[q]);
      }
      store_run<W>(dpre + r * 2 * f + c, o, n);
      store_run<W>(dpre + r * 2 * f + f + c, ou, n);
    } else {
      load_run<W>(pre + r * f + c, g, n);
#pragma unroll
      for (int q = 0; q < W; ++q) o[q] = d[q] * act_slope(act, g[q]);
      store_run<W>(dpre + r * f + c, o, n);
    }
  }
}

typedef LinShape<4, 4, 2, 2> LinLarge;  // 128 x 128
typedef LinShape<2, 4, 2, 2> LinSmall;  // 64 x 128

template <typename T, bool BKC, bool PAIR, bool VEC, typename SH>
int launch_rows_shape(LinearArgs& a, hipStream_t s) {
  const int f = PAIR ? a.N / 2 : a.N, obn = PAIR ? SH::BN / 2 : SH::BN;
  // every group adds at most one partial tile to the whole ones
  const int64_t tiles_r = a.offsets
      ? a.rows / SH::BM + std::min<int64_t>(a.groups + 1, a.rows)
      : (a.rows + SH::BM - 1) / SH::BM;
  const int64_t tiles = tiles_r * ((f + obn - 1) / obn);
  if (tiles > (int64_t)1 << 30) return fail(PULSAR_ERR_INVALID, "linear: launch too large");
  linear_rows_kernel<T, BKC, PAIR, VEC, SH>
      <<<(unsigned)((tiles + kXcds - 1) / kXcds * kXcds), SH::kThreads, 0, s>>>(a);
  PULSAR_LAUNCH_CHECK();
  return PULSAR_OK;
}

template <typename T>
int launch_rows(LinearArgs& a, bool b_kc, hipStream_t s) {
  const int ev = 16 / (int)sizeof(T);
  const bool pair = a.act == PULSAR_ACT_SWIGLU;
  const int f = pair ? a.N / 2 : a.N;
  const bool vec = aligned16(a.A) && aligned16(a.B) && a.lda % ev == 0 && a.ldb % ev == 0 &&
                   a.b_group % ev == 0 && a.K % ev == 0 && (b_kc || f % ev == 0);
  const int64_t t128 = ((a.rows + 127) / 128) * (((int64_t)a.N + 127) / 128);
  const bool large = t128 >= 256;
  auto go = [&](auto kc, auto pr, auto vc) {
    constexpr bool KC = decltype(kc)::value, P = decltype(pr)::value, V = decltype(vc)::value;
    if (large) return launch_rows_shape<T, KC, P, V, LinLarge>(a, s);
    return launch_rows_shape<T, KC, P, V, LinSmall>(a, s);
  };
  auto pick_vec = [&](auto kc, auto pr) {
    return vec ? go(kc, pr, std::true_type{}) : go(kc, pr, std::false_type{});
  };
  auto pick_pair = [&](auto kc) {
    return pair ? pick_vec(kc, std::true_type{}) : pick_vec(kc, std::false_type{});
  };
  return b_kc ? pick_pair(std::true_type{}) : pick_pair(std::false_type{});
}

// Rows of each of a weight gradient's splits: enough workgroups to fill the chip twice where
// the tiles alone do not, no split shorter than 512 rows. The bound is the average group.
int wgrad_splits(int64_t rows, int groups, int64_t tiles) {
  if (tiles >= 384) return 1;
  const int64_t avg = rows / std::max(groups, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(tiles, 1), avg / 512));
}
int64_t wgrad_tiles(int64_t d_in, int64_t d_out, int groups) {
  return ((d_in + 127) / 128) * ((d_out + 127) / 128) * groups;
}

template <typename T>
int launch_wgrad(LinearArgs& a, bool vec, int side, hipStream_t s) {
  typedef LinLarge SH;
  a.tiles_m = (a.M + SH::BM - 1) / SH::BM;
  a.tiles_n = (a.N + SH::BN - 1) / SH::BN;
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n * a.groups * a.splits;
  if (tiles > (int64_t)1 << 30) return fail(PULSAR_ERR_INVALID, "linear: launch too large");
  const unsigned grid = (unsigned)((tiles + kXcds - 1) / kXcds * kXcds);
  auto go = [&](auto v, auto sd) {
    linear_wgrad_kernel<T, decltype(v)::value, decltype(sd)::value, SH><<<grid, SH::kThreads, 0, s>>>(a);
  };
  auto pick = [&](auto v) {
    if (side == 0) go(v, std::integral_constant<int, 0>{});
    else if (side == 1) go(v, std::integral_constant<int, 1>{});
    else go(v, std::integral_constant<int, 2>{});
  };
  if (vec) pick(std::true_type{});
  else pick(std::false_type{});
  PULSAR_LAUNCH_CHECK();
  if (a.splits > 1) {
    const int64_t n_c = (int64_t)a.groups * a.M * a.N;
    const int64_t n_db = side == 0 ? 0 : (int64_t)a.groups * (side == 1 ? a.M : a.N);
    linear_merge_kernel<T><<<blocks_for((n_c + 3) / 4 + (n_db + 3) / 4, 256), 256, 0, s>>>(
        a.part, a.part_db, reinterpret_cast<T*>(a.C), reinterpret_cast<T*>(a.db), n_c, n_db, a.splits);
    PULSAR_LAUNCH_CHECK();
  }
  return PULSAR_OK;
}

// The checks and the launch that dense and grouped calls share. Weight element (e, i, o) is
// w[e w_group + i w_in + o w_out], one of w_in and w_out 1.
struct Weight {
  const void* p;
  int64_t group, in, out;
};

int check_common(int64_t rows, int64_t groups, int64_t d_in, int64_t d_out, const Weight& w,
                 int act, int dtype, const char* what) {
  const std::string n = std::string(what) + ": ";
  if (dtype != PULSAR_F32 && dtype != PULSAR_BF16)
    return fail(PULSAR_ERR_INVALID, n + "dtype must be PULSAR_F32 or PULSAR_BF16");
  if (rows < 0 || d_in < 1 || d_out < 1 || groups < 1 || rows > 0x7fffff00 || d_in > 0x7fffff00 ||
      d_out > 0x7fffff00 || groups > 65536)
    return fail(PULSAR_ERR_INVALID, n + "bad shape");
  if (act < PULSAR_ACT_NONE || act > PULSAR_ACT_SWIGLU)
    return fail(PULSAR_ERR_INVALID, n + "unknown activation");
  if (act == PULSAR_ACT_SWIGLU && d_out % 2 != 0)
    return fail(PULSAR_ERR_INVALID, n + "swiglu needs an even number of output columns");
  if (w.in != 1 && w.out != 1)
    return fail(PULSAR_ERR_INVALID, n + "one of the weight's strides must be 1");
  if (w.in < 1 || w.out < 1 || w.group < 0 || (w.in == 1 && d_out > 1 && w.out < d_in) ||
      (w.in != 1 && d_in > 1 && w.in < d_out))
    return fail(PULSAR_ERR_INVALID, n + "weight rows overlap");
  return PULSAR_OK;
}

// Whether the weight is stored with its input dimension contiguous.
bool in_contiguous(const Weight& w) { return w.in == 1; }

int forward(const void* x, int64_t x_rs, int64_t x_rows, const int32_t* index, const Weight& w,
            const void* bias, int bias_dtype, const void* residual, int64_t res_rs, void* y,
            void* pre, const int32_t* offsets, int64_t groups, int64_t rows, int64_t d_in,
            int64_t d_out, int act, int dtype, hipStream_t s) {
  if (rows == 0) return PULSAR_OK;
  LinearArgs a = {};
  const bool kc = in_contiguous(w);
  a.A = x; a.lda = x_rs; a.a_rows = index; a.a_nrows = x_rows;
  a.B = w.p; a.ldb = kc ? w.out : w.in; a.b_group = w.group;
  a.offsets = offsets; a.groups = (int)groups; a.rows = (int)rows;
  a.N = (int)d_out; a.K = (int)d_in;
  a.C = y; a.ldc = act == PULSAR_ACT_SWIGLU ? d_out / 2 : d_out;
  a.pre = pre; a.ldpre = d_out;
  a.bias = bias; a.bias_dtype = bias_dtype;
  a.residual = residual; a.ldr = res_rs;
  a.act = act;
  return dtype == PULSAR_BF16 ? launch_rows<bf16>(a, kc, s) : launch_rows<float>(a, kc, s);
}

int64_t workspace_bytes(int64_t rows, int64_t groups, int64_t d_in, int64_t d_out, int act,
                        int dtype) {
  if (rows < 0 || groups < 1 || d_in < 1 || d_out < 1) return -1;
  const int64_t es = dtype == PULSAR_BF16 ? 2 : 4;
  const int64_t dpre = act == PULSAR_ACT_NONE ? 0 : (rows * d_out * es + 255) / 256 * 256;
  const int splits = wgrad_splits(rows, (int)groups, wgrad_tiles(d_in, d_out, (int)groups));
  const int64_t part = splits > 1 ? splits * groups * (d_in * d_out + d_out) * 4 : 0;
  return dpre + part;
}

template <typename T>
int backward_t(const void* dy, const void* x, int64_t x_rs, int64_t x_rows, const int32_t* index,
               const Weight& w, const void* pre, void* dx, void* dw, void* db,
               const int32_t* offsets, int64_t groups, int64_t rows, int64_t d_in, int64_t d_out,
               int act, void* workspace, hipStream_t s) {
  const int ev = 16 / (int)sizeof(T);
  const void* dpre = dy;
  char* ws = static_cast<char*>(workspace);
  if (act != PULSAR_ACT_NONE && rows > 0) {
    const int f = (int)(act == PULSAR_ACT_SWIGLU ? d_out / 2 : d_out);
    const int64_t n = rows * ((f + ev - 1) / ev);
    linear_act_grad_kernel<T, 16 / (int)sizeof(T)>
        <<<(unsigned)std::min<int64_t>((n + 255) / 256, 8192), 256, 0, s>>>(
            static_cast<const T*>(pre), static_cast<const T*>(dy), reinterpret_cast<T*>(ws), rows,
            f, act);
    PULSAR_LAUNCH_CHECK();
    dpre = ws;
    ws += (rows * d_out * (int64_t)sizeof(T) + 255) / 256 * 256;
  }
  const bool kc = in_contiguous(w);
  if (rows > 0) {
    LinearArgs a = {};
    a.A = dpre; a.lda = d_out; a.a_nrows = rows;
    // dx = dpre w^T: n is the input dimension, k the output one
    a.B = w.p; a.ldb = kc ? w.out : w.in; a.b_group = w.group;
    a.offsets = offsets; a.groups = (int)groups; a.rows = (int)rows;
    a.N = (int)d_in; a.K = (int)d_out;
    a.C = dx; a.ldc = d_in;
    a.act = PULSAR_ACT_NONE;
    const int rc = launch_rows<T>(a, !kc, s);
    if (rc != PULSAR_OK) return rc;
  }
  LinearArgs a = {};
  // C in the weight's own order: its contiguous dimension is n
  const bool dpre_a = kc;
  if (dpre_a) {
    a.A = dpre; a.lda = d_out; a.a_nrows = rows; a.M = (int)d_out;
    a.B = x; a.ldb = x_rs; a.b_rows = index; a.b_nrows = x_rows; a.N = (int)d_in;
  } else {
    a.A = x; a.lda = x_rs; a.a_rows = index; a.a_nrows = x_rows; a.M = (int)d_in;
    a.B = dpre; a.ldb = d_out; a.b_nrows = rows; a.N = (int)d_out;
  }
  a.offsets = offsets; a.groups = (int)groups; a.rows = (int)rows;
  a.C = dw; a.ldc = a.N; a.c_group = (int64_t)a.M * a.N;
  a.db = db;
  a.splits = wgrad_splits(rows, (int)groups, wgrad_tiles(d_in, d_out, (int)groups));
  if (a.splits > 1) {
    a.part = reinterpret_cast<float*>(ws);
    a.part_db = a.part + (int64_t)a.splits * groups * d_in * d_out;
  }
  const bool vec = aligned16(a.A) && aligned16(a.B) && a.lda % ev == 0 && a.ldb % ev == 0 &&
                   a.M % ev == 0 && a.N % ev == 0;
  return launch_wgrad<T>(a, vec, db ? (dpre_a ? 1 : 2) : 0, s);
}

int null_check(const char* what) {
  return fail(PULSAR_ERR_INVALID, std::string(what) + ": null pointer");
}

int backward(const void* dy, const void* x, int64_t x_rs, int64_t x_rows, const int32_t* index,
             const Weight& w, const void* pre, void* dx, void* dw, void* db, const int32_t* offsets,
             int64_t groups, int64_t rows, int64_t d_in, int64_t d_out, int act, int dtype,
             void* workspace, hipStream_t s, const char* what) {
  const int rc = check_common(rows, groups, d_in, d_out, w, act, dtype, what);
  if (rc != PULSAR_OK) return rc;
  if (!dw || (rows > 0 && (!dy || (!x && x_rows > 0) || !w.p || !dx || (act != PULSAR_ACT_NONE && !pre))))
    return null_check(what);
  if (rows > 0 && x_rs < d_in && x_rows > 1)
    return fail(PULSAR_ERR_INVALID, std::string(what) + ": rows of x overlap");
  if (workspace_bytes(rows, groups, d_in, d_out, act, dtype) > 0 &&
      (!workspace || !aligned16(workspace)))
    return fail(PULSAR_ERR_INVALID, std::string(what) + ": workspace missing or not 16-byte aligned");
  if (dtype == PULSAR_BF16)
    return backward_t<bf16>(dy, x, x_rs, x_rows, index, w, pre, dx, dw, db, offsets, groups, rows,
                            d_in, d_out, act, workspace, s);
  return backward_t<float>(dy, x, x_rs, x_rows, index, w, pre, dx, dw, db, offsets, groups, rows,
                           d_in, d_out, act, workspace, s);
}

int forward_checked(const void* x, int64_t x_rs, int64_t x_rows, const int32_t* index,
                    const Weight& w, const void* bias, int bias_dtype, const void* residual,
                    int64_t res_rs, void* y, void* pre, const int32_t* offsets, int64_t groups,
                    int64_t rows, int64_t d_in, int64_t d_out, int act, int dtype, hipStream_t s,
                    const char* what) {
  const int rc = check_common(rows, groups, d_in, d_out, w, act, dtype, what);
  if (rc != PULSAR_OK) return rc;
  if (rows > 0 && (!y || (!x && x_rows > 0) || !w.p)) return null_check(what);
  if (bias && bias_dtype != PULSAR_F32 && bias_dtype != PULSAR_BF16)
    return fail(PULSAR_ERR_INVALID, std::string(what) + ": bias dtype must be PULSAR_F32 or PULSAR_BF16");
  if (rows > 0 && x_rs < d_in && x_rows > 1)
    return fail(PULSAR_ERR_INVALID, std::string(what) + ": rows of x overlap");
  return forward(x, x_rs, x_rows, index, w, bias, bias_dtype, residual, res_rs, y, pre, offsets,
                 groups, rows, d_in, d_out, act, dtype, s);
}

}  // namespace

}  // namespace pulsar

using namespace pulsar;

extern "C" {

int pulsar_fused_linear_forward(const void* x, int64_t x_rs, const void* w, int64_t w_out,
                                int64_t w_in, const void* bias, int bias_dtype,
                                const void* residual, int64_t residual_rs, void* y, void* pre,
                                int64_t rows, int64_t d_in, int64_t d_out, int activation,
                                int dtype, hipStream_t stream) {
  return forward_checked(x, x_rs, rows, nullptr, Weight{w, 0, w_in, w_out}, bias, bias_dtype,
                         residual, residual_rs, y, pre, nullptr, 1, rows, d_in, d_out, activation,
                         dtype, stream, "fused_linear_forward");
}

int64_t pulsar_fused_linear_backward_workspace_bytes(int64_t rows, int64_t d_in, int64_t d_out,
                                                     int activation, int dtype) {
  return workspace_bytes(rows, 1, d_in, d_out, activation, dtype);
}

int pulsar_fused_linear_backward(const void* dy, const void* x, int64_t x_rs, const void* w,
                                 int64_t w_out, int64_t w_in, const void* pre, void* dx, void* dw,
                                 void* db, int64_t rows, int64_t d_in, int64_t d_out,
                                 int activation, int dtype, void* workspace, hipStream_t stream) {
  return backward(dy, x, x_rs, rows, nullptr, Weight{w, 0, w_in, w_out}, pre, dx, dw, db, nullptr,
                  1, rows, d_in, d_out, activation, dtype, workspace, stream,
                  "fused_linear_backward");
}

int pulsar_grouped_linear_forward(const void* x, int64_t x_rs, int64_t x_rows,
                                  const int32_t* row_index, const int32_t* offsets, const void* w,
                                  int64_t w_group, int64_t w_in, int64_t w_out, const void* bias,
                                  int bias_dtype, void* y, void* pre, int64_t rows,
                                  int64_t groups, int64_t d_in, int64_t d_out, int activation,
                                  int dtype, hipStream_t stream) {
  PULSAR_REQUIRE(offsets, "grouped_linear_forward: null pointer");
  return forward_checked(x, x_rs, x_rows, row_index, Weight{w, w_group, w_in, w_out}, bias,
                         bias_dtype, nullptr, 0, y, pre, offsets, groups, rows, d_in, d_out,
                         activation, dtype, stream, "grouped_linear_forward");
}

int64_t pulsar_grouped_linear_backward_workspace_bytes(int64_t rows, int64_t groups, int64_t d_in,
                                                       int64_t d_out, int activation, int dtype) {
  return workspace_bytes(rows, groups, d_in, d_out, activation, dtype);
}

int pulsar_grouped_linear_backward(const void* dy, const void* x, int64_t x_rs, int64_t x_rows,
                                   const int32_t* row_index, const int32_t* offsets, const void* w,
                                   int64_t w_group, int64_t w_in, int64_t w_out, const void* pre,
                                   void* dx, void* dw, void* db, int64_t rows, int64_t groups,
                                   int64_t d_in, int64_t d_out, int activation, int dtype,
                                   void* workspace, hipStream_t stream) {
  PULSAR_REQUIRE(offsets, "grouped_linear_backward: null pointer");
  return backward(dy, x, x_rs, x_rows, row_index, Weight{w, w_group, w_in, w_out}, pre, dx, dw, db,
                  offsets, groups, rows, d_in, d_out, activation, dtype, workspace, stream,
                  "grouped_linear_backward");
}

}  // extern "C"
