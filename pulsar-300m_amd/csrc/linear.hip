// Dense and ragged (grouped by expert) products with bias, activation and residual in the
// epilogue, and their gradients: fused_linear_* and grouped_linear_* of the op surface.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "linear_device.h"

namespace pulsar {

namespace {

// Products over ragged rows: C[i][n] = epi(sum_k A[row(i)][k] B_group[n][k]). PAIR (SwiGLU): a
// tile's columns are BN / 2 gate columns and their up-projection twins.
template <typename T, bool BKC, bool PAIR, typename SH>
__device__ __forceinline__ void rows_tile(const LinearArgs& a, uint4* lds, int tc, int group, int r0, int r1) {
  constexpr int RT = SH::RT, CT = SH::CT, BM = SH::BM, BN = SH::BN;
  constexpr Map MAP = out_map<T, BKC>();
  constexpr int NCT = PAIR ? CT / 2 : CT;  // tiles of output columns per wave
  constexpr int BW = NCT >= 4 ? 4 : 2;
  static_assert(CT == Slab::CT, "the epilogue's rows");
  typedef Operand<T, BM, true, PLAIN, SH::kThreads> OA;
  typedef Operand<T, BN, BKC, MAP, SH::kThreads> OB;
  uint4 *sA = lds, *sB = lds + 2 * OA::kChunks;
  static_assert(2 * (OA::kChunks + OB::kChunks) * 16 >= SH::WR * SH::WC * Slab::kFloats * 4,
                "the epilogue's rows fit");

  const int f = PAIR ? a.N / 2 : a.N;          // output columns
  constexpr int OBN = PAIR ? BN / 2 : BN;      // output columns of a tile
  const int n0 = tc * OBN;
  const bool none = group >= a.groups;  // rows of no group: zeros
  constexpr bool SPLIT = !SH::kShared;
  int kfirst = 0, K = none ? 0 : a.K;
  if (SPLIT && a.part) split_range<T>(K, a.splits, (int)blockIdx.y, kfirst, K);

  const T* A = reinterpret_cast<const T*>(a.A) + kfirst;
  const T* B = reinterpret_cast<const T*>(a.B) + (none ? 0 : group) * a.b_group + kfirst * (BKC ? 1 : a.ldb);
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
      const int64_t n = PAIR ? (c < OBN ? min(n0 + c, f - 1) : a.up + min(n0 + c - OBN, f - 1))
                             : min(n0 + c, f - 1);
      return B + n * a.ldb;
    });
  } else {
    ob.init_nc(B, a.ldb, nullptr, 0, [&](int c, int& lim) {
      const bool up = PAIR && c >= OBN;
      lim = up ? a.up + f : f;
      return up ? a.up + n0 + c - OBN : n0 + c;
    });
  }

  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row_w = wv / SH::WC * RT * 16, col_w = wv % SH::WC * NCT * 16;
  lin_f32x4 acc[RT][CT];
  clear(acc);
  bool again = true;  // fp32: the split products, and the plain ones where they were not finite
  if constexpr (sizeof(T) == 4) {
    const SplitReader<BM, true, 1> ra(row_w);
    const SplitReader<BN, BKC, BW> rb(col_w), ru(OBN + col_w);
    auto read_b = [&](const uint4* lb, float(&x)[CT][8]) {
      constexpr int BT = decltype(rb)::kTiles;
#pragma unroll
      for (int j = 0; j < NCT; j += BT) {
        rb.read(lb, j, x + j);
        if constexpr (PAIR) ru.read(lb, j, x + NCT + j);
      }
    };
    split_loop<SH>(oa, ob, K, sA, sB, acc, ra, read_b, [](int, const Split&, Split(&)[CT]) {});
    again = any_not_finite(acc);
    if (again) clear(acc);
  }
  if (again) {
    typedef typename Frag<T>::type F;
    const Reader<T, BM, true, PLAIN, 1, RT> ra(row_w);
    const Reader<T, BN, BKC, MAP, BW, NCT> rb(col_w), ru(OBN + col_w);
    auto read_b = [&](const uint4* lb, int s, F(&fb)[CT]) {
      rb.read(lb, s, fb);
      if constexpr (PAIR) ru.read(lb, s, fb + NCT);
    };
    pipe_loop<T, SH>(oa, ob, K, sA, sB, acc, ra, read_b, [](int, const F&, F(&)[CT]) {});
  }

  __syncthreads();  // the tiles' memory now holds the epilogue's rows
  const Slab slab{reinterpret_cast<float*>(lds) + wv * Slab::kFloats};
  const EpilogueBias<T, MAP, PAIR> bias(a, group, none, n0 + col_w, f);
  rows_epilogue<T, MAP, BW, PAIR, SPLIT>(a, acc, slab, bias, none, r0 + row_w, r1, n0 + col_w, f);
}

// One workgroup a tile. With one workgroup a CU (256 x 256) the tiles that do not fill a whole
// round of an XCD's 32 CUs would still take one: where they fill no more than half or a quarter
// of it, each is shared by two or four workgroups, 128 or 64 rows each.
//   256 x 256 in bf16: a step's operands (64 KB) arrive in about 1.0 us at a CU, its products take
// 1.06 us; together 1.5, and a tile's epilogue 9 us more. Hence the largest tile that the registers
// hold, which reads least. 16384 x 2048 by 8192 k 522 us (1.05 PFLOP/s; matrix cores busy 57 %);
// by 1024 k 63 - 73 (1.09 - 0.94); 65536 ragged rows, SwiGLU, 165 (0.83, 201 MB written).
//   fp32, 128 x 128: 350 vector instructions split a step's operands for 96 matrix ones, which
// bounds it: 9324 ragged rows of 1024 k x 1024 161 us (122 TFLOP/s; 0.153 PFLOP/s is what a large
// product on the fp32 matrix instructions reaches).
template <typename T, bool BKC, bool PAIR, typename SH>
__global__ void __launch_bounds__(SH::kThreads, SH::WPS) linear_rows_kernel(LinearArgs a) {
  constexpr int OBN = PAIR ? SH::BN / 2 : SH::BN;
  __shared__ uint4 lds[2 * 8 * (SH::BM + SH::BN)];
  const int tiles_c = ((PAIR ? a.N / 2 : a.N) + OBN - 1) / OBN;
  int tr, tc, group, r0, r1, parts = 1, part = 0;
  RowTiles<SH::BM> tiles(a);
  if constexpr (SH::kShared) {
    if (!place_shared(tiles.total, tiles_c, tr, tc, part, parts)) return;
  } else {
    if (!place_tile(tiles.total, tiles_c, tr, tc)) return;
  }
  if (!tiles.find(tr, group, r0, r1)) return;
  if constexpr (SH::kShared) {
    if (parts > 1) {
      r0 += part * (SH::BM / parts);
      if (r0 >= r1) return;
      if (parts == 2)
        rows_tile<T, BKC, PAIR, LinShape<SH::RT / 2, SH::CT, SH::WR, SH::WC, SH::WPS>>(a, lds, tc, group, r0, r1);
      else
        rows_tile<T, BKC, PAIR, LinShape<SH::RT / 4, SH::CT, SH::WR, SH::WC, SH::WPS>>(a, lds, tc, group, r0, r1);
      return;
    }
  }
  rows_tile<T, BKC, PAIR, SH>(a, lds, tc, group, r0, r1);
}

// Weight gradient: C_group[m][n] = sum over the group's rows r of A[r][m] B[r][n], rows through
// the optional indices. SIDE: the operand whose column sums (the bias gradient) are taken
// along, by one more product with ones in the tiles at 0 of the other dimension (0 none, 1 A,
// 2 B). ROWS: the operand whose rows an index names, likewise.
//   A dense one of 1024 x 2048 over 16384 rows takes 77 us in 256 x 256 tiles and 8 splits (0.89
// PFLOP/s, matrix cores busy 45 %; the splits' sums 11 us more); a ragged one of 65536 gathered
// rows in 16 uneven groups 191 us (0.72, 36 %): its end waits for the largest group's tiles.
template <typename T, int SIDE, int ROWS, typename SH>
__global__ void __launch_bounds__(SH::kThreads, SH::WPS) linear_wgrad_kernel(LinearArgs a) {
  constexpr int RT = SH::RT, CT = SH::CT, BM = SH::BM, BN = SH::BN;
  constexpr Map MAP = out_map<T, false>();
  constexpr int BWR = RT >= 4 ? 4 : 2, BWC = CT >= 4 ? 4 : 2;
  typedef Operand<T, BM, false, MAP, SH::kThreads, ROWS == 1> OA;
  typedef Operand<T, BN, false, MAP, SH::kThreads, ROWS == 2> OB;
  __shared__ uint4 lds[2 * (OA::kChunks + OB::kChunks)];
  uint4 *sA = lds, *sB = lds + 2 * OA::kChunks;
  static_assert(sizeof(lds) >= SH::WR * SH::WC * Slab::kFloats * 4, "the epilogue's rows fit");

  int group, split, mt, tc;
  if (!place_wgrad(a, group, split, mt, tc)) return;
  int r0, r1;
  group_span(a, group, r0, r1);
  r1 = max(r0, r1);
  if (a.splits > 1) {
    const int64_t per = ((r1 - r0 + a.splits - 1) / a.splits + OA::BK - 1) / OA::BK * OA::BK;
    r0 = (int)min(r0 + split * per, (int64_t)r1);
    r1 = (int)min(r0 + per, (int64_t)r1);
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
  lin_f32x4 acc[RT][CT], sum[1][SIDE == 1 ? RT : CT];
  clear(acc);
  clear(sum);
  const bool sums = SIDE == 1 ? tc == 0 && wc == 0 : SIDE == 2 ? mt == 0 && wr == 0 : false;
  bool again = true;
  if constexpr (sizeof(T) == 4) {
    const SplitReader<BM, false, BWR> ra(row_w);
    const SplitReader<BN, false, BWC> rb(col_w);
    auto read_b = [&](const uint4* lb, float(&x)[CT][8]) {
#pragma unroll
      for (int j = 0; j < CT; j += BWC) rb.read(lb, j, x + j);
    };
    lin_bf16x8 ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = 1.f;
    auto extra = [&](int i, const Split& fa, Split(&fb)[CT]) {
      if constexpr (SIDE == 1) {
        if (sums) sum[0][i] = mma(ones, fa.h, mma(ones, fa.m, mma(ones, fa.l, sum[0][i])));
      }
      if constexpr (SIDE == 2) {
        if (sums && i == 0)
#pragma unroll
          for (int j = 0; j < CT; ++j) sum[0][j] = mma(fb[j].h, ones, mma(fb[j].m, ones, mma(fb[j].l, ones, sum[0][j])));
      }
    };
    split_loop<SH>(oa, ob, r1 - r0, sA, sB, acc, ra, read_b, extra);
    again = any_not_finite(acc) || (SIDE != 0 && any_not_finite(sum));
    if (again) {
      clear(acc);
      clear(sum);
    }
  }
  if (again) {
    typedef typename Frag<T>::type F;
    F ones;
#pragma unroll
    for (int e = 0; e < OA::EV; ++e) ones[e] = 1.f;
    const Reader<T, BM, false, MAP, BWR, RT> ra(row_w);
    const Reader<T, BN, false, MAP, BWC, CT> rb(col_w);
    auto read_b = [&](const uint4* lb, int s, F(&fb)[CT]) { rb.read(lb, s, fb); };
    auto extra = [&](int i, const F& fa, F(&fb)[CT]) {
      if constexpr (SIDE == 1) {
        if (sums) sum[0][i] = mma(ones, fa, sum[0][i]);
      }
      if constexpr (SIDE == 2) {
        if (sums && i == 0)
#pragma unroll
          for (int j = 0; j < CT; ++j) sum[0][j] = mma(fb[j], ones, sum[0][j]);
      }
    };
    pipe_loop<T, SH>(oa, ob, r1 - r0, sA, sB, acc, ra, read_b, extra);
  }

  __syncthreads();  // the tiles' memory now holds the epilogue's rows
  const Slab slab{reinterpret_cast<float*>(lds) + wv * Slab::kFloats};
  wgrad_epilogue<T, MAP, BWR, BWC, SIDE>(a, acc, sum[0], slab, sums, group, split, m0 + row_w, n0 + col_w);
}

// The epilogue of a dense product in splits: sums of the partial ones, in order. 8 columns a thread.
template <typename T, bool PAIR>
__global__ void __launch_bounds__(256) linear_finish_kernel(LinearArgs a) {
  const int f = PAIR ? a.N / 2 : a.N, per = (f + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / per;
  if (r >= a.rows) return;
  const int col = (int)(i - r * per) * 8;
  float bias[2][8], v[8], u[8];
  load_bias<PAIR>(a, 0, false, col, f, bias);
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = u[q] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.part + ((int64_t)s * a.rows + r) * a.N + col;
    float x[8];
    load_run<8>(p, x, f - col);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += x[q];
    if constexpr (PAIR) {
      load_run<8>(p + f, x, f - col);
#pragma unroll
      for (int q = 0; q < 8; ++q) u[q] += x[q];
    }
  }
  finish_run<T, PAIR, false>(a, a.act, r, col, f, v, u, bias);
}

// Sums of a weight gradient's splits, in order; `count` elements of one split's partials, the
// first `n_c` of them C's (contiguous), the rest db's. 8 splits of 1024 x 2048: 11 us, 71 MB in all.
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

// dpre = act'(pre) dy over [rows][N]; SwiGLU: pre [rows][2 f], dy [rows][f]. 16 bytes a thread. Rows
// of dpre are ld elements apart, zeros past the N-th. Bound by memory: SwiGLU over 65536 rows of
// 2 x 512 bf16 moves 336 MB in 57 - 59 us (5.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) linear_act_grad_kernel(const T* pre, const T* dy, T* dpre,
                                                              int64_t rows, int f, int ld, int act) {
  constexpr int W = 16 / (int)sizeof(T);
  const int per = (f + W - 1) / W, N = act == PULSAR_ACT_SWIGLU ? 2 * f : f;
  const int64_t total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * W, n = f - c;
    float g[W], d[W], o[W];
    load_run<W>(dy + r * f + c, d, n);
    load_run<W>(pre + r * N + c, g, n);
    T* out = dpre + r * ld;
    if (act == PULSAR_ACT_SWIGLU) {
      float u[W], ou[W];
      load_run<W>(pre + r * N + f + c, u, n);
#pragma unroll
      for (int q = 0; q < W; ++q) {  // dy last: dy g may pass fp32's range where dy silu(g) does not
        ou[q] = d[q] * (g[q] * fast_sigmoid(g[q]));
        o[q] = d[q] * (u[q] * act_slope(PULSAR_ACT_SILU, g[q]));
      }
      store_run<W>(out + f + c, ou, n);
    } else {
#pragma unroll
      for (int q = 0; q < W; ++q) o[q] = d[q] * act_slope(act, g[q]);
    }
    store_run<W>(out + c, o, n);
    if (n <= W)
      for (int q = N; q < ld; ++q) out[q] = from_f<T>(0.f);
  }
}

// Copies of matrices into rows of whole aligned chunks, zeros past their columns: `halves` runs of
// `cols` columns each, at src_ld per row, to runs of `run` columns. One thread a chunk.
struct PackJob {
  const void* src;
  void* dst;
  int64_t rows, src_ld, src_group;  // rows of each group
  int64_t chunks;                   // in all
  int cols, halves, run;
  const int32_t* offsets;           // weights of groups without rows are left out (nullptr: none are)
};
struct PackJobs {
  PackJob job[3];
};
template <typename U>
__global__ void __launch_bounds__(256) linear_pack_kernel(PackJobs jobs) {
  constexpr int W = 16 / (int)sizeof(U);
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int k = 0;
  while (k < 3 && i >= jobs.job[k].chunks) i -= jobs.job[k++].chunks;
  if (k == 3) return;
  const PackJob& j = jobs.job[k];
  const int per = j.run / W;
  const int64_t run = i / per, row = run / j.halves, group = row / j.rows;
  if (j.offsets && j.offsets[group + 1] <= j.offsets[group]) return;
  const int c = (int)(i % per) * W, n = j.cols - c;
  const U* p = reinterpret_cast<const U*>(j.src) + group * j.src_group + row % j.rows * j.src_ld +
               run % j.halves * j.cols + c;
  U v[W];
  if (n >= W) {
    __builtin_memcpy(v, p, 16);
  } else {
#pragma unroll
    for (int q = 0; q < W; ++q) v[q] = q < n ? p[q] : 0;
  }
  uint4 o;
  __builtin_memcpy(&o, v, 16);
  reinterpret_cast<uint4*>(j.dst)[i] = o;
}

typedef LinShape<8, 4, 2, 4, 2> LinWide;   // 256 x 256
typedef LinShape<4, 4, 2, 2, 2> LinLarge;  // 128 x 128
typedef LinShape<2, 4, 2, 2, 2> LinSmall;  // 64 x 128

template <typename T, bool BKC, bool PAIR, typename SH>
int launch_rows_shape(LinearArgs& a, hipStream_t s) {
  const int f = PAIR ? a.N / 2 : a.N, obn = PAIR ? SH::BN / 2 : SH::BN;
  // every group adds at most one partial tile to the whole ones
  const int64_t tiles_r = a.offsets
      ? a.rows / SH::BM + std::min<int64_t>(a.groups + 1, a.rows)
      : (a.rows + SH::BM - 1) / SH::BM;
  const int64_t tiles = tiles_r * ((f + obn - 1) / obn);
  a.max_tiles = (int)tiles_r;
  if (tiles > (int64_t)1 << 30) return fail(PULSAR_ERR_INVALID, "linear: launch too large");
  int64_t slots = (tiles + kXcds - 1) / kXcds;
  if (SH::kShared) {
    // of a known number of tiles, those of the whole ranges and of the last one, which is shorter;
    // otherwise up to a round more
    if (a.offsets)
      slots += kXcdCus;
    else
      slots = std::max(shared_slots((int)slots), shared_slots((int)((tiles - 1) % slots + 1)));
  }
  linear_rows_kernel<T, BKC, PAIR, SH>
      <<<dim3((unsigned)(slots * kXcds), a.part ? a.splits : 1), SH::kThreads, 0, s>>>(a);
  PULSAR_LAUNCH_CHECK();
  return PULSAR_OK;
}

// Expected us of a product in tiles of BM x BN, by what bounds them here: each CU streams the
// operands of its tiles from the caches at `rate` bytes/us (35 KB/us for the few-row kernels,
// 45-49 for the tile kernels with two workgroups a CU, 38 for 256 x 256, whose tiles also pay
// `each` us of start and end that nothing overlaps) or multiplies at flop_rate (5 MFLOP/us in
// bf16; in fp32 0.25 - 0.33 in the few-row kernels, 0.5 - 0.6 in the tiles), whichever takes
// longer, after about 4 us of launch and first loads. Measured against
// it, us (model): 16 rows x 1024 x 1024 in 16 x 16 tiles 5.7 (5.8), in 16 x 32 6.3 (6.7); 512
// rows 32 x 64 9.7 (9.5), 32 x 32 12.0 (11.3), 64 x 64 12.4 (11.3); 4096 columns x 4096 k, 64
// rows in 32 x 32 19.7 (18.6), 32 x 64 26 (25.9); 2048 rows in 64 x 128 12.6 (12.5); 16384 x 2048
// x 1024 in 128 x 128 85 (87), in 256 x 256 77 (79). A ragged launch has about 0.6 partial tiles a
// group, at least one, and no whole rounds: a quarter of one is added beyond the first.
// `splits` workgroups share a tile's sum, and their partial ones meet in a second launch.
struct Sizes {
  double rows, groups, N, K;
  bool ragged, half, pair, b_kc;
};
double rows_cost(const Sizes& z, int BM, int BN, double rate, double flop_rate, double each, int splits) {
  double rt = std::ceil(z.rows / BM);
  if (z.ragged) rt = std::max(std::min(z.groups, z.rows), z.rows / BM + 0.6 * z.groups);
  const double n = rt * std::ceil(z.N / BN) / 256;
  double rounds = z.ragged ? (n <= 1 ? 1 : n + 0.25) : std::ceil(n * splits) / splits;
  if (each > 0) {  // shared tiles: a quarter of a round takes 0.45 of its time, a half 0.65
    const double rest = n - std::floor(n);
    rounds = std::floor(n) + (rest == 0 ? 0 : rest <= 0.25 ? 0.45 : rest <= 0.5 ? 0.65 : 1);
  }
  const double bytes = (BM + BN) * z.K * (z.half ? 2 : 4), flops = 2.0 * BM * BN * z.K;
  const double merge = splits > 1 ? 5 + z.rows * z.N * 8 * splits / 4e6 : 0;
  return 4 + rounds * (each + std::max(bytes / rate, flops / flop_rate)) + merge;
}

// How a product is cut: the shape that the model expects to be fastest, the few-row ones (0 - 5) or
// the tiles (64 x 128, 128 x 128, 256 x 256), and the workgroups that share a sum over k, which takes
// a second launch and their partial sums' way through memory (5 us and 4 MB/us). A split has to
// save a sixth of the expected time in bf16 and 4 % in fp32, about what the model is off by there.
// Unsplit and split, us: 256 rows x 4096 x 4096 in bf16 36 and 28, in fp32 100 and 65; 2331 x 1024 by
// 4096 k in fp32 184 and 134, 64 x 1024 18.8 and 16.8; not split in bf16: 1 x 1024 by 4096 k 8.5 and
// 11.4, 512 x 512 by 4096 13.8 and 18.2. Only dense products are split: ragged ones have the groups'
// times as many tiles.
struct RowsPlan {
  int shape, splits;
  int64_t part_bytes;
};
RowsPlan rows_plan(const Sizes& z) {
  RowsPlan best = {-1, 1, 0};
  double least = 0;
  auto offer = [&](int id, int splits, double us) {
    if (best.shape < 0 || us < least) best.shape = id, best.splits = splits, least = us;
  };
  const double gain = z.half ? 0.85 : 0.96;
  for (int s = 1; s == 1 || (!z.ragged && s <= 16 && z.K >= 256 * s); ++s) {
    if (s == 2 && (least *= gain) <= 9) break;  // the second launch alone leaves no gain
    for (int i = z.pair ? 1 : 0; i < 6; ++i)
      offer(i, s, rows_cost(z, 16 * kFewShapes[i].rt, 16 * kFewShapes[i].ct, 35e3,
                            z.half ? 5e6 : z.b_kc ? 0.33e6 : 0.25e6, 0, s));
    offer(6, s, rows_cost(z, 64, 128, 45e3, z.half ? 5e6 : 0.5e6, 0, s));
    offer(7, s, rows_cost(z, 128, 128, 49e3, z.half ? 5e6 : 0.6e6, 0, s));
    if (z.half && s == 1) offer(8, s, rows_cost(z, 256, 256, 38e3, 5e6, 10, s));
  }
  if (best.splits > 1) best.part_bytes = (int64_t)(best.splits * z.rows * z.N * 4);
  return best;
}

template <typename T>
int launch_rows(LinearArgs& a, const RowsPlan& plan, bool b_kc, hipStream_t s) {
  constexpr bool half = sizeof(T) == 2;
  const bool pair = a.act == PULSAR_ACT_SWIGLU;
  a.splits = plan.splits;
  auto go = [&](auto kc, auto pr) {
    constexpr bool KC = decltype(kc)::value, P = decltype(pr)::value;
    if constexpr (half) {
      if (plan.shape == 8) return launch_rows_shape<T, KC, P, LinWide>(a, s);
    }
    return plan.shape == 7 ? launch_rows_shape<T, KC, P, LinLarge>(a, s)
                           : launch_rows_shape<T, KC, P, LinSmall>(a, s);
  };
  int rc;
  if (plan.shape < 6)
    rc = launch_linear_few(a, half ? PULSAR_BF16 : PULSAR_F32, b_kc, plan.shape, s);
  else if (b_kc)
    rc = pair ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
  else
    rc = pair ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
  if (rc != PULSAR_OK || !a.part) return rc;
  const int64_t n = (int64_t)a.rows * (((pair ? a.N / 2 : a.N) + 7) / 8);
  if (pair)
    linear_finish_kernel<T, true><<<blocks_for(n, 256), 256, 0, s>>>(a);
  else
    linear_finish_kernel<T, false><<<blocks_for(n, 256), 256, 0, s>>>(a);
  PULSAR_LAUNCH_CHECK();
  return PULSAR_OK;
}

// How a weight gradient is cut: tile shape and splits of the sum over rows. Splits: enough
// workgroups to fill the chip twice where the tiles alone do not, none shorter than 512 rows of
// an average group.
struct WgradPlan {
  bool wide;
  int splits;
};
WgradPlan wgrad_plan(int64_t rows, int64_t groups, int64_t d_in, int64_t d_out, int dtype) {
  auto tiles = [&](int64_t t) { return ((d_in + t - 1) / t) * ((d_out + t - 1) / t) * groups; };
  auto splits = [&](int64_t n, int64_t fill) {
    return (int)std::max<int64_t>(1, std::min(fill / std::max<int64_t>(n, 1), rows / groups / 512));
  };
  const int wide = splits(tiles(256), 256);
  // 256 x 256 where they fill the chip with few splits (16384 x 2048 x 2048: 488 us in all against
  // 548, 16384 x 1024 x 1024, 16 splits: 97 against 90); ragged groups keep the smaller tiles,
  // whose sum is as long as the largest group's (65536 rows in 16 groups: 191 against 229)
  if (dtype == PULSAR_BF16 && groups == 1 && wide <= 8 && tiles(256) * wide >= 224) return {true, wide};
  return {false, tiles(128) >= 384 ? 1 : splits(tiles(128), 512)};
}

template <typename T, typename SH>
int launch_wgrad(LinearArgs& a, int side, hipStream_t s) {
  a.tiles_m = (a.M + SH::BM - 1) / SH::BM;
  a.tiles_n = (a.N + SH::BN - 1) / SH::BN;
  const int64_t per = (int64_t)a.tiles_m * a.tiles_n * a.splits, tiles = per * a.groups;
  if (tiles > (int64_t)1 << 30) return fail(PULSAR_ERR_INVALID, "linear: launch too large");
  const int64_t run = (int64_t)kXcds * wgrad_run((int)per);
  const unsigned grid = (unsigned)((tiles + run - 1) / run * run);
  auto go = [&](auto sd) {
    constexpr int S = decltype(sd)::value;
    if (a.a_rows)
      linear_wgrad_kernel<T, S, 1, SH><<<grid, SH::kThreads, 0, s>>>(a);
    else if (a.b_rows)
      linear_wgrad_kernel<T, S, 2, SH><<<grid, SH::kThreads, 0, s>>>(a);
    else
      linear_wgrad_kernel<T, S, 0, SH><<<grid, SH::kThreads, 0, s>>>(a);
  };
  if (side == 0)
    go(std::integral_constant<int, 0>{});
  else if (side == 1)
    go(std::integral_constant<int, 1>{});
  else
    go(std::integral_constant<int, 2>{});
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
  if (rows < 0 || d_in < 1 || d_out < 1 || groups < 1 || rows > 0x7fffff00 || d_in > 1 << 30 ||
      d_out > 1 << 30 || groups > 65536)
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

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// A stored matrix: groups of rows, a row contiguous.
struct Matrix {
  const void* p;
  int64_t ld, group, groups, rows, cols;
  int halves = 1;  // of the columns
  const int32_t* offsets = nullptr;  // weights of a ragged call: its groups
};

// Workspace handed out in 256-byte steps; with base == nullptr it only counts.
struct Space {
  char* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* r = base + used;
    used += round_up(bytes, 256);
    return r;
  }
};

// The kernels read operands in whole 16-byte chunks; a matrix whose rows do not lie that way (odd
// widths, slices of wider buffers) is copied first, into rows padded with zeros. The copy costs
// its bytes twice; reading such rows in place ran at a third of the aligned rate (517 rows x
// 1023 x 777: 25-31 us). Of a ragged call's weights only groups that have rows are copied (4 rows
// of 64 experts of 1023 x 1021: 64 -> 33 us).
struct Packing {
  PackJobs jobs = {};
  int n = 0;
  int es;
  Space& ws;
  Packing(int es_, Space& ws_) : es(es_), ws(ws_) {}
  Matrix operator()(Matrix m) {
    const int64_t ev = 16 / es, cols = m.cols / m.halves;
    if (aligned16(m.p) && m.ld % ev == 0 && (m.groups == 1 || m.group % ev == 0) && cols % ev == 0) return m;
    const int64_t run = round_up(cols, ev);
    PackJob& j = jobs.job[n++];
    j.src = m.p; j.rows = m.rows; j.src_ld = m.ld; j.src_group = m.group;
    j.cols = (int)cols; j.halves = m.halves; j.run = (int)run; j.offsets = m.offsets;
    m.ld = run * m.halves;
    m.group = m.rows * m.ld;
    j.chunks = m.groups * m.group / ev;
    m.p = j.dst = ws.take(m.groups * m.group * es);
    return m;
  }
  int launch(hipStream_t s) const {
    int64_t chunks = 0;
    for (int i = 0; i < n; ++i) chunks += jobs.job[i].chunks;
    if (chunks == 0) return PULSAR_OK;
    if (chunks > (int64_t)1 << 38) return fail(PULSAR_ERR_INVALID, "linear: operands too large");
    if (es == 2)
      linear_pack_kernel<uint16_t><<<blocks_for(chunks, 256), 256, 0, s>>>(jobs);
    else
      linear_pack_kernel<uint32_t><<<blocks_for(chunks, 256), 256, 0, s>>>(jobs);
    PULSAR_LAUNCH_CHECK();
    return PULSAR_OK;
  }
};

// One call's operands, as the C entries take them.
struct Call {
  const void* x;
  int64_t x_rs, x_rows;
  const int32_t* index;
  const int32_t* offsets;
  bool ragged;
  Weight w;
  int64_t rows, groups, d_in, d_out;
  int act, dtype;
  const char* what;

  Sizes sizes(int64_t N, int64_t K, bool pair, bool b_kc) const {
    return {(double)rows, (double)groups, (double)N, (double)K, ragged, dtype == PULSAR_BF16,
            pair, b_kc};
  }
  int es() const { return dtype == PULSAR_BF16 ? 2 : 4; }
  Matrix x_matrix() const { return {x, x_rs, 0, 1, x_rows, d_in}; }
  Matrix w_matrix(bool pair) const {
    if (in_contiguous(w)) return {w.p, w.out, w.group, groups, d_out, d_in, 1, offsets};
    return {w.p, w.in, w.group, groups, d_in, d_out, pair ? 2 : 1, offsets};
  }
  int check() const {
    const int rc = check_common(rows, groups, d_in, d_out, w, act, dtype, what);
    if (rc != PULSAR_OK) return rc;
    // the kernels multiply row indexes and strides in 32 bits
    if (x_rs > 0x7fffffff || w.in > 0x7fffffff || w.out > 0x7fffffff)
      return fail(PULSAR_ERR_INVALID, std::string(what) + ": row strides must be below 2^31 elements");
    if (x_rows < 0 || (rows > 0 && x_rs < d_in && x_rows > 1))
      return fail(PULSAR_ERR_INVALID, std::string(what) + ": rows of x overlap");
    return PULSAR_OK;
  }
  // The workspace's size does not depend on the index, so only the calls look at it.
  int check_rows() const {
    return index || x_rows == rows ? PULSAR_OK
                                   : fail(PULSAR_ERR_INVALID, std::string(what) + ": without an index x must have `rows` rows");
  }
  int null_pointer() const { return fail(PULSAR_ERR_INVALID, std::string(what) + ": null pointer"); }
  int no_workspace() const {
    return fail(PULSAR_ERR_INVALID, std::string(what) + ": workspace missing or not 16-byte aligned");
  }
};

// The operands of a forward call as its kernel takes them, and the workspace they need.
struct ForwardPlan {
  Space ws;
  Packing pack;
  Matrix x, w;
  RowsPlan rows;
  float* part;
  ForwardPlan(const Call& c, void* workspace)
      : ws{static_cast<char*>(workspace)}, pack(c.es(), ws), x(pack(c.x_matrix())),
        w(pack(c.w_matrix(c.act == PULSAR_ACT_SWIGLU))),
        rows(rows_plan(c.sizes(c.d_out, c.d_in, c.act == PULSAR_ACT_SWIGLU, in_contiguous(c.w)))),
        part(rows.part_bytes ? static_cast<float*>(ws.take(rows.part_bytes)) : nullptr) {}
};

int forward(const Call& c, const void* bias, int bias_dtype, const void* residual, int64_t res_rs,
            void* y, void* pre, void* workspace, hipStream_t s) {
  int rc = c.check();
  if (rc == PULSAR_OK) rc = c.check_rows();
  if (rc != PULSAR_OK) return rc;
  if (bias && bias_dtype != PULSAR_F32 && bias_dtype != PULSAR_BF16)
    return fail(PULSAR_ERR_INVALID, std::string(c.what) + ": bias dtype must be PULSAR_F32 or PULSAR_BF16");
  if (c.rows == 0) return PULSAR_OK;
  if (!y || (!c.x && c.x_rows > 0) || !c.w.p) return c.null_pointer();
  ForwardPlan plan(c, workspace);
  if (plan.ws.used > 0 && (!workspace || !aligned16(workspace))) return c.no_workspace();
  const int rp = plan.pack.launch(s);
  if (rp != PULSAR_OK) return rp;
  const bool kc = in_contiguous(c.w), pair = c.act == PULSAR_ACT_SWIGLU;
  const int64_t f = pair ? c.d_out / 2 : c.d_out;
  LinearArgs a = {};
  a.A = plan.x.p; a.lda = plan.x.ld; a.a_rows = c.index; a.a_nrows = c.x_rows;
  a.B = plan.w.p; a.ldb = plan.w.ld; a.b_group = plan.w.group;
  a.up = (int)(kc || plan.w.p == c.w.p ? f : plan.w.ld / 2);
  a.offsets = c.offsets; a.groups = (int)c.groups; a.rows = (int)c.rows;
  a.N = (int)c.d_out; a.K = (int)c.d_in;
  a.C = y; a.ldc = f;
  a.pre = pre; a.ldpre = c.d_out;
  a.bias = bias; a.bias_dtype = bias_dtype;
  a.residual = residual; a.ldr = res_rs;
  a.act = c.act;
  a.part = plan.part;
  return c.dtype == PULSAR_BF16 ? launch_rows<bf16>(a, plan.rows, kc, s) : launch_rows<float>(a, plan.rows, kc, s);
}

struct BackwardPlan {
  Space ws;
  Packing pack;
  Matrix x, w, dpre;
  RowsPlan rows;
  WgradPlan wgrad;
  float *part = nullptr, *part_db = nullptr;  // of the weight gradient; dx's lie there first
  BackwardPlan(const Call& c, const void* dy, void* workspace)
      : ws{static_cast<char*>(workspace)}, pack(c.es(), ws), x(pack(c.x_matrix())),
        w(pack(c.w_matrix(false))), dpre{dy, c.d_out, 0, 1, c.rows, c.d_out},
        rows(rows_plan(c.sizes(c.d_in, c.d_out, false, !in_contiguous(c.w)))),
        wgrad(wgrad_plan(c.rows, c.groups, c.d_in, c.d_out, c.dtype)) {
    if (c.act == PULSAR_ACT_NONE) {
      dpre = pack(dpre);
    } else {
      dpre.ld = round_up(c.d_out, 16 / c.es());
      dpre.p = ws.take(c.rows * dpre.ld * c.es());
    }
    const int64_t n = wgrad.splits > 1 ? wgrad.splits * c.groups * c.d_in * c.d_out * 4 : 0;
    if (n || rows.part_bytes) part = static_cast<float*>(ws.take(std::max(n, rows.part_bytes)));
    if (n) part_db = static_cast<float*>(ws.take(wgrad.splits * c.groups * c.d_out * 4));
  }
};

template <typename T>
int backward_t(const Call& c, const BackwardPlan& plan, const void* dy, const void* pre, void* dx,
               void* dw, void* db, hipStream_t s) {
  const bool kc = in_contiguous(c.w);
  if (c.rows > 0) {
    const int rp = plan.pack.launch(s);
    if (rp != PULSAR_OK) return rp;
    if (c.act != PULSAR_ACT_NONE) {
      constexpr int ev = 16 / (int)sizeof(T);
      const int f = (int)(c.act == PULSAR_ACT_SWIGLU ? c.d_out / 2 : c.d_out);
      const int64_t n = c.rows * ((f + ev - 1) / ev);
      linear_act_grad_kernel<T><<<(unsigned)std::min<int64_t>((n + 255) / 256, 8192), 256, 0, s>>>(
          static_cast<const T*>(pre), static_cast<const T*>(dy),
          static_cast<T*>(const_cast<void*>(plan.dpre.p)), c.rows, f, (int)plan.dpre.ld, c.act);
      PULSAR_LAUNCH_CHECK();
    }
    // dx = dpre w^T: n is the input dimension, k the output one
    LinearArgs a = {};
    a.A = plan.dpre.p; a.lda = plan.dpre.ld; a.a_nrows = c.rows;
    a.B = plan.w.p; a.ldb = plan.w.ld; a.b_group = plan.w.group;
    a.offsets = c.offsets; a.groups = (int)c.groups; a.rows = (int)c.rows;
    a.N = (int)c.d_in; a.K = (int)c.d_out;
    a.C = dx; a.ldc = c.d_in;
    if (plan.rows.splits > 1) a.part = plan.part;
    const int rc = launch_rows<T>(a, plan.rows, !kc, s);
    if (rc != PULSAR_OK) return rc;
  }
  // dw in the weight's own order: its contiguous dimension is n
  LinearArgs a = {};
  if (kc) {
    a.A = plan.dpre.p; a.lda = plan.dpre.ld; a.a_nrows = c.rows; a.M = (int)c.d_out;
    a.B = plan.x.p; a.ldb = plan.x.ld; a.b_rows = c.index; a.b_nrows = c.x_rows; a.N = (int)c.d_in;
  } else {
    a.A = plan.x.p; a.lda = plan.x.ld; a.a_rows = c.index; a.a_nrows = c.x_rows; a.M = (int)c.d_in;
    a.B = plan.dpre.p; a.ldb = plan.dpre.ld; a.b_nrows = c.rows; a.N = (int)c.d_out;
  }
  a.offsets = c.offsets; a.groups = (int)c.groups; a.rows = (int)c.rows;
  a.C = dw; a.ldc = a.N; a.c_group = (int64_t)a.M * a.N;
  a.db = db;
  a.splits = plan.wgrad.splits;
  a.part = plan.part;
  a.part_db = plan.part_db;
  const int side = db ? (kc ? 1 : 2) : 0;
  if constexpr (sizeof(T) == 2) {
    if (plan.wgrad.wide) return launch_wgrad<T, LinWide>(a, side, s);
  }
  return launch_wgrad<T, LinLarge>(a, side, s);
}

int backward(const Call& c, const void* dy, const void* pre, void* dx, void* dw, void* db,
             void* workspace, hipStream_t s) {
  int rc = c.check();
  if (rc == PULSAR_OK) rc = c.check_rows();
  if (rc != PULSAR_OK) return rc;
  if (!dw || (c.rows > 0 && (!dy || (!c.x && c.x_rows > 0) || !c.w.p || !dx ||
                             (c.act != PULSAR_ACT_NONE && !pre))))
    return c.null_pointer();
  BackwardPlan plan(c, dy, workspace);
  if (plan.ws.used > 0 && (!workspace || !aligned16(workspace))) return c.no_workspace();
  return c.dtype == PULSAR_BF16 ? backward_t<bf16>(c, plan, dy, pre, dx, dw, db, s)
                                : backward_t<float>(c, plan, dy, pre, dx, dw, db, s);
}

int64_t forward_bytes(const Call& c) {
  return c.check() != PULSAR_OK ? -1 : c.rows == 0 ? 0 : ForwardPlan(c, nullptr).ws.used;
}
int64_t backward_bytes(const Call& c, const void* dy) {
  return c.check() != PULSAR_OK ? -1 : BackwardPlan(c, dy, nullptr).ws.used;
}

}  // namespace

}  // namespace pulsar

using namespace pulsar;

extern "C" {

int64_t pulsar_fused_linear_forward_workspace_bytes(const void* x, int64_t x_rs, const void* w,
                                                    int64_t w_out, int64_t w_in, int64_t rows,
                                                    int64_t d_in, int64_t d_out, int activation,
                                                    int dtype) {
  return forward_bytes(Call{x, x_rs, rows, nullptr, nullptr, false, Weight{w, 0, w_in, w_out}, rows, 1, d_in,
                            d_out, activation, dtype, "fused_linear_forward"});
}

int pulsar_fused_linear_forward(const void* x, int64_t x_rs, const void* w, int64_t w_out,
                                int64_t w_in, const void* bias, int bias_dtype,
                                const void* residual, int64_t residual_rs, void* y, void* pre,
                                int64_t rows, int64_t d_in, int64_t d_out, int activation,
                                int dtype, void* workspace, hipStream_t stream) {
  return forward(Call{x, x_rs, rows, nullptr, nullptr, false, Weight{w, 0, w_in, w_out}, rows, 1, d_in, d_out,
                      activation, dtype, "fused_linear_forward"},
                 bias, bias_dtype, residual, residual_rs, y, pre, workspace, stream);
}

int64_t pulsar_fused_linear_backward_workspace_bytes(const void* dy, const void* x, int64_t x_rs,
                                                     const void* w, int64_t w_out, int64_t w_in,
                                                     int64_t rows, int64_t d_in, int64_t d_out,
                                                     int activation, int dtype) {
  return backward_bytes(Call{x, x_rs, rows, nullptr, nullptr, false, Weight{w, 0, w_in, w_out}, rows, 1, d_in,
                             d_out, activation, dtype, "fused_linear_backward"}, dy);
}

int pulsar_fused_linear_backward(const void* dy, const void* x, int64_t x_rs, const void* w,
                                 int64_t w_out, int64_t w_in, const void* pre, void* dx, void* dw,
                                 void* db, int64_t rows, int64_t d_in, int64_t d_out,
                                 int activation, int dtype, void* workspace, hipStream_t stream) {
  return backward(Call{x, x_rs, rows, nullptr, nullptr, false, Weight{w, 0, w_in, w_out}, rows, 1, d_in,
                       d_out, activation, dtype, "fused_linear_backward"},
                  dy, pre, dx, dw, db, workspace, stream);
}

int64_t pulsar_grouped_linear_forward_workspace_bytes(const void* x, int64_t x_rs, int64_t x_rows,
                                                      const void* w, int64_t w_group, int64_t w_in,
                                                      int64_t w_out, int64_t rows, int64_t groups,
                                                      int64_t d_in, int64_t d_out, int activation,
                                                      int dtype) {
  return forward_bytes(Call{x, x_rs, x_rows, nullptr, nullptr, true, Weight{w, w_group, w_in, w_out}, rows,
                            groups, d_in, d_out, activation, dtype, "grouped_linear_forward"});
}

int pulsar_grouped_linear_forward(const void* x, int64_t x_rs, int64_t x_rows,
                                  const int32_t* row_index, const int32_t* offsets, const void* w,
                                  int64_t w_group, int64_t w_in, int64_t w_out, const void* bias,
                                  int bias_dtype, void* y, void* pre, int64_t rows,
                                  int64_t groups, int64_t d_in, int64_t d_out, int activation,
                                  int dtype, void* workspace, hipStream_t stream) {
  PULSAR_REQUIRE(offsets, "grouped_linear_forward: null pointer");
  return forward(Call{x, x_rs, x_rows, row_index, offsets, true, Weight{w, w_group, w_in, w_out}, rows,
                      groups, d_in, d_out, activation, dtype, "grouped_linear_forward"},
                 bias, bias_dtype, nullptr, 0, y, pre, workspace, stream);
}

int64_t pulsar_grouped_linear_backward_workspace_bytes(const void* dy, const void* x, int64_t x_rs,
                                                       int64_t x_rows, const void* w,
                                                       int64_t w_group, int64_t w_in, int64_t w_out,
                                                       int64_t rows, int64_t groups, int64_t d_in,
                                                       int64_t d_out, int activation, int dtype) {
  return backward_bytes(Call{x, x_rs, x_rows, nullptr, nullptr, true, Weight{w, w_group, w_in, w_out}, rows,
                             groups, d_in, d_out, activation, dtype, "grouped_linear_backward"}, dy);
}

int pulsar_grouped_linear_backward(const void* dy, const void* x, int64_t x_rs, int64_t x_rows,
                                   const int32_t* row_index, const int32_t* offsets, const void* w,
                                   int64_t w_group, int64_t w_in, int64_t w_out, const void* pre,
                                   void* dx, void* dw, void* db, int64_t rows, int64_t groups,
                                   int64_t d_in, int64_t d_out, int activation, int dtype,
                                   void* workspace, hipStream_t stream) {
  PULSAR_REQUIRE(offsets, "grouped_linear_backward: null pointer");
  return backward(Call{x, x_rs, x_rows, row_index, offsets, true, Weight{w, w_group, w_in, w_out}, rows,
                       groups, d_in, d_out, activation, dtype, "grouped_linear_backward"},
                  dy, pre, dx, dw, db, workspace, stream);
}

}  // extern "C"
