// Dense and ragged (grouped by expert) products with bias, activation and residual in the
// epilogue, and their gradients: fused_linear_* and grouped_linear_* of the op surface.
#include <algorithm>
#include <type_traits>

#include "linear_device.h"

namespace pulsar {

namespace {

// Products over ragged rows: C[i][n] = epi(sum_k A[row(i)][k] B_group[n][k]). PAIR (SwiGLU): a
// tile's columns are BN / 2 gate columns and their up-projection twins N / 2 further on.
template <typename T, bool BKC, bool PAIR, bool VEC, typename SH>
__global__ void __launch_bounds__(SH::kThreads, SH::WPS) linear_rows_kernel(LinearArgs a) {
  constexpr int RT = SH::RT, CT = SH::CT, BM = SH::BM, BN = SH::BN;
  constexpr Map MAP = out_map<T, BKC>();
  constexpr int NCT = PAIR ? CT / 2 : CT;  // tiles of output columns per wave
  constexpr int BW = NCT >= 4 ? 4 : 2;
  static_assert(MAP == PLAIN || NCT % (MAP == WIDE ? 2 : BW) == 0, "whole runs per wave");
  typedef Operand<T, BM, true, PLAIN, SH::kThreads> OA;
  typedef Operand<T, BN, BKC, MAP, SH::kThreads> OB;
  __shared__ uint4 lds[2 * (OA::kChunks + OB::kChunks)];
  uint4 *sA = lds, *sB = lds + 2 * OA::kChunks;
  static_assert(sizeof(lds) >= SH::WR * SH::WC * Slab<CT>::kFloats * 4, "the epilogue's slabs fit");

  const int f = PAIR ? a.N / 2 : a.N;          // output columns
  constexpr int OBN = PAIR ? BN / 2 : BN;      // output columns of a tile
  const int tiles_c = (f + OBN - 1) / OBN;
  int group = 0, r0 = 0, r1 = 0, tr, tc;
  if (!place_tile(count_tiles<BM>(a), tiles_c, tr, tc)) return;
  if (!find_tile<BM>(a, tr, group, r0, r1)) return;
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

  typedef typename Frag<T>::type F;
  const Reader<T, BM, true, PLAIN, 1> ra(row_w);
  const Reader<T, BN, BKC, MAP, BW> rb(col_w), ru(OBN + col_w);
  auto rd = [&](const uint4* la, const uint4* lb, int s, F(&fa)[RT], F(&fb)[CT], int part) {
    if (part == 0) {
      rb.template read<NCT>(lb, s, fb);
      if constexpr (PAIR) ru.template read<NCT>(lb, s, fb + NCT);
    } else {
      ra.template read<RT>(la, s, fa);
    }
  };
  if constexpr (VEC) {
    pipe_loop<T, SH>(oa, ob, K, sA, sB, acc, rd, [](int, F(&)[RT], F(&)[CT]) {});
  } else {
    staged_loop<T>(oa, ob, K, sA, sB, [&](const uint4* la, const uint4* lb) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        F fa[RT], fb[CT];
        rd(la, lb, s, fa, fb, 0);
        rd(la, lb, s, fa, fb, 1);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < CT; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
      }
    });
  }

  __syncthreads();  // the tiles' memory now holds the epilogue's rows
  rows_epilogue<T, MAP, BW, PAIR>(a, acc, reinterpret_cast<float*>(lds) + wv * Slab<CT>::kFloats, group, none,
                                  r0 + row_w, r1, n0 + col_w, f);
}

// Weight gradient: C_group[m][n] = sum over the group's rows r of A[r][m] B[r][n], rows through
// the optional indices. SIDE: the operand whose column sums (the bias gradient) are taken
// along, by one more product with ones in the tiles at 0 of the other dimension (0 none, 1 A,
// 2 B).
template <typename T, bool VEC, int SIDE, typename SH>
__global__ void __launch_bounds__(SH::kThreads, SH::WPS) linear_wgrad_kernel(LinearArgs a) {
  constexpr int RT = SH::RT, CT = SH::CT, BM = SH::BM, BN = SH::BN;
  constexpr Map MAP = out_map<T, false>();
  constexpr int BWR = RT >= 4 ? 4 : 2, BWC = CT >= 4 ? 4 : 2;
  typedef Operand<T, BM, false, MAP, SH::kThreads> OA;
  typedef Operand<T, BN, false, MAP, SH::kThreads> OB;
  __shared__ uint4 lds[2 * (OA::kChunks + OB::kChunks)];
  uint4 *sA = lds, *sB = lds + 2 * OA::kChunks;
  static_assert(sizeof(lds) >= SH::WR * SH::WC * Slab<CT>::kFloats * 4, "the epilogue's slabs fit");

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

  typedef typename Frag<T>::type F;
  const Reader<T, BM, false, MAP, BWR> ra(row_w);
  const Reader<T, BN, false, MAP, BWC> rb(col_w);
  auto rd = [&](const uint4* la, const uint4* lb, int s, F(&fa)[RT], F(&fb)[CT], int part) {
    if (part == 0)
      rb.template read<CT>(lb, s, fb);
    else
      ra.template read<RT>(la, s, fa);
  };
  auto extra = [&](int i, F(&fa)[RT], F(&fb)[CT]) {
    if constexpr (SIDE == 1) {
      if (sums) sum[i] = mma(ones, fa[i], sum[i]);
    }
    if constexpr (SIDE == 2) {
      if (sums && i == 0)
#pragma unroll
        for (int j = 0; j < CT; ++j) sum[j] = mma(fb[j], ones, sum[j]);
    }
  };
  if constexpr (VEC) {
    pipe_loop<T, SH>(oa, ob, r1 - r0, sA, sB, acc, rd, extra);
  } else {
    staged_loop<T>(oa, ob, r1 - r0, sA, sB, [&](const uint4* la, const uint4* lb) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        F fa[RT], fb[CT];
        rd(la, lb, s, fa, fb, 0);
        rd(la, lb, s, fa, fb, 1);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
#pragma unroll
          for (int j = 0; j < CT; ++j) acc[i][j] = mma(fb[j], fa[i], acc[i][j]);
          extra(i, fa, fb);
        }
      }
    });
  }

  __syncthreads();  // the tiles' memory now holds the epilogue's rows
  wgrad_epilogue<T, MAP, BWR, BWC, SIDE>(a, acc, sum, reinterpret_cast<float*>(lds) + wv * Slab<CT>::kFloats,
                                         sums, group, split, m0 + row_w, n0 + col_w);
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
        ou[q] = d[q] * g[q] * fast_sigmoid(g[q]);
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

typedef LinShape<8, 4, 2, 4, 2> LinWide;   // 256 x 256
typedef LinShape<4, 4, 2, 2, 2> LinLarge;  // 128 x 128
typedef LinShape<2, 4, 2, 2, 2> LinSmall;  // 64 x 128

template <typename T, bool BKC, bool PAIR, bool VEC, typename SH>
int launch_rows_shape(LinearArgs& a, hipStream_t s) {
  const int f = PAIR ? a.N / 2 : a.N, obn = PAIR ? SH::BN / 2 : SH::BN;
  // every group adds at most one partial tile to the whole ones
  const int64_t tiles_r = a.offsets
      ? a.rows / SH::BM + std::min<int64_t>(a.groups + 1, a.rows)
      : (a.rows + SH::BM - 1) / SH::BM;
  const int64_t tiles = tiles_r * ((f + obn - 1) / obn);
  a.max_tiles = (int)tiles_r;
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
  // the launch's tiles, a ragged group adding half of one on average
  auto tiles = [&](int r, int c) {
    return ((a.rows + r - 1) / r + (a.offsets ? a.groups / 2 : 0)) * (((int64_t)a.N + c - 1) / c);
  };
  const int64_t t128 = tiles(128, 128), t256 = tiles(256, 256);
  const double steps = (a.K + 4 * ev * 2 - 1) / (4 * ev * 2);
  const bool large = t128 >= 256;
  const bool wide = ((t256 + 255) / 256) * (10 + 1.7 * steps) < ((t128 + 511) / 512) * (5.7 + 0.98 * steps);
  auto go = [&](auto kc, auto pr, auto vc) {
    constexpr bool KC = decltype(kc)::value, P = decltype(pr)::value, V = decltype(vc)::value;
    if constexpr (V && sizeof(T) == 2) {
      if (wide) return launch_rows_shape<T, KC, P, V, LinWide>(a, s);
    }
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
#ifndef WGRAD_WIDE
#define WGRAD_WIDE (groups == 1 && tiles(256) * wide >= 224)
#endif
  if (dtype == PULSAR_BF16 && WGRAD_WIDE) return {true, wide};
  return {false, tiles(128) >= 384 ? 1 : splits(tiles(128), 512)};
}

template <typename T, bool VEC, typename SH>
int launch_wgrad(LinearArgs& a, int side, hipStream_t s) {
  a.tiles_m = (a.M + SH::BM - 1) / SH::BM;
  a.tiles_n = (a.N + SH::BN - 1) / SH::BN;
  const int64_t per = (int64_t)a.tiles_m * a.tiles_n * a.splits, tiles = per * a.groups;
  if (tiles > (int64_t)1 << 30) return fail(PULSAR_ERR_INVALID, "linear: launch too large");
  const int64_t run = kXcds * std::max<int64_t>(1, per / kXcds);  // place_wgrad's
  const unsigned grid = (unsigned)((tiles + run - 1) / run * run);
  if (side == 0)
    linear_wgrad_kernel<T, VEC, 0, SH><<<grid, SH::kThreads, 0, s>>>(a);
  else if (side == 1)
    linear_wgrad_kernel<T, VEC, 1, SH><<<grid, SH::kThreads, 0, s>>>(a);
  else
    linear_wgrad_kernel<T, VEC, 2, SH><<<grid, SH::kThreads, 0, s>>>(a);
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
  const int splits = wgrad_plan(rows, groups, d_in, d_out, dtype).splits;
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
  const WgradPlan plan = wgrad_plan(rows, groups, d_in, d_out, sizeof(T) == 2 ? PULSAR_BF16 : PULSAR_F32);
  a.splits = plan.splits;
  if (a.splits > 1) {
    a.part = reinterpret_cast<float*>(ws);
    a.part_db = a.part + (int64_t)a.splits * groups * d_in * d_out;
  }
  const bool vec = aligned16(a.A) && aligned16(a.B) && a.lda % ev == 0 && a.ldb % ev == 0 &&
                   a.M % ev == 0 && a.N % ev == 0;
  const int side = db ? (dpre_a ? 1 : 2) : 0;
  if constexpr (sizeof(T) == 2) {
    if (plan.wide && vec) return launch_wgrad<T, true, LinWide>(a, side, s);
  }
  return vec ? launch_wgrad<T, true, LinLarge>(a, side, s) : launch_wgrad<T, false, LinLarge>(a, side, s);
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
