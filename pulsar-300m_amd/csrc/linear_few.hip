// Products with few rows in a group (decoding): the weights are read once and bound the time.
#include <algorithm>

#include "linear_device.h"

namespace pulsar {

namespace {

// A chunk of 16 bytes, or zeros.
__device__ __forceinline__ uint4 load_chunk(const void* p, bool in) {
  uint4 r = {0u, 0u, 0u, 0u};
  if (in) r = *reinterpret_cast<const uint4*>(p);
  return r;
}

// Floats from one row of a workgroup's sums in LDS to the next: 4 apart from a multiple of the banks.
template <int CT>
constexpr int kSumStride = 16 * CT + 4;

// Writes one row tile of accumulators: LDS row i16, columns in order.
template <Map MAP, int BW, int NCT, int CT>
__device__ __forceinline__ void slab_write_tile(float* slab, const lin_f32x4 (&acc)[CT]) {
  const int lane = (int)threadIdx.x & 63, i16 = lane & 15, kq = lane >> 4;
#pragma unroll
  for (int j = 0; j < CT; ++j) {
    // tiles beyond NCT are the second set of a pair, 16 NCT columns on
    const int u = j % NCT;
    float* p = slab + i16 * kSumStride<CT> + j / NCT * 16 * NCT;
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

// A workgroup owns 16 RT rows of a group and 16 NCT output columns; its W waves take a run of k
// each, with D steps of operands in flight in registers, and add their sums through LDS at the
// end. Weights that are contiguous along k go from memory straight into matrix-core order; bf16
// weights contiguous along the output columns pass through the wave's own corner of LDS and its
// transposing read; fp32 ones are loaded a column run per lane, tiles sharing a run.
//   Bound by the latency of a few dependent loads (offsets, row index, operands), and from some
// hundred rows by what a CU streams: 16 rows x 1024 x 1024 in bf16 5.9 us with 64 workgroups (2.2
// MB), 4 experts of one row 6.6 us (8.4 MB, 1.3 TB/s), 517 x 777 by 1023 k 12 us.
template <typename T, bool BKC, bool PAIR, int RT, int CT, int W, int D>
__global__ void __launch_bounds__(64 * W) linear_few_kernel(LinearArgs a) {
  typedef typename Frag<T>::type F;
  constexpr int NCT = PAIR ? CT / 2 : CT, BM = 16 * RT, OBN = 16 * NCT;
  constexpr int EV = 16 / (int)sizeof(T), KS = 4 * EV;  // k's of a step: 32 bf16, 16 fp32
  constexpr bool TR = !BKC && sizeof(T) == 2;
  constexpr Map MAP = !BKC && sizeof(T) == 4 ? BLOCK : PLAIN;
  constexpr int BW = NCT;
  constexpr int SS = kSumStride<CT>;
  constexpr int kStage = TR ? CT * 64 : 1;  // chunks of a step's weights, per wave
  constexpr int kBytes = 16 * W * kStage, kSums = W * BM * SS * 4;
  __shared__ __attribute__((aligned(16))) char lds[kBytes > kSums ? kBytes : kSums];

  const int f = PAIR ? a.N / 2 : a.N, tiles_c = (f + OBN - 1) / OBN;
  int tr, tc, group, r0, r1;
  RowTiles<BM> tiles(a);
  if (!place_tile(tiles.total, tiles_c, tr, tc) || !tiles.find(tr, group, r0, r1)) return;
  const bool none = group >= a.groups;
  const int n0 = tc * OBN;
  const int lane = (int)threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int i16 = lane & 15, kq = lane >> 4;

  // this workgroup's k's, and this wave's steps of them
  int kfirst = 0, kend = a.K;
  if (a.part) split_range<T>(a.K, a.splits, (int)blockIdx.y, kfirst, kend);
  const int all = none ? 0 : (kend + KS - 1) / KS, per = (all + W - 1) / W;
  const int s0 = min(wv * per, all), s1 = min(s0 + per, all);

  const T* Bp = reinterpret_cast<const T*>(a.B) + (none ? 0 : group) * a.b_group + kfirst * (BKC ? 1 : a.ldb);
  // column of tile t: gate tiles, then their twins
  auto tile_col = [&](int t) { return PAIR && t >= NCT ? a.up + n0 + (t - NCT) * 16 : n0 + t * 16; };
  auto tile_lim = [&](int t) { return PAIR && t >= NCT ? a.up + f : f; };
  auto kx = [](int k) { return CT == 1 ? 0 : CT == 2 ? k >> 3 & 1 : (k >> 1 & 1) | (k >> 3 & 1) << 1; };
  auto kr = [](int k) { return CT == 1 ? k ^ (k >> 3 & 1) << 2 : k; };
  constexpr int NB = BKC ? CT : TR ? CT : MAP == BLOCK ? CT : 1;
  const T* bp[NB];
  bool bn[NB];  // inside the matrix (!BKC)
  if constexpr (BKC) {
#pragma unroll
    for (int t = 0; t < CT; ++t)
      bp[t] = Bp + (int64_t)min(tile_col(t) + i16, tile_lim(t) - 1) * a.ldb + kq * EV;
  } else if constexpr (TR) {
    // chunk c of a step: LDS [32 k][CT tiles][2 chunks]; load h covers 32 / CT k rows. A
    // transposing read takes 32 bytes of k rows k .. k + 3 and k + 8 .. k + 11 at once: row k
    // sits at kr(k) and its tile t at t ^ kx(k), which puts them on different banks of the 64
#pragma unroll
    for (int h = 0; h < CT; ++h) {
      const int c = lane + 64 * h, k = kr(c / (2 * CT)), t = c / 2 % CT ^ kx(k);
      const int col = tile_col(t) + 8 * (c & 1);
      bn[h] = col < tile_lim(t);
      bp[h] = Bp + (int64_t)k * a.ldb + (bn[h] ? col : 0);
    }
  } else {
    // run b of BW tiles: columns BW i16 .. of the run
#pragma unroll
    for (int b = 0; b < CT / BW; ++b) {
      const int col = tile_col(b * BW) + BW * i16;
      bn[b] = col < tile_lim(b * BW);
      bp[b] = Bp + (int64_t)(4 * kq) * a.ldb + (bn[b] ? col : 0);
    }
  }
  uint4 wbuf[D][CT], xbuf[D][RT];
  auto load_w = [&](int s, uint4 (&w)[CT]) {
    const int k0 = s * KS;
    if constexpr (BKC) {
      const bool in = s < s1 && k0 + kq * EV < kend;
#pragma unroll
      for (int t = 0; t < CT; ++t) w[t] = load_chunk(bp[t] + k0, in);
    } else if constexpr (TR) {
#pragma unroll
      for (int h = 0; h < CT; ++h) {
        const int k = k0 + kr((lane + 64 * h) / (2 * CT));
        w[h] = load_chunk(bp[h] + (int64_t)k0 * a.ldb, s < s1 && k < kend && bn[h]);
      }
    } else {
      float* o = reinterpret_cast<float*>(w);  // tile t, element j at 4 t + j
#pragma unroll
      for (int b = 0; b < CT / BW; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = k0 + 4 * kq + j;
          float v[BW] = {};
          const float* p = reinterpret_cast<const float*>(bp[b]) + (int64_t)(k0 + j) * a.ldb;
          if (s < s1 && k < kend && bn[b]) __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
          for (int q = 0; q < BW; ++q) o[4 * (b * BW + q) + j] = v[q];
        }
    }
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load_w(s0 + d, wbuf[d]);

  // rows: behind the weights' loads, whose addresses do not wait for the row index
  const T* xp[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    int64_t r = min(r0 + 16 * i + i16, r1 - 1);
    bool in = true;
    if (a.a_rows) {
      r = none ? 0 : a.a_rows[r];
      in = r >= 0 && r < a.a_nrows;
    }
    xp[i] = in ? reinterpret_cast<const T*>(a.A) + r * a.lda + kfirst + kq * EV : nullptr;
  }
  auto load_x = [&](int s, uint4 (&x)[RT]) {
    const int k0 = s * KS;
    const bool in = s < s1 && k0 + kq * EV < kend;
#pragma unroll
    for (int i = 0; i < RT; ++i) x[i] = load_chunk(xp[i] + k0, in && xp[i]);
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load_x(s0 + d, xbuf[d]);

  lin_f32x4 acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = lin_f32x4{0.f, 0.f, 0.f, 0.f};
  uint4* stage = reinterpret_cast<uint4*>(lds) + wv * kStage;
  for (int s = s0; s < s1; s += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      F fb[CT];
      if constexpr (TR) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4* lds_s4;
#pragma unroll
        for (int h = 0; h < CT; ++h) stage[lane + 64 * h] = wbuf[d][h];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          const int k = 8 * kq + (i16 >> 2);
          auto at = [&](int r) {
            return reinterpret_cast<const char*>(stage) + kr(r) * (CT * 32) + (t ^ kx(r)) * 32 + (i16 & 3) * 8;
          };
          const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)at(k));
          const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)at(k + 4));
          fb[t] = __builtin_bit_cast(F, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
      } else {
#pragma unroll
        for (int t = 0; t < CT; ++t) fb[t] = __builtin_bit_cast(F, wbuf[d][t]);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
          acc[i][j] = mma(fb[j], __builtin_bit_cast(F, xbuf[d][i]), acc[i][j]);
      load_w(s + d + D, wbuf[d]);
      load_x(s + d + D, xbuf[d]);
    }
  }

  // sums of the waves, in order
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);
  float* own = sums + wv * BM * SS;
  if constexpr (RT == 1) {
    slab_write_tile<MAP, BW, NCT>(own, acc[0]);
  } else {
#pragma unroll
    for (int i = 0; i < RT; ++i) slab_write_tile<MAP, BW, NCT>(own + 16 * i * SS, acc[i]);
  }
  __syncthreads();
  const int act = none ? PULSAR_ACT_NONE : a.act;
  constexpr int RUNS = BM * NCT * 2;  // of 8 columns
  for (int t = (int)threadIdx.x; t < RUNS; t += 64 * W) {
    const int p = t / (NCT * 2), lc = t % (NCT * 2) * 8, col = n0 + lc;
    const int64_t r = r0 + p;
    if (r >= r1 || col >= f) continue;
    float bias[2][8], v[8], u[8];
    load_bias<PAIR>(a, group, none, col, f, bias);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = u[q] = 0.f;
    for (int w = 0; w < W; ++w) {
      const float* l = sums + (w * BM + p) * SS + lc;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        v[q] += l[q];
        if constexpr (PAIR) u[q] += l[OBN + q];
      }
    }
    finish_run<T, PAIR, true>(a, act, r, col, f, v, u, bias);
  }
}

template <typename T, bool BKC, bool PAIR, int RT, int CT, int W, int D>
int launch_few_shape(LinearArgs& a, hipStream_t s) {
  const int f = PAIR ? a.N / 2 : a.N, obn = (PAIR ? CT / 2 : CT) * 16;
  const int64_t tiles_r = a.offsets
      ? a.rows / (16 * RT) + std::min<int64_t>(a.groups + 1, a.rows)
      : (a.rows + 16 * RT - 1) / (16 * RT);
  const int64_t tiles = tiles_r * ((f + obn - 1) / obn);
  if (tiles > (int64_t)1 << 30) return fail(PULSAR_ERR_INVALID, "linear: launch too large");
  a.max_tiles = (int)tiles_r;
  linear_few_kernel<T, BKC, PAIR, RT, CT, W, D>
      <<<dim3((unsigned)((tiles + kXcds - 1) / kXcds * kXcds), a.part ? a.splits : 1), 64 * W, 0, s>>>(a);
  PULSAR_LAUNCH_CHECK();
  return PULSAR_OK;
}

// (row tiles, column tiles, waves, steps in flight) of each shape, as kFewShapes.
template <typename T, bool BKC, bool PAIR>
int launch_few(LinearArgs& a, int shape, hipStream_t s) {
  switch (shape) {
    case 0:
      if constexpr (!PAIR) return launch_few_shape<T, BKC, PAIR, 1, 1, 8, 8>(a, s);
      break;
    case 1: return launch_few_shape<T, BKC, PAIR, 1, 2, 8, 4>(a, s);
    case 2: return launch_few_shape<T, BKC, PAIR, 2, 2, 8, 4>(a, s);
    case 3: return launch_few_shape<T, BKC, PAIR, 1, 4, 8, 4>(a, s);
    case 4: return launch_few_shape<T, BKC, PAIR, 2, 4, 8, 2>(a, s);
    case 5: return launch_few_shape<T, BKC, PAIR, 4, 4, 4, 2>(a, s);
  }
  return fail(PULSAR_ERR_INVALID, "linear: no such shape");
}

}  // namespace

int launch_linear_few(LinearArgs& a, int dtype, bool b_kc, int shape, hipStream_t s) {
  const bool pair = a.act == PULSAR_ACT_SWIGLU;
  return dispatch_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (b_kc) return pair ? launch_few<T, true, true>(a, shape, s) : launch_few<T, true, false>(a, shape, s);
    return pair ? launch_few<T, false, true>(a, shape, s) : launch_few<T, false, false>(a, shape, s);
  });
}

}  // namespace pulsar
