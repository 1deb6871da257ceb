// Dense and ragged products with their epilogues (linear.hip): arguments and the parts shared
// with the activation kernels.
#pragma once

#include "common.h"

namespace pulsar {

typedef __bf16 lin_bf16x8 __attribute__((ext_vector_type(8)));
typedef float lin_f32x4 __attribute__((ext_vector_type(4)));

// One launch: C[m][n] = sum_k A[m][k] B[n][k] over each group.
//   Products (forward, gradient of x): m runs over the ragged rows, n and k over the weight's
//   two dimensions. Rows of group e are [offsets[e], offsets[e + 1]); rows past the last group
//   are written as zeros. offsets == nullptr: one group of `rows` rows.
//   Weight gradient: m and n run over the weight's dimensions, k over the rows of the group.
struct LinearArgs {
  const void* A;
  const void* B;
  int64_t lda, ldb;        // elements from one row of the stored matrix to the next
  int64_t b_group;         // products: elements from one group's weight to the next
  const int32_t* a_rows;   // row i of A is stored row a_rows[i] (nullptr: i)
  const int32_t* b_rows;   // the same of B (weight gradient)
  int64_t a_nrows, b_nrows;  // stored rows; an index outside them reads as a row of zeros
  const int32_t* offsets;
  int groups;
  int rows;                // ragged rows in all
  int M, N, K;             // M: weight gradient only; K: products only
  int up;                  // SwiGLU: B's first row or column of the up projection
  void* C;
  int64_t ldc, c_group;
  void* pre;               // products: pre-activation values (nullptr: not kept)
  int64_t ldpre;
  const void* bias;        // products: [groups][N] (nullptr: none)
  int bias_dtype;
  const void* residual;    // products: added after the activation (nullptr: none)
  int64_t ldr;
  int act;
  void* db;                // weight gradient: [groups][dim] sums of dpre's rows, storage type
  int splits;              // workgroups that share a sum over k; with several, partial sums:
  float* part;             //   weight gradient: [split][groups][M][N], products (dense): [split][rows][N]
  float* part_db;          //   weight gradient: [split][groups][dim]
  int tiles_m, tiles_n;    // weight gradient: tiles of one group
  int max_tiles;           // products: bound of the row tiles
};

// Products with few rows a group (linear_few.hip), in shapes of 16-row and 16-column tiles of a
// workgroup (the first not for SwiGLU).
struct FewShape {
  int rt, ct;
};
constexpr FewShape kFewShapes[6] = {{1, 1}, {1, 2}, {2, 2}, {1, 4}, {2, 4}, {4, 4}};
// Few or many, a split of k is whole chunks of 128 bytes: the k's [first, first + count) of split `s`.
template <typename T>
__host__ __device__ inline void split_range(int K, int splits, int s, int& first, int& count) {
  constexpr int BK = 128 / (int)sizeof(T);
  const int per = ((K + splits - 1) / splits + BK - 1) / BK * BK;
  first = (int)((int64_t)s * per < K ? (int64_t)s * per : K);
  count = K - first < per ? K - first : per;
}
int launch_linear_few(LinearArgs& a, int dtype, bool b_kc, int shape, hipStream_t s);

// Sigmoid by the exponential and reciprocal instructions: each within one step of fp32, the
// argument's scaling to base 2 within |v| half steps, so that v sigmoid(v) is off by at most
// (3 + v^2 e^-|v|) half steps.
__device__ __forceinline__ float fast_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504f));
}

// The activation of 8 values, chosen once for them.
__device__ __forceinline__ void act_values(int act, float (&v)[8]) {
  switch (act) {
    case PULSAR_ACT_RELU:
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = v[q] < 0.f ? 0.f : v[q];  // NaN stays NaN
      break;
    case PULSAR_ACT_SILU:
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] *= fast_sigmoid(v[q]);
      break;
    case PULSAR_ACT_GELU:
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] *= 0.5f * (1.f + erff(v[q] * 0.70710678f));
      break;
    case PULSAR_ACT_GELU_TANH:
      // 0.5 (1 + tanh(u)) = sigmoid(2 u)
#pragma unroll
      for (int q = 0; q < 8; ++q)
        v[q] *= fast_sigmoid(1.59576912f * (v[q] + 0.044715f * v[q] * v[q] * v[q]));
      break;
    case PULSAR_ACT_SIGMOID:
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = fast_sigmoid(v[q]);
      break;
    default: break;
  }
}
// The activation's derivative.
// The slopes are taken at v held to a range past which they are 0 or 1 in fp32, so that no
// infinite v meets a zero factor (NaN passes through).
__device__ __forceinline__ float hold(float v, float b) { return v > b ? b : (v < -b ? -b : v); }
__device__ __forceinline__ float act_slope(int act, float v) {
  switch (act) {
    case PULSAR_ACT_RELU: return v > 0.f ? 1.f : (v <= 0.f ? 0.f : v);
    case PULSAR_ACT_SILU: {
      v = hold(v, 100.f);
      const float s = fast_sigmoid(v);
      return s * (1.f + v * (1.f - s));
    }
    case PULSAR_ACT_GELU:
      v = hold(v, 30.f);
      return 0.5f * (1.f + erff(v * 0.70710678f)) + v * 0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * v * v);
    case PULSAR_ACT_GELU_TANH: {
      v = hold(v, 30.f);
      const float v2 = v * v;
      const float s = fast_sigmoid(1.59576912f * v * (1.f + 0.044715f * v2));
      return s + v * s * (1.f - s) * 1.59576912f * (1.f + 0.134145f * v2);
    }
    case PULSAR_ACT_SIGMOID: {
      const float s = fast_sigmoid(v);
      return s * (1.f - s);
    }
    default: return 1.f;
  }
}

}  // namespace pulsar
