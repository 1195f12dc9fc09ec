// Bias, activation and residual of a dense layer, as the epilogue of its matrix product.
#pragma once

#include "matmul_values.cuh"

namespace dl {

#ifdef __CUDACC__
// Derivatives of the activation are kept for the backward pass, in fp32 or -- 16-bit layers -- in fp16 times 2^14: 11 bits, where the
// layer's own type may have 8, and down to 4e-12, where sigmoids saturate.
constexpr float kSlopeScale = 16384.f;

// act(z) in place, and its derivatives, four at a time.
template <int N>
__device__ __forceinline__ void activate(float (&z)[N], float (&slope)[N], int act) {
    if (act == DL_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < N; ++j) slope[j] = 1.f;
    } else if (act == DL_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            slope[j] = z[j] > 0.f ? 1.f : 0.f;
            z[j] = z[j] > 0.f || z[j] != z[j] ? z[j] : 0.f;
        }
    } else if (act == DL_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float phi = 0.5f * (1.f + erff(z[j] * 0.70710678118654752f));
            // far out the density is zero, and infinity times zero would not be
            slope[j] = phi + (fabsf(z[j]) > 15.f ? 0.f : z[j] * expf(-0.5f * z[j] * z[j]) * 0.39894228040143268f);
            z[j] = z[j] == -INFINITY ? 0.f : z[j] * phi;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float s = __fdividef(1.f, 1.f + expf(-z[j]));   // zero below -88, where expf overflows
            slope[j] = s * (1.f - s);
            if (act == DL_ACT_SIGMOID) {
                z[j] = s;
            } else {
                slope[j] = s + (slope[j] == 0.f ? 0.f : z[j] * slope[j]);
                z[j] = z[j] == -INFINITY ? 0.f : z[j] * s;
            }
        }
    }
}

// y = act(sum + bias) + residual.  rows_are_features: the rows of the product are the layer's outputs, else its columns are; the result
// lies [batch][feature] or, feature_major, [feature][batch].
struct DenseEpilogue {
    static constexpr int kPlanes = 3;
    void *y;
    const void *bias, *residual;
    void *slope;
    int64_t y_pitch, residual_row, residual_col;   // of the residual: values to the product's next row, to its next column
    int type, act;
    bool rows_are_features, feature_major;

    // Neighbouring columns of the product are neighbours in memory, or neighbouring rows are.
    __device__ __forceinline__ bool by_column(int, int) const { return rows_are_features != feature_major; }
    __device__ __forceinline__ bool by_row(int, int) const { return rows_are_features == feature_major; }

    // One output of one sample.
    __device__ __forceinline__ void one(int feature, int sample, float sum) const {
        float v[1] = {bias != nullptr ? sum + load_as_float(bias, feature, type) : sum}, d[1];
        activate(v, d, act);
        // residual_row: to the next feature, as rows_are_features
        if (residual != nullptr) v[0] += load_as_float(residual, feature * residual_row + sample * residual_col, type);
        const int64_t i = feature_major ? feature * y_pitch + sample : sample * y_pitch + feature;
        if (type == kFloat32) reinterpret_cast<float *>(y)[i] = v[0];
        else reinterpret_cast<uint16_t *>(y)[i] = to_16bit(v[0], type);
        if (slope != nullptr) {
            if (type == kFloat32) reinterpret_cast<float *>(slope)[i] = d[0];
            else reinterpret_cast<uint16_t *>(slope)[i] = to_16bit(d[0] * kSlopeScale, kFloat16);
        }
    }

    template <int N>
    __device__ __forceinline__ void down(int, int row, int col, const float (&sum)[N], int m, int valid) const {
        if (row >= m) return;
        const float row_bias = bias != nullptr && rows_are_features ? load_as_float(bias, row, type) : 0.f;
        float v[N], d[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = sum[j] + row_bias;
            if (bias != nullptr && !rows_are_features && j < valid) v[j] += load_as_float(bias, col + j, type);
        }
        activate(v, d, act);
        if (residual != nullptr) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j < valid) v[j] += load_as_float(residual, row * residual_row + (col + j) * residual_col, type);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (j >= valid) continue;
            const int64_t i = (col + j) * y_pitch + row;
            if (type == kFloat32) reinterpret_cast<float *>(y)[i] = v[j];
            else reinterpret_cast<uint16_t *>(y)[i] = to_16bit(v[j], type);
            if (slope != nullptr) {
                if (type == kFloat32) reinterpret_cast<float *>(slope)[i] = d[j];
                else reinterpret_cast<uint16_t *>(slope)[i] = to_16bit(d[j] * kSlopeScale, kFloat16);
            }
        }
    }
    template <int N, int STEP>
    __device__ __forceinline__ void across(int, int row, int col, const float (&sum)[N][4], int m, int valid) const {
        float col_bias[4] = {0.f, 0.f, 0.f, 0.f}, more[N][4];
        if (bias != nullptr && !rows_are_features) load4(bias, col, type, valid, col_bias);
        if (residual != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = row + i * STEP;
                if (residual_col == 1) {
                    load4(residual, r * residual_row + col, type, r < m ? valid : 0, more[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) more[i][j] = r < m && j < valid ? load_as_float(residual, r * residual_row + (col + j) * residual_col, type) : 0.f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row + i * STEP;
            if (r >= m) break;
            const float row_bias = bias != nullptr && rows_are_features ? load_as_float(bias, r, type) : 0.f;
            float v[4], d[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = sum[i][j] + (rows_are_features ? row_bias : col_bias[j]);
            activate(v, d, act);
            if (residual != nullptr) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += more[i][j];
            }
            const int64_t at = r * y_pitch + col;
            store4(y, at, type, valid, v);
            if (slope != nullptr) {
                if (type != kFloat32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[j] *= kSlopeScale;
                }
                store4(slope, at, type == kFloat32 ? kFloat32 : kFloat16, valid, d);
            }
        }
    }
};

// Dense layers of few samples (dense_rows.cu): false where the tensor cores are to be used.
bool dense_rows_applicable(int64_t batch, int type);
int launch_dense_rows(const void *x, int64_t x_pitch, bool x_feature_major, const void *w, const DenseEpilogue &epilogue, int64_t batch,
                      int64_t inner, int64_t outer, int type, int sms, cudaStream_t st);
#endif  // __CUDACC__

}  // namespace dl
