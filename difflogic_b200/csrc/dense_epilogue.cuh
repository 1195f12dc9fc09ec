// Bias, activation and residual of a dense layer, as the epilogue of its matrix product.
#pragma once

#include "matmul_values.cuh"

namespace dl {

#ifdef __CUDACC__
// Derivatives of the activation are kept for the backward pass, in fp32 or -- bf16 layers -- in fp16 times 2^14: 11 bits, where the
// layer's own type has 8, and down to 4e-12, where sigmoids saturate.  (11 bits are too few for fp16 layers: rounded derivatives and their
// rounded products with the gradient left results 1.76 times as far off as their own rounding does.)
constexpr float kSlopeScale = 16384.f;

// act(z) in place, and its derivatives where they are wanted.
template <bool SLOPE, int N>
__device__ __forceinline__ void activate(float (&z)[N], float (&slope)[N], int act) {
    if (act == DL_ACT_NONE) {
        if (SLOPE) {
#pragma unroll
            for (int j = 0; j < N; ++j) slope[j] = 1.f;
        }
    } else if (act == DL_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (SLOPE) slope[j] = z[j] > 0.f ? 1.f : 0.f;
            z[j] = z[j] > 0.f || z[j] != z[j] ? z[j] : 0.f;
        }
    } else if (act == DL_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float phi = 0.5f * (1.f + erff(z[j] * 0.70710678118654752f));
            // far out the density is zero, and infinity times zero would not be
            if (SLOPE) slope[j] = phi + (fabsf(z[j]) > 15.f ? 0.f : z[j] * expf(-0.5f * z[j] * z[j]) * 0.39894228040143268f);
            z[j] = z[j] == -INFINITY ? 0.f : z[j] * phi;
        }
    } else if (act == DL_ACT_SIGMOID) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            z[j] = __fdividef(1.f, 1.f + expf(-z[j]));   // zero below -88, where expf overflows
            if (SLOPE) slope[j] = z[j] * (1.f - z[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float s = __fdividef(1.f, 1.f + expf(-z[j]));
            if (SLOPE) {
                const float d = s * (1.f - s);
                slope[j] = s + (d == 0.f ? 0.f : z[j] * d);
            }
            z[j] = z[j] == -INFINITY ? 0.f : z[j] * s;
        }
    }
}

// y = act(sum + bias) + residual.  rows_are_features: the rows of the product are the layer's outputs, else its columns are; the result
// lies [batch][feature] or, feature_major, [feature][batch].
struct DenseOutput {
    void *y;
    const void *bias, *residual;
    void *slope;
    int64_t y_pitch, residual_row, residual_col;   // of the residual: values to the product's next row, to its next column
    int type, act;
    bool rows_are_features, feature_major;

    // One output of one sample, where the rows are the features.
    __device__ __forceinline__ void one(int feature, int sample, float sum) const {
        float v[1] = {bias != nullptr ? sum + load_as_float(bias, feature, type) : sum}, d[1];
        activate<true>(v, d, act);
        if (residual != nullptr) v[0] += load_as_float(residual, feature * residual_row + sample * residual_col, type);
        const int64_t i = feature_major ? feature * y_pitch + sample : sample * y_pitch + feature;
        if (type == kFloat32) reinterpret_cast<float *>(y)[i] = v[0];
        else reinterpret_cast<uint16_t *>(y)[i] = to_16bit(v[0], type);
        if (slope != nullptr) {
            if (type != kBFloat16) reinterpret_cast<float *>(slope)[i] = d[0];
            else reinterpret_cast<uint16_t *>(slope)[i] = to_16bit(d[0] * kSlopeScale, kFloat16);
        }
    }
};

// Dense layers of few samples (dense_rows.cu): false where the tensor cores are to be used.
bool dense_rows_applicable(int64_t batch, int type);
int launch_dense_rows(const void *x, int64_t x_pitch, bool x_feature_major, const void *w, const DenseOutput &output, int64_t batch,
                      int64_t inner, int64_t outer, int type, int sms, cudaStream_t st);
#endif  // __CUDACC__

}  // namespace dl
