// Dense layers: y = act(x w^T + bias) + residual and its gradients, by the matrix products of matmul.cuh; what lays out their operands,
// and the entry points.
//
// Forward and backward pass of 8192 samples, 4096 -> 4096, bf16, SiLU and residual: 804 us = 1026 TFLOP/s, of which the forward product
// 244 us (its epilogue reads the residual and writes y and the derivative, which the next tile's products do not all hide), the
// pre-activation's gradient 34 (memory), the input's 198 and the weight's 220.  Small layers are bound by their chain of eight kernels of
// 5 to 20 us, and by the host: 1001 samples, 783 -> 2001, fp16, 90 us from Python and 68 in a captured graph; 128 samples, 784 -> 8000,
// fp32, 90 and 86.
#include <type_traits>

#include "dense_epilogue.cuh"
#include "matmul_launch.cuh"

namespace dl {

int dense_async_error() { return matmul_error_flag(); }

// T: as the values are stored.
template <class T>
__device__ __forceinline__ float to_float(T v) {
    return (float)v;
}
template <class T>
__device__ __forceinline__ T from_float(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}
// Two 16-bit values, packed: conversions of two values at a time run at several times the rate of single ones.
template <class T>
__device__ __forceinline__ uint32_t two_of(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// 64 bytes of neighbouring values, and value j of them.
struct Units {
    uint4 u[4];
};
template <class T>
__device__ __forceinline__ float value_of(const Units &from, int j) {
    constexpr int kUnit = 16 / sizeof(T);
    const uint4 &u = from.u[j / kUnit];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(w[j % 4]);
    } else {
        const uint16_t half = (uint16_t)(w[j % 8 / 2] >> (j % 2 * 16));
        return to_float(*reinterpret_cast<const T *>(&half));
    }
}

// How the derivatives of a layer of T are kept.
template <class T>
using SlopeOf = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __half, float>::type;
template <class T>
constexpr float kScaleOf = std::is_same<T, __nv_bfloat16>::value ? kSlopeScale : 1.f;

// 32 rows of values, a row in each lane, to where they lie in memory: rows `pitch` values apart, those from m on and columns from n on
// left out.  whole: rows lie and end on 16-byte units; else a lane stores a value and a warp the 64 bytes of one row or two at a time.
template <class T>
__device__ __forceinline__ void store_rows(uint8_t *slot, int lane, const float (&v)[64 / sizeof(T)], T *to, int64_t pitch, int row, int col, int m, int n,
                                           bool whole) {
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[j]);
        else w[j] = two_of<T>(v[2 * j], v[2 * j + 1]);
    }
    slot_row(slot, lane, w);
    __syncwarp();
    if (whole) {
        const int r = row + lane / 4, c = col + lane % 4 * (16 / (int)sizeof(T));
        T *at = to + r * pitch + c;
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = *slot_unit(slot, lane, i);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (r + 8 * i < m && c < n) *reinterpret_cast<uint4 *>(at + 8 * i * pitch) = u[i];
    } else {
        constexpr int kRow = 64 / sizeof(T), kAtOnce = 32 / kRow;   // values of a row, rows that 32 lanes take
        const int mine = lane / kRow, c = lane % kRow;
        T *at = to + (row + mine) * pitch + col + c;
#pragma unroll 8
        for (int r = mine; r < 32; r += kAtOnce, at += kAtOnce * pitch) {
            const T value = *reinterpret_cast<const T *>(slot + r * 64 + ((c * (int)sizeof(T) / 16 ^ (r / 2 % 4)) << 4) + c * (int)sizeof(T) % 16);
            if (row + r < m && col + c < n) *at = value;
        }
    }
    __syncwarp();
}

template <class T>
struct DenseEpilogue {
    static constexpr bool kWholeTiles = false;
    static constexpr int kColumns = 64 / sizeof(T);   // 64 bytes
    using Slope = SlopeOf<T>;
    DenseOutput o;
    bool whole;            // rows of y and slope lie and end on 16-byte units
    bool residual_whole;   // those of the residual too
    bool bias_wide;

    struct Place {
        int row, col, m, n;   // of the warp's first value
    };
    __device__ __forceinline__ Place begin(const Tile &, const MatmulShape &s, int row, int col, int) const { return {row, col, s.m, s.n}; }

    struct Ahead {
        uint4 u[4];   // of the residual, as slot_unit's
    };
    __device__ __forceinline__ void fetch(const Place &p, int across, int lane, Ahead &a) const {
        if (!residual_whole) return;
        const int r = p.row + lane / 4, c = p.col + across + lane % 4 * (16 / (int)sizeof(T));
        const T *from = reinterpret_cast<const T *>(o.residual) + r * o.residual_row + c;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            a.u[i] = r + 8 * i < p.m && c < p.n ? *reinterpret_cast<const uint4 *>(from + 8 * i * o.residual_row) : make_uint4(0, 0, 0, 0);
    }

    template <bool SLOPE>
    __device__ __forceinline__ void rows(const Place &p, int across, const float (&v)[kColumns], const Ahead &a, uint8_t *stage, int lane) const {
        const T *bias = reinterpret_cast<const T *>(o.bias), *residual = reinterpret_cast<const T *>(o.residual);
        const int row = p.row + lane, col = p.col + across;
        const bool there = row < p.m;
        constexpr int kUnit = 16 / sizeof(T);   // values of 16 bytes
        float z[kColumns], d[kColumns];
        if (bias == nullptr || o.rows_are_features) {
            const float b = bias != nullptr && there ? to_float(bias[row]) : 0.f;
#pragma unroll
            for (int j = 0; j < kColumns; ++j) z[j] = v[j] + b;
        } else if (bias_wide && col + kColumns <= p.n) {   // the same for all lanes
            Units b;
#pragma unroll
            for (int j = 0; j < 4; ++j) b.u[j] = *reinterpret_cast<const uint4 *>(bias + col + j * kUnit);
#pragma unroll
            for (int j = 0; j < kColumns; ++j) z[j] = v[j] + value_of<T>(b, j);
        } else {
#pragma unroll
            for (int j = 0; j < kColumns; ++j) z[j] = v[j] + (col + j < p.n ? to_float(bias[col + j]) : 0.f);
        }
        activate<SLOPE>(z, d, o.act);
        if (residual != nullptr) {
            if (residual_whole) {
#pragma unroll
                for (int i = 0; i < 4; ++i) *slot_unit(stage, lane, i) = a.u[i];
            } else {
                constexpr int kRow = 64 / sizeof(T), kAtOnce = 32 / kRow;   // as store_rows'
                const int mine = lane / kRow, c = lane % kRow;
#pragma unroll 8
                for (int r = mine; r < 32; r += kAtOnce)
                    *reinterpret_cast<T *>(stage + r * 64 + ((c * (int)sizeof(T) / 16 ^ (r / 2 % 4)) << 4) + c * (int)sizeof(T) % 16) =
                        p.row + r < p.m && col + c < p.n ? residual[(p.row + r) * o.residual_row + (col + c) * o.residual_col] : from_float<T>(0.f);
            }
            __syncwarp();
            Units more;
            slot_read_row(stage, lane, more.u);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kColumns; ++j) z[j] += value_of<T>(more, j);
        }
        store_rows(stage, lane, z, reinterpret_cast<T *>(o.y), o.y_pitch, p.row, col, p.m, p.n, whole);
        if (SLOPE) {
            constexpr int kAtOnce = 64 / sizeof(Slope);   // fp16 layers: two pieces
#pragma unroll
            for (int c = 0; c < kColumns; c += kAtOnce) {
                float part[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) part[j] = d[c + j] * kScaleOf<T>;
                store_rows(stage, lane, part, reinterpret_cast<Slope *>(o.slope), o.y_pitch, p.row, col + c, p.m, p.n, whole);
            }
        }
    }

    // Results that lie the other way: neighbouring lanes have neighbouring values.
    template <bool SLOPE>
    __device__ __forceinline__ void columns(const Place &p, int across, const float (&v)[kColumns], int lane) const {
        const T *bias = reinterpret_cast<const T *>(o.bias), *residual = reinterpret_cast<const T *>(o.residual);
        const int row = p.row + lane, col = p.col + across, left = p.n - col;
        if (row >= p.m) return;
        const float row_bias = bias != nullptr && o.rows_are_features ? to_float(bias[row]) : 0.f;
        float z[kColumns], d[kColumns];
#pragma unroll
        for (int j = 0; j < kColumns; ++j)
            z[j] = v[j] + (bias != nullptr && !o.rows_are_features && j < left ? to_float(bias[col + j]) : row_bias);
        activate<SLOPE>(z, d, o.act);
        if (residual != nullptr) {
            const T *from = residual + row * o.residual_row + col * o.residual_col;
#pragma unroll
            for (int j = 0; j < kColumns; ++j)
                if (j < left) z[j] += to_float(from[j * o.residual_col]);
        }
        T *y = reinterpret_cast<T *>(o.y) + col * o.y_pitch + row;
        Slope *slope = reinterpret_cast<Slope *>(o.slope) + col * o.y_pitch + row;
#pragma unroll
        for (int j = 0; j < kColumns; ++j) {
            if (j >= left) continue;
            y[j * o.y_pitch] = from_float<T>(z[j]);
            if (SLOPE) slope[j * o.y_pitch] = from_float<Slope>(d[j] * kScaleOf<T>);
        }
    }

    __device__ __forceinline__ void piece(const Place &p, int across, const float (&v)[kColumns], const Ahead &a, uint8_t *stage, int lane) const {
        if (p.row >= p.m) return;
        if (o.rows_are_features == o.feature_major) {
            if (o.slope != nullptr) rows<true>(p, across, v, a, stage, lane);
            else rows<false>(p, across, v, a, stage, lane);
        } else {
            if (o.slope != nullptr) columns<true>(p, across, v, lane);
            else columns<false>(p, across, v, lane);
        }
    }
};

// Gradients: the sums as they are, in the layer's type.
template <class T>
struct PlainEpilogue {
    static constexpr bool kWholeTiles = false;
    static constexpr int kColumns = 64 / sizeof(T);
    T *out;
    int64_t pitch;
    bool whole;    // rows lie and end on 16-byte units
    struct Place {
        int row, col, m, n;   // of the warp's first value
    };
    __device__ __forceinline__ Place begin(const Tile &, const MatmulShape &s, int row, int col, int) const { return {row, col, s.m, s.n}; }
    using Ahead = NothingAhead;
    __device__ __forceinline__ void fetch(const Place &, int, int, Ahead &) const {}
    __device__ __forceinline__ void piece(const Place &p, int across, const float (&v)[kColumns], const Ahead &, uint8_t *stage, int lane) const {
        if (p.row < p.m) store_rows(stage, lane, v, out, pitch, p.row, p.col + across, p.m, p.n, whole);
    }
};

// rows x cols values, `pitch` apart, into planes of padded rows: 16-bit types as they are, fp32 as triples.
__global__ void __launch_bounds__(kThreads)
lay_out_kernel(const void *__restrict__ src, int64_t rows, int64_t cols, int64_t pitch, int type, uint16_t *__restrict__ dst, int64_t dst_pitch,
               int64_t plane) {
    grid_dependency_wait();
    grid_dependents_launch();
    const int64_t quads = (cols + 3) / 4, total = rows * quads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t row = i / quads, col = (i - row * quads) * 4, to = row * dst_pitch + col;
        const int valid = (int)(cols - col < 4 ? cols - col : 4);
        float v[4];
        load4(src, row * pitch + col, type, valid, v);
        uint16_t p[3][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (type == kFloat32) split_triple(v[j], p[0][j], p[1][j], p[2][j]);
            else p[0][j] = to_16bit(v[j], type);   // the value itself
        }
        // padded rows: the last quad of a row may write its whole unit
        *reinterpret_cast<ushort4 *>(dst + to) = make_ushort4(p[0][0], p[0][1], p[0][2], p[0][3]);
        if (type == kFloat32) {
            *reinterpret_cast<ushort4 *>(dst + plane + to) = make_ushort4(p[1][0], p[1][1], p[1][2], p[1][3]);
            *reinterpret_cast<ushort4 *>(dst + 2 * plane + to) = make_ushort4(p[2][0], p[2][1], p[2][2], p[2][3]);
        }
    }
}

// gz = gy * slope into planes (none where the gradient of y can be used as it is: dst null), and the sums of its columns (sum_rows: of
// its rows) over a strip of rows.  A block takes 32 lanes x 16 bytes of columns and a strip, 8 rows at a time, four of each warp on their
// way.  WHOLE: rows lie and end on 16-byte units.
template <class T>
constexpr int kGradientColumns = 32 * 16 / (int)sizeof(T);

template <class T, bool WHOLE>
__global__ void __launch_bounds__(kThreads)
pre_gradient_kernel(const T *__restrict__ gy, const void *__restrict__ slope, int64_t rows, int64_t cols, uint16_t *__restrict__ dst,
                    int64_t dst_pitch, int64_t plane, int64_t strip, float *__restrict__ partial, int sum_rows) {
    using Slope = SlopeOf<T>;
    constexpr int kValues = 16 / sizeof(T), kAhead = 4, kGroups = kThreads / 32;
    __shared__ float s_sum[kGroups][kGradientColumns<T>];
    grid_dependency_wait();
    grid_dependents_launch();
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const int64_t col = (int64_t)blockIdx.x * kGradientColumns<T> + lane * kValues, first = (int64_t)blockIdx.y * strip,
                  last = first + strip < rows ? first + strip : rows;
    const int left = (int)(cols - col < kValues ? cols - col : kValues);
    const Slope *slopes = reinterpret_cast<const Slope *>(slope);
    float total[kValues] = {};
    struct __align__(16) Pack {
        T v[kValues];
    };
    struct __align__(16) SlopePack {
        Slope v[kValues];
    };
    for (int64_t row = first + group; row < last; row += kGroups * kAhead) {
        float v[kAhead][kValues];
        if constexpr (WHOLE) {
            Pack g[kAhead];
            SlopePack d[kAhead];
            const bool there = left > 0;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int64_t r = row + i * kGroups < last ? row + i * kGroups : last - 1, at = r * cols + (there ? col : 0);
                g[i] = *reinterpret_cast<const Pack *>(gy + at);
                if (slope != nullptr) d[i] = *reinterpret_cast<const SlopePack *>(slopes + at);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int j = 0; j < kValues; ++j) {
                    v[i][j] = there && row + i * kGroups < last ? to_float(g[i].v[j]) : 0.f;
                    if (slope != nullptr) v[i][j] *= to_float(d[i].v[j]) * (1.f / kScaleOf<T>);
                }
        } else {
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int j = 0; j < kValues; ++j) {
                    const int64_t r = row + i * kGroups, at = r * cols + col + j;
                    v[i][j] = r < last && j < left ? to_float(gy[at]) : 0.f;
                    if (slope != nullptr && r < last && j < left) v[i][j] *= to_float(slopes[at]) * (1.f / kScaleOf<T>);
                }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * kGroups;
            if (dst != nullptr && r < last && left > 0) {   // planes' rows are padded: a whole unit may be written
                uint16_t *to = dst + r * dst_pitch + col;
                if constexpr (sizeof(T) == 4) {
                    uint16_t p[3][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) split_triple(v[i][j], p[0][j], p[1][j], p[2][j]);
#pragma unroll
                    for (int q = 0; q < 3; ++q)
                        *reinterpret_cast<ushort4 *>(to + q * plane) = make_ushort4(p[q][0], p[q][1], p[q][2], p[q][3]);
                } else {
                    *reinterpret_cast<uint4 *>(to) = make_uint4(two_of<T>(v[i][0], v[i][1]), two_of<T>(v[i][2], v[i][3]), two_of<T>(v[i][4], v[i][5]),
                                                                two_of<T>(v[i][6], v[i][7]));
                }
            }
            float r_sum = 0.f;
#pragma unroll
            for (int j = 0; j < kValues; ++j) {
                total[j] += v[i][j];
                r_sum += v[i][j];
            }
            if (partial != nullptr && sum_rows) {   // the features are rows: this row's share of the block's samples
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) r_sum += __shfl_xor_sync(0xffffffffu, r_sum, off);
                if (lane == 0 && r < last) partial[(int64_t)blockIdx.x * rows + r] = r_sum;
            }
        }
    }
    if (partial == nullptr || sum_rows) return;
#pragma unroll
    for (int j = 0; j < kValues; ++j) s_sum[group][lane * kValues + j] = total[j];
    __syncthreads();
    if (threadIdx.x >= kGradientColumns<T>) return;
    const int64_t c = (int64_t)blockIdx.x * kGradientColumns<T> + threadIdx.x;
    if (c >= cols) return;
    float r = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) r += s_sum[g][threadIdx.x];
    partial[blockIdx.y * cols + c] = r;
}

template <class T>
static void launch_pre_gradient(const void *gy, const void *slope, int64_t rows, int64_t cols, uint16_t *dst, int64_t dst_pitch, int64_t plane,
                                int64_t strips, int64_t strip, float *partial, int sum_rows, cudaStream_t st) {
    const dim3 grid((unsigned)ceil_div(cols, kGradientColumns<T>), (unsigned)strips);
    const bool whole = aligned_to(gy, 16) && aligned_to(slope, 16) && cols * sizeof(T) % 16 == 0;
    launch_dependent(true, whole ? pre_gradient_kernel<T, true> : pre_gradient_kernel<T, false>, grid, dim3(kThreads), 0, st,
                     reinterpret_cast<const T *>(gy), slope, rows, cols, dst, dst_pitch, plane, strip, partial, sum_rows);
}

// Adds the partial sums up, in their order.
__global__ void __launch_bounds__(kThreads)
bias_gradient_kernel(const float *__restrict__ partial, int64_t parts, int64_t features, void *__restrict__ out, int type) {
    grid_dependency_wait();
    grid_dependents_launch();
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= features) return;
    float r = 0.f;
    for (int64_t p = 0; p < parts; ++p) r += partial[p * features + i];
    if (type == kFloat32) reinterpret_cast<float *>(out)[i] = r;
    else reinterpret_cast<uint16_t *>(out)[i] = to_16bit(r, type);
}

// What of an operand the copies can read in place: 16-bit values whose base and rows lie on units of 16 bytes.
static bool in_place(const void *p, int64_t pitch, int type) { return type != kFloat32 && aligned_to(p, 16) && pitch % 8 == 0; }

struct DenseLayout {
    int planes;
    int64_t x_rows, x_cols, x_pitch;   // as it lies in memory
    bool lay_x, lay_w;
    int64_t x_plane_pitch, x_plane, w_plane_pitch, w_plane;   // of the planes that the library lays out
    int64_t x_bytes, w_bytes;
};

static DenseLayout dense_layout(int64_t batch, int64_t inner, int64_t outer, int64_t x_pitch, bool x_feature_major, int type, const void *x,
                                const void *w) {
    DenseLayout l = {};
    l.planes = type == kFloat32 ? 3 : 1;
    l.x_rows = x_feature_major ? inner : batch;
    l.x_cols = x_feature_major ? batch : inner;
    l.x_pitch = x_pitch;
    l.lay_x = !in_place(x, x_pitch, type);
    l.lay_w = !in_place(w, inner, type);
    l.x_plane_pitch = padded(l.x_cols);
    l.x_plane = l.x_rows * l.x_plane_pitch;
    l.w_plane_pitch = padded(inner);
    l.w_plane = outer * l.w_plane_pitch;
    l.x_bytes = l.lay_x ? padded_bytes(l.planes * l.x_plane * 2) : 0;
    l.w_bytes = l.lay_w ? padded_bytes(l.planes * l.w_plane * 2) : 0;
    return l;
}

static int lay_out(const void *src, int64_t rows, int64_t cols, int64_t pitch, int type, void *dst, int64_t dst_pitch, int64_t plane, int sms,
                   cudaStream_t st, const char *what) {
    int64_t blocks = ceil_div(rows * ceil_div(cols, 4), kThreads);
    if (blocks > 16 * sms) blocks = 16 * sms;
    launch_dependent(true, lay_out_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, src, rows, cols, pitch, type,
                     reinterpret_cast<uint16_t *>(dst), dst_pitch, plane);
    return launch_status(what);
}

template <class T>
static bool whole_units(const void *p, int64_t values) {
    return aligned_to(p, 16) && values * sizeof(T) % 16 == 0;
}

template <int PLANES, class T>
static int launch_layer(const Product &p, const MatmulPlan &plan, const DenseOutput &o, float *partial, int sms, cudaStream_t st, const char *what) {
    DenseEpilogue<T> e = {};
    e.o = o;
    e.bias_wide = aligned_to(o.bias, 16);
    e.whole = whole_units<T>(o.y, p.n) && whole_units<T>(o.y, o.y_pitch) && (o.slope == nullptr || aligned_to(o.slope, 16));
    e.residual_whole = o.residual != nullptr && o.rows_are_features == o.feature_major && o.residual_col == 1 && whole_units<T>(o.residual, p.n) &&
                       whole_units<T>(o.residual, o.residual_row);
    return launch_product<PLANES>(p, plan, e, partial, sms, st, what);
}

// Whether the layer's outputs are the rows of the product: as they lie in the result, so that neighbouring columns are stored by
// neighbouring lanes; but few samples fill half of a tile's 64 columns rather than half of its 128 rows.
static bool features_as_rows(int64_t batch, bool feature_major) { return feature_major || batch <= 64; }

static MatmulPlan plan_forward(int64_t batch, int64_t inner, int64_t outer, bool feature_major, int planes, int sms, int choice) {
    return features_as_rows(batch, feature_major) ? plan_matmul(outer, batch, inner, 1, planes, false, sms, choice)
                                                  : plan_matmul(batch, outer, inner, 1, planes, false, sms, choice);
}

static int gradient_columns(int type) { return type == kFloat32 ? kGradientColumns<float> : kGradientColumns<__half>; }

// Strips of rows of a pre-activation gradient, enough for whole SMs.
static int64_t strips_of(int64_t rows, int64_t cols, int type, int sms, int64_t *strip) {
    int64_t strips = ceil_div(4 * sms, ceil_div(cols, gradient_columns(type)));
    if (strips > ceil_div(rows, 32)) strips = ceil_div(rows, 32);
    if (strips > 65535) strips = 65535;
    *strip = ceil_div(rows, strips);
    return ceil_div(rows, *strip);
}

static bool dense_sizes(int64_t batch, int64_t inner, int64_t outer, int type, const char *what, int *status) {
    *status = DL_OK;
    if (batch < 0 || inner <= 0 || outer <= 0 || batch > INT32_MAX / 2 || inner > INT32_MAX / 2 || outer > INT32_MAX / 2)
        *status = fail(DL_ERR_INVALID_ARG, "%s: bad size", what);
    else if (type < kFloat32 || type > kFloat16)
        *status = fail(DL_ERR_INVALID_ARG, "%s: unknown type %d", what, type);
    return *status == DL_OK;
}

}  // namespace dl

using namespace dl;

extern "C" DL_API void dl_dense_forward_sizes(const void *x, int64_t x_pitch, int x_feature_major, const void *w, int64_t batch, int64_t inner,
                                             int64_t outer, int y_feature_major, int type, int64_t *sizes) {
    const int choice = matmul_choice(&type);
    sizes[0] = sizes[1] = sizes[2] = 0;
    if (batch <= 0 || inner <= 0 || outer <= 0 || dense_rows_applicable(batch, type)) return;
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    sizes[0] = l.x_bytes;
    sizes[1] = l.w_bytes;
    sizes[2] = plan_forward(batch, inner, outer, y_feature_major != 0, l.planes, current_sms(), choice).partial_bytes;
}

extern "C" DL_API int64_t dl_dense_planes_bytes(int64_t rows, int64_t cols, int type) {
    if (rows <= 0 || cols <= 0) return 0;
    return padded_bytes((type == kFloat32 ? 3 : 1) * rows * padded(cols) * 2);
}

extern "C" DL_API int dl_dense_lay_out(const void *src, int64_t rows, int64_t cols, int64_t pitch, int type, void *planes, void *stream) {
    const char *what = "dl_dense_lay_out";
    int status;
    if (!dense_sizes(0, rows, cols, type, what, &status)) return status;
    DL_REQUIRE(src && planes && aligned_to(planes, 16), DL_ERR_INVALID_ARG, "%s: null pointer or planes that are not 16-byte aligned", what);
    DL_REQUIRE(pitch >= cols, DL_ERR_INVALID_ARG, "%s: rows overlap", what);
    return lay_out(src, rows, cols, pitch, type, planes, padded(cols), rows * padded(cols), current_sms(), as_stream(stream), what);
}

extern "C" DL_API int dl_dense_forward(const void *x, int64_t x_pitch, int x_feature_major, const void *w, const void *bias, const void *residual,
                                       int64_t residual_batch, int64_t residual_feature, int act, void *y, int y_feature_major, void *slope,
                                       void *x_planes, void *w_planes, void *workspace, int64_t batch, int64_t inner, int64_t outer, int type,
                                       void *stream) {
    const char *what = "dl_dense_forward";
    const int choice = matmul_choice(&type);
    int status;
    if (!dense_sizes(batch, inner, outer, type, what, &status)) return status;
    DL_REQUIRE(act >= DL_ACT_NONE && act <= DL_ACT_GELU, DL_ERR_INVALID_ARG, "%s: unknown activation %d", what, act);
    if (batch == 0) return DL_OK;
    DL_REQUIRE(x && w && y, DL_ERR_INVALID_ARG, "%s: null pointer", what);
    DL_REQUIRE(x_pitch >= (x_feature_major ? batch : inner), DL_ERR_INVALID_ARG, "%s: rows of x overlap", what);
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    const int sms = current_sms();
    cudaStream_t st = as_stream(stream);
    if (dense_rows_applicable(batch, type)) {
        const DenseOutput e = {y, bias, residual, slope, y_feature_major ? batch : outer, residual_feature, residual_batch, type, act, true,
                               y_feature_major != 0};
        return launch_dense_rows(x, x_pitch, x_feature_major != 0, w, e, batch, inner, outer, type, sms, st);
    }
    const MatmulPlan plan = plan_forward(batch, inner, outer, y_feature_major != 0, l.planes, sms, choice);
    DL_REQUIRE((!l.lay_x || x_planes) && (!l.lay_w || w_planes) && (plan.partial_bytes == 0 || workspace), DL_ERR_INVALID_ARG,
               "%s: a workspace is missing", what);
    DL_REQUIRE(aligned_to(x_planes, 16) && aligned_to(w_planes, 16) && aligned_to(workspace, 16), DL_ERR_INVALID_ARG,
               "%s: workspaces must be 16-byte aligned", what);
    if (l.lay_x && (status = lay_out(x, l.x_rows, l.x_cols, x_pitch, type, x_planes, l.x_plane_pitch, l.x_plane, sms, st, what)) != DL_OK) return status;
    if (l.lay_w && (status = lay_out(w, outer, inner, inner, type, w_planes, l.w_plane_pitch, l.w_plane, sms, st, what)) != DL_OK) return status;
    const Operand ox = {l.lay_x ? x_planes : x, l.lay_x ? l.x_plane_pitch : x_pitch, l.x_plane, x_feature_major != 0};
    const Operand ow = {l.lay_w ? w_planes : w, l.lay_w ? l.w_plane_pitch : inner, l.w_plane, false};
    const bool rows_are_features = features_as_rows(batch, y_feature_major != 0);
    Product p = {};
    p.a = rows_are_features ? ow : ox;
    p.b = rows_are_features ? ox : ow;
    p.m = rows_are_features ? outer : batch;
    p.n = rows_are_features ? batch : outer;
    p.k = inner;
    p.batch = 1;
    p.planes = p.planes_z = l.planes;
    p.bfloat = type != kFloat16;
    p.exact = true;
    const DenseOutput o = {y, bias, residual, slope, y_feature_major ? batch : outer, rows_are_features ? residual_feature : residual_batch,
                           rows_are_features ? residual_batch : residual_feature, type, act, rows_are_features, y_feature_major != 0};
    float *partial = reinterpret_cast<float *>(workspace);
    if (type == kFloat32) return launch_layer<3, float>(p, plan, o, partial, sms, st, what);
    if (type == kBFloat16) return launch_layer<1, __nv_bfloat16>(p, plan, o, partial, sms, st, what);
    return launch_layer<1, __half>(p, plan, o, partial, sms, st, what);
}

namespace dl {

template <int PLANES, class T>
static int launch_gradient(const Product &p, const MatmulPlan &plan, void *out, int64_t pitch, float *partial, int sms, cudaStream_t st,
                           const char *what) {
    PlainEpilogue<T> e = {};
    e.out = reinterpret_cast<T *>(out);
    e.pitch = pitch;
    e.whole = whole_units<T>(out, p.n) && whole_units<T>(out, pitch);
    return launch_product<PLANES>(p, plan, e, partial, sms, st, what);
}
static int launch_gradient(const Product &p, const MatmulPlan &plan, void *out, int64_t pitch, int type, float *partial, int sms, cudaStream_t st,
                           const char *what) {
    if (type == kFloat32) return launch_gradient<3, float>(p, plan, out, pitch, partial, sms, st, what);
    if (type == kBFloat16) return launch_gradient<1, __nv_bfloat16>(p, plan, out, pitch, partial, sms, st, what);
    return launch_gradient<1, __half>(p, plan, out, pitch, partial, sms, st, what);
}

struct DenseBackward {
    int planes;
    bool lay_gz;
    int64_t g_rows, g_cols, g_pitch, g_plane, strips, strip, parts;
    MatmulPlan to_x, to_w;
    int64_t g_bytes, bias_bytes, partial_bytes, x_bytes, w_bytes;   // workspace: gz planes, partial bias sums, splits of a product, x and w laid out
    int64_t total() const { return g_bytes + bias_bytes + partial_bytes + x_bytes + w_bytes; }
};

static DenseBackward plan_backward(const DenseLayout &l, int64_t batch, int64_t inner, int64_t outer, bool g_feature_major, int type, bool act,
                                   const void *gy, bool lay_x, bool lay_w, int sms, int choice) {
    DenseBackward b = {};
    b.planes = type == kFloat32 ? 3 : 1;
    b.g_rows = g_feature_major ? outer : batch;
    b.g_cols = g_feature_major ? batch : outer;
    b.lay_gz = act || !in_place(gy, b.g_cols, type);
    b.g_pitch = padded(b.g_cols);
    b.g_plane = b.g_rows * b.g_pitch;
    b.g_bytes = b.lay_gz ? padded_bytes(b.planes * b.g_plane * 2) : 0;
    b.strips = strips_of(b.g_rows, b.g_cols, type, sms, &b.strip);
    b.parts = g_feature_major ? ceil_div(b.g_cols, gradient_columns(type)) : b.strips;
    b.bias_bytes = padded_bytes(b.parts * outer * 4);
    b.to_x = plan_matmul(batch, inner, outer, 1, b.planes, false, sms, choice);
    b.to_w = plan_matmul(outer, inner, batch, 1, b.planes, false, sms, choice);
    b.partial_bytes = padded_bytes(b.to_x.partial_bytes > b.to_w.partial_bytes ? b.to_x.partial_bytes : b.to_w.partial_bytes);
    b.x_bytes = lay_x ? l.x_bytes : 0;
    b.w_bytes = lay_w ? l.w_bytes : 0;
    return b;
}

}  // namespace dl

extern "C" DL_API int64_t dl_dense_backward_workspace_bytes(const void *gy, int g_feature_major, int has_slope, const void *x, int64_t x_pitch,
                                                            int x_feature_major, const void *w, int lay_x, int lay_w, int64_t batch, int64_t inner,
                                                            int64_t outer, int type) {
    const int choice = matmul_choice(&type);
    if (batch <= 0 || inner <= 0 || outer <= 0) return 0;
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    return plan_backward(l, batch, inner, outer, g_feature_major != 0, type, has_slope != 0, gy, lay_x != 0, lay_w != 0, current_sms(), choice).total();
}

extern "C" DL_API int dl_dense_backward(const void *gy, int g_feature_major, const void *slope, const void *x, int64_t x_pitch, int x_feature_major,
                                        const void *w, const void *x_planes, const void *w_planes, void *gx, void *gw, void *gb, void *workspace,
                                        int64_t batch, int64_t inner, int64_t outer, int type, void *stream) {
    const char *what = "dl_dense_backward";
    const int choice = matmul_choice(&type);
    int status;
    if (!dense_sizes(batch, inner, outer, type, what, &status)) return status;
    DL_REQUIRE(batch > 0, DL_ERR_INVALID_ARG, "%s: empty batch", what);
    DL_REQUIRE(gy && (x || !gw || x_planes) && (w || !gx || w_planes), DL_ERR_INVALID_ARG, "%s: null pointer", what);
    DL_REQUIRE(workspace && aligned_to(workspace, 16), DL_ERR_INVALID_ARG, "%s: the workspace is missing or not 16-byte aligned", what);
    const int sms = current_sms();
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    const bool lay_x = gw && l.lay_x && !x_planes, lay_w = gx && l.lay_w && !w_planes;
    const DenseBackward b = plan_backward(l, batch, inner, outer, g_feature_major != 0, type, slope != nullptr, gy, lay_x, lay_w, sms, choice);
    DL_REQUIRE((!lay_x || x) && (!lay_w || w), DL_ERR_INVALID_ARG, "%s: null pointer", what);
    cudaStream_t st = as_stream(stream);
    uint8_t *at = reinterpret_cast<uint8_t *>(workspace);
    uint16_t *gz = reinterpret_cast<uint16_t *>(at);
    float *sums = reinterpret_cast<float *>(at + b.g_bytes), *partial = reinterpret_cast<float *>(at + b.g_bytes + b.bias_bytes);
    if (lay_x) {
        void *to = at + b.total() - b.w_bytes - b.x_bytes;
        if ((status = lay_out(x, l.x_rows, l.x_cols, x_pitch, type, to, l.x_plane_pitch, l.x_plane, sms, st, what)) != DL_OK) return status;
        x_planes = to;
    }
    if (lay_w) {
        void *to = at + b.total() - b.w_bytes;
        if ((status = lay_out(w, outer, inner, inner, type, to, l.w_plane_pitch, l.w_plane, sms, st, what)) != DL_OK) return status;
        w_planes = to;
    }
    if (b.lay_gz || gb) {
        const auto launch = type == kFloat32 ? launch_pre_gradient<float> : type == kBFloat16 ? launch_pre_gradient<__nv_bfloat16> : launch_pre_gradient<__half>;
        launch(gy, slope, b.g_rows, b.g_cols, b.lay_gz ? gz : nullptr, b.g_pitch, b.g_plane, b.strips, b.strip, gb ? sums : nullptr, g_feature_major, st);
        if ((status = launch_status(what)) != DL_OK) return status;
    }
    if (gb) {
        launch_dependent(true, bias_gradient_kernel, dim3((unsigned)ceil_div(outer, kThreads)), dim3(kThreads), 0, st, (const float *)sums, b.parts,
                         outer, gb, type);
        if ((status = launch_status(what)) != DL_OK) return status;
    }
    Operand g = {b.lay_gz ? (const void *)gz : gy, b.lay_gz ? b.g_pitch : b.g_cols, b.g_plane, false};
    Product p = {};
    p.batch = 1;
    p.planes = p.planes_z = b.planes;
    p.bfloat = type != kFloat16;
    p.exact = true;
    if (gx) {   // gz [batch][outer] w [outer][inner], summed over the outputs
        p.a = g;
        p.a.mn = g_feature_major != 0;
        p.b = {l.lay_w ? w_planes : w, l.lay_w ? l.w_plane_pitch : inner, l.w_plane, true};
        p.m = batch;
        p.n = inner;
        p.k = outer;
        if ((status = launch_gradient(p, b.to_x, gx, inner, type, partial, sms, st, what)) != DL_OK) return status;
    }
    if (gw) {   // gz^T x, summed over the batch
        p.a = g;
        p.a.mn = g_feature_major == 0;
        p.b = {l.lay_x ? x_planes : x, l.lay_x ? l.x_plane_pitch : x_pitch, l.x_plane, x_feature_major == 0};
        p.m = outer;
        p.n = inner;
        p.k = batch;
        if ((status = launch_gradient(p, b.to_w, gw, inner, type, partial, sms, st, what)) != DL_OK) return status;
    }
    return DL_OK;
}

