// Dense layers: y = act(x w^T + bias) + residual and its gradients, by the matrix products of matmul.cuh; what lays out their operands,
// and the entry points.
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
template <class T>
struct __align__(4 * sizeof(T)) Quad {
    T v[4];
};
// Four neighbouring values of which `left` are there; wide: their address is a multiple of their size.
template <class T>
__device__ __forceinline__ void read_quad(const T *p, bool wide, int left, float (&v)[4]) {
    if (wide && left >= 4) {
        const Quad<T> q = *reinterpret_cast<const Quad<T> *>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_float(q.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < left ? to_float(p[j]) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void write_quad(T *p, bool wide, int left, const float (&v)[4]) {
    if (wide && left >= 4) {
        Quad<T> q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q.v[j] = from_float<T>(v[j]);
        *reinterpret_cast<Quad<T> *>(p) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < left) p[j] = from_float<T>(v[j]);
    }
}
template <class T>
__device__ __forceinline__ bool quads_at(const T *p, int64_t pitch) {
    return (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(T) - 1)) == 0 && pitch % 4 == 0;
}

template <class T>
struct DenseEpilogue {
    static constexpr bool kWholeTiles = false;
    using Slope = typename std::conditional<sizeof(T) == 4, float, __half>::type;
    DenseOutput o;

    struct Place {
        int row, col, m, n;   // of the lane's first value; lane = row, where neighbouring rows are neighbours in memory
        int whole;            // columns that the warp's pieces may reach over and be whole, on addresses that allow wide accesses
        int64_t at;
        bool wide, bias_wide, residual_wide;
    };
    // Neighbouring columns of the product are neighbours in memory, or neighbouring rows are.
    __device__ __forceinline__ bool by_rows() const { return o.rows_are_features == o.feature_major; }

    __device__ __forceinline__ Place begin(const Tile &, const MatmulShape &s, int row, int col, int lane) const {
        Place p;
        p.m = s.m;
        p.n = s.n;
        if (by_rows()) {
            p.row = row + lane / 4;
            p.col = col + lane % 4 * 4;
            p.at = (int64_t)p.row * o.y_pitch + p.col;
        } else {
            p.row = row + lane;
            p.col = col;
            p.at = (int64_t)p.col * o.y_pitch + p.row;
        }
        const T *y = reinterpret_cast<const T *>(o.y), *r = reinterpret_cast<const T *>(o.residual);
        p.wide = quads_at(y, o.y_pitch);
        p.bias_wide = quads_at(reinterpret_cast<const T *>(o.bias), 0);
        p.residual_wide = o.residual_col == 1 && quads_at(r, o.residual_row);
        const bool fast = by_rows() && p.wide && row + 32 <= s.m && (o.bias == nullptr || o.rows_are_features || p.bias_wide) &&
                          (o.residual == nullptr || p.residual_wide);
        p.whole = fast ? s.n - col : 0;
        return p;
    }

    template <bool SLOPE>
    __device__ __forceinline__ void whole_piece(const Place &p, int across, float (&q)[4][4]) const {
        const T *bias = reinterpret_cast<const T *>(o.bias), *residual = reinterpret_cast<const T *>(o.residual);
        float z[16], d[16];
        Quad<T> more[4];
        if (residual != nullptr) {
            const T *from = residual + p.row * o.residual_row + p.col + across;
#pragma unroll
            for (int i = 0; i < 4; ++i) more[i] = *reinterpret_cast<const Quad<T> *>(from + 8 * i * o.residual_row);
        }
        float b[4][4] = {};
        if (bias != nullptr) {
            if (o.rows_are_features) {
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i][0] = b[i][1] = b[i][2] = b[i][3] = to_float(bias[p.row + 8 * i]);
            } else {
                const Quad<T> c = *reinterpret_cast<const Quad<T> *>(bias + p.col + across);
#pragma unroll
                for (int i = 0; i < 16; ++i) b[i / 4][i % 4] = to_float(c.v[i % 4]);
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = q[i / 4][i % 4] + b[i / 4][i % 4];
        activate<SLOPE>(z, d, o.act);
        if (residual != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] += to_float(more[i / 4].v[i % 4]);
        }
        const int64_t step = 8 * o.y_pitch;
        T *y = reinterpret_cast<T *>(o.y) + p.at + across;
        Slope *slope = reinterpret_cast<Slope *>(o.slope) + p.at + across;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Quad<T> v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v.v[j] = from_float<T>(z[4 * i + j]);
            *reinterpret_cast<Quad<T> *>(y + i * step) = v;
            if (SLOPE) {
                Quad<Slope> u;
#pragma unroll
                for (int j = 0; j < 4; ++j) u.v[j] = from_float<Slope>(d[4 * i + j] * (sizeof(T) == 4 ? 1.f : kSlopeScale));
                *reinterpret_cast<Quad<Slope> *>(slope + i * step) = u;
            }
        }
    }

    __device__ __forceinline__ void piece(const Place &p, int across, const float (&v)[kPieceColumns], float *stage, int lane) const {
        const T *bias = reinterpret_cast<const T *>(o.bias), *residual = reinterpret_cast<const T *>(o.residual);
        T *y = reinterpret_cast<T *>(o.y);
        Slope *slope = reinterpret_cast<Slope *>(o.slope);
        constexpr float kScale = sizeof(T) == 4 ? 1.f : kSlopeScale;
        const int col = p.col + across;
        if (!by_rows()) {
            if (p.row >= p.m) return;
            const float row_bias = bias != nullptr && o.rows_are_features ? to_float(bias[p.row]) : 0.f;
            const int left = p.n - col;
            float z[kPieceColumns], d[kPieceColumns];
#pragma unroll
            for (int j = 0; j < kPieceColumns; ++j)
                z[j] = v[j] + (bias != nullptr && !o.rows_are_features && j < left ? to_float(bias[col + j]) : row_bias);
            activate<true>(z, d, o.act);
            if (residual != nullptr) {
                const T *from = residual + p.row * o.residual_row + col * o.residual_col;
#pragma unroll
                for (int j = 0; j < kPieceColumns; ++j)
                    if (j < left) z[j] += to_float(from[j * o.residual_col]);
            }
            const int64_t at = p.at + across * o.y_pitch;
#pragma unroll
            for (int j = 0; j < kPieceColumns; ++j) {
                if (j >= left) continue;
                y[at + j * o.y_pitch] = from_float<T>(z[j]);
                if (slope != nullptr) slope[at + j * o.y_pitch] = from_float<Slope>(d[j] * kScale);
            }
            return;
        }
        piece_store(stage, lane, v);
        float q[4][4];
        piece_quads(stage, lane, q);
        __syncwarp();
        if (across + kPieceColumns <= p.whole) {
            if (slope != nullptr) whole_piece<true>(p, across, q);
            else whole_piece<false>(p, across, q);
            return;
        }
        const int left = p.n - col;
        if (left <= 0) return;
        // a piece over the edge, or on addresses that allow single values only
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = p.row + 8 * i;
            if (row >= p.m) continue;
            float d[4], b[4] = {0.f, 0.f, 0.f, 0.f};
            if (bias != nullptr) {
                if (o.rows_are_features) b[0] = b[1] = b[2] = b[3] = to_float(bias[row]);
                else read_quad(bias + col, p.bias_wide, left, b);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) q[i][j] += b[j];
            activate<true>(q[i], d, o.act);
            if (residual != nullptr) {
                const T *from = residual + row * o.residual_row + col * o.residual_col;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < left) q[i][j] += to_float(from[j * o.residual_col]);
            }
            const int64_t at = p.at + across + 8 * i * o.y_pitch;
            write_quad(y + at, p.wide, left, q[i]);
            if (slope != nullptr) {
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] *= kScale;
                write_quad(slope + at, p.wide, left, d);
            }
        }
    }
};

// Gradients: the sums as they are, in the layer's type.
template <class T>
struct PlainEpilogue {
    static constexpr bool kWholeTiles = false;
    T *out;
    int64_t pitch;
    struct Place {
        int row, col, m, n, whole;   // as DenseEpilogue's
        T *at;
        bool wide;
    };
    __device__ __forceinline__ Place begin(const Tile &, const MatmulShape &s, int row, int col, int lane) const {
        const int r = row + lane / 4, c = col + lane % 4 * 4;
        const bool wide = quads_at(out, pitch);
        return {r, c, s.m, s.n, wide && row + 32 <= s.m ? s.n - col : 0, out + r * pitch + c, wide};
    }
    __device__ __forceinline__ void piece(const Place &p, int across, const float (&v)[kPieceColumns], float *stage, int lane) const {
        piece_store(stage, lane, v);
        float q[4][4];
        piece_quads(stage, lane, q);
        __syncwarp();
        T *to = p.at + across;
        const int64_t step = 8 * pitch;
        if (across + kPieceColumns <= p.whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                Quad<T> u;
#pragma unroll
                for (int j = 0; j < 4; ++j) u.v[j] = from_float<T>(q[i][j]);
                *reinterpret_cast<Quad<T> *>(to + i * step) = u;
            }
            return;
        }
        const int left = p.n - p.col - across;
        if (left <= 0) return;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p.row + 8 * i < p.m) write_quad(to + i * step, p.wide, left, q[i]);
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
// its rows) over a strip of rows.  A block takes 128 columns (32 lanes of 4) and a strip; 8 row groups.
__global__ void __launch_bounds__(kThreads)
pre_gradient_kernel(const void *__restrict__ gy, const void *__restrict__ slope, int64_t rows, int64_t cols, int type,
                    uint16_t *__restrict__ dst, int64_t dst_pitch, int64_t plane, int64_t strip, float *__restrict__ partial, int sum_rows) {
    __shared__ float s_sum[kThreads / 32][128];
    grid_dependency_wait();
    grid_dependents_launch();
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const int64_t col = (int64_t)blockIdx.x * 128 + lane * 4, first = (int64_t)blockIdx.y * strip, last = first + strip < rows ? first + strip : rows;
    const int valid = (int)(cols - col < 4 ? cols - col : 4);
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t row = first + group; row < last; row += kThreads / 32) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (valid > 0) {
            load4(gy, row * cols + col, type, valid, v);
            if (slope != nullptr) {
                float d[4];
                load4(slope, row * cols + col, type == kFloat32 ? kFloat32 : kFloat16, valid, d);
                const float scale = type == kFloat32 ? 1.f : 1.f / kSlopeScale;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] *= d[j] * scale;
            }
            if (dst != nullptr) {
                const int64_t to = row * dst_pitch + col;
                uint16_t p[3][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (type == kFloat32) split_triple(v[j], p[0][j], p[1][j], p[2][j]);
                    else p[0][j] = to_16bit(v[j], type);
                }
                *reinterpret_cast<ushort4 *>(dst + to) = make_ushort4(p[0][0], p[0][1], p[0][2], p[0][3]);
                if (type == kFloat32) {
                    *reinterpret_cast<ushort4 *>(dst + plane + to) = make_ushort4(p[1][0], p[1][1], p[1][2], p[1][3]);
                    *reinterpret_cast<ushort4 *>(dst + 2 * plane + to) = make_ushort4(p[2][0], p[2][1], p[2][2], p[2][3]);
                }
            }
        }
        if (partial != nullptr && sum_rows) {   // the features are rows: this row's share of 128 samples
            float r = v[0] + v[1] + v[2] + v[3];
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) r += __shfl_xor_sync(0xffffffffu, r, off);
            if (lane == 0) partial[(int64_t)blockIdx.x * rows + row] = r;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) total[j] += v[j];
    }
    if (partial == nullptr || sum_rows) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) s_sum[group][lane * 4 + j] = total[j];
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (threadIdx.x < 128 && c < cols) {
        float r = 0.f;
#pragma unroll
        for (int g = 0; g < kThreads / 32; ++g) r += s_sum[g][threadIdx.x];
        partial[blockIdx.y * cols + c] = r;
    }
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

// Whether the layer's outputs are the rows of the product: as they lie in the result, so that neighbouring columns are stored by
// neighbouring lanes; but few samples fill half of a tile's 64 columns rather than half of its 128 rows.
static bool features_as_rows(int64_t batch, bool feature_major) { return feature_major || batch <= 64; }

static MatmulPlan plan_forward(int64_t batch, int64_t inner, int64_t outer, bool feature_major, int planes, int sms) {
    return features_as_rows(batch, feature_major) ? plan_matmul(outer, batch, inner, 1, planes, false, sms)
                                                  : plan_matmul(batch, outer, inner, 1, planes, false, sms);
}

// Strips of rows of a pre-activation gradient, enough for whole SMs.
static int64_t strips_of(int64_t rows, int64_t cols, int sms, int64_t *strip) {
    int64_t strips = ceil_div(4 * sms, ceil_div(cols, 128));
    if (strips > ceil_div(rows, 8)) strips = ceil_div(rows, 8);
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
    sizes[0] = sizes[1] = sizes[2] = 0;
    if (batch <= 0 || inner <= 0 || outer <= 0 || dense_rows_applicable(batch, type)) return;
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    sizes[0] = l.x_bytes;
    sizes[1] = l.w_bytes;
    sizes[2] = plan_forward(batch, inner, outer, y_feature_major != 0, l.planes, current_sms()).partial_bytes;
}

extern "C" DL_API int dl_dense_forward(const void *x, int64_t x_pitch, int x_feature_major, const void *w, const void *bias, const void *residual,
                                       int64_t residual_batch, int64_t residual_feature, int act, void *y, int y_feature_major, void *slope,
                                       void *x_planes, void *w_planes, void *workspace, int64_t batch, int64_t inner, int64_t outer, int type,
                                       void *stream) {
    const char *what = "dl_dense_forward";
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
    const MatmulPlan plan = plan_forward(batch, inner, outer, y_feature_major != 0, l.planes, sms);
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
    if (type == kFloat32) return launch_product<3>(p, plan, DenseEpilogue<float>{o}, partial, sms, st, what);
    if (type == kBFloat16) return launch_product<1>(p, plan, DenseEpilogue<__nv_bfloat16>{o}, partial, sms, st, what);
    return launch_product<1>(p, plan, DenseEpilogue<__half>{o}, partial, sms, st, what);
}

namespace dl {

static int launch_gradient(const Product &p, const MatmulPlan &plan, void *out, int64_t pitch, int type, float *partial, int sms, cudaStream_t st,
                           const char *what) {
    if (type == kFloat32) return launch_product<3>(p, plan, PlainEpilogue<float>{reinterpret_cast<float *>(out), pitch}, partial, sms, st, what);
    if (type == kBFloat16)
        return launch_product<1>(p, plan, PlainEpilogue<__nv_bfloat16>{reinterpret_cast<__nv_bfloat16 *>(out), pitch}, partial, sms, st, what);
    return launch_product<1>(p, plan, PlainEpilogue<__half>{reinterpret_cast<__half *>(out), pitch}, partial, sms, st, what);
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
                                   const void *gy, bool lay_x, bool lay_w, int sms) {
    DenseBackward b = {};
    b.planes = type == kFloat32 ? 3 : 1;
    b.g_rows = g_feature_major ? outer : batch;
    b.g_cols = g_feature_major ? batch : outer;
    b.lay_gz = act || !in_place(gy, b.g_cols, type);
    b.g_pitch = padded(b.g_cols);
    b.g_plane = b.g_rows * b.g_pitch;
    b.g_bytes = b.lay_gz ? padded_bytes(b.planes * b.g_plane * 2) : 0;
    b.strips = strips_of(b.g_rows, b.g_cols, sms, &b.strip);
    b.parts = g_feature_major ? ceil_div(b.g_cols, 128) : b.strips;
    b.bias_bytes = padded_bytes(b.parts * outer * 4);
    b.to_x = plan_matmul(batch, inner, outer, 1, b.planes, false, sms);
    b.to_w = plan_matmul(outer, inner, batch, 1, b.planes, false, sms);
    b.partial_bytes = padded_bytes(b.to_x.partial_bytes > b.to_w.partial_bytes ? b.to_x.partial_bytes : b.to_w.partial_bytes);
    b.x_bytes = lay_x ? l.x_bytes : 0;
    b.w_bytes = lay_w ? l.w_bytes : 0;
    return b;
}

}  // namespace dl

extern "C" DL_API int64_t dl_dense_backward_workspace_bytes(const void *gy, int g_feature_major, int has_slope, const void *x, int64_t x_pitch,
                                                            int x_feature_major, const void *w, int lay_x, int lay_w, int64_t batch, int64_t inner,
                                                            int64_t outer, int type) {
    if (batch <= 0 || inner <= 0 || outer <= 0) return 0;
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    return plan_backward(l, batch, inner, outer, g_feature_major != 0, type, has_slope != 0, gy, lay_x != 0, lay_w != 0, current_sms()).total();
}

extern "C" DL_API int dl_dense_backward(const void *gy, int g_feature_major, const void *slope, const void *x, int64_t x_pitch, int x_feature_major,
                                        const void *w, const void *x_planes, const void *w_planes, void *gx, void *gw, void *gb, void *workspace,
                                        int64_t batch, int64_t inner, int64_t outer, int type, void *stream) {
    const char *what = "dl_dense_backward";
    int status;
    if (!dense_sizes(batch, inner, outer, type, what, &status)) return status;
    DL_REQUIRE(batch > 0, DL_ERR_INVALID_ARG, "%s: empty batch", what);
    DL_REQUIRE(gy && (x || !gw || x_planes) && (w || !gx || w_planes), DL_ERR_INVALID_ARG, "%s: null pointer", what);
    DL_REQUIRE(workspace && aligned_to(workspace, 16), DL_ERR_INVALID_ARG, "%s: the workspace is missing or not 16-byte aligned", what);
    const int sms = current_sms();
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    const bool lay_x = gw && l.lay_x && !x_planes, lay_w = gx && l.lay_w && !w_planes;
    const DenseBackward b = plan_backward(l, batch, inner, outer, g_feature_major != 0, type, slope != nullptr, gy, lay_x, lay_w, sms);
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
        launch_dependent(true, pre_gradient_kernel, dim3((unsigned)ceil_div(b.g_cols, 128), (unsigned)b.strips), dim3(kThreads), 0, st, gy, slope,
                         b.g_rows, b.g_cols, type, b.lay_gz ? gz : (uint16_t *)nullptr, b.g_pitch, b.g_plane, b.strip, gb ? sums : (float *)nullptr,
                         g_feature_major);
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

