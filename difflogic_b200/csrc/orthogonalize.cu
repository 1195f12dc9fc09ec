// Newton-Schulz steps on matrices by the matrix products of matmul.cuh, the Muon step made of them, and their entry points.
#include <math.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "gram_steps.h"
#include "matmul_launch.cuh"

namespace dl {

int orthogonalize_async_error() { return matmul_error_flag(); }

// What is orthogonalised: `count` matrices behind each other at entry 0, or one at every entry; with momenta the update of a step,
// made of gradients and momenta as they are read.
struct Matrices {
    static constexpr int kMost = 16;
    const void *g[kMost];
    float *momentum[kMost];   // null: g as it is
    float *weight[kMost];
    int64_t stride;           // values from one matrix to the next at entry 0
    int type;
    float keep, nesterov;     // 1 - momentum; the momentum, or 1: the update is the momentum itself
};

// Sums of squares of a matrix, one per block, in 64 bits: fp32 values of any size fit.  Momenta are moved on.
__global__ void __launch_bounds__(kThreads)
square_sums_kernel(const Matrices all, int64_t count, double *__restrict__ partial) {
    __shared__ double s_part[kThreads / 32];
    grid_dependency_wait();
    grid_dependents_launch();
    const int64_t z = blockIdx.y, base = all.stride * z, quads = (count + 3) / 4;
    const int entry = all.stride ? 0 : (int)z;
    const void *g = all.g[entry];
    float *momentum = all.momentum[entry];
    double sum = 0;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < quads; i += (int64_t)gridDim.x * kThreads) {
        const int valid = (int)(count - i * 4 < 4 ? count - i * 4 : 4);
        float v[4];
        load4(g, base + i * 4, all.type, valid, v);
        if (momentum != nullptr) {
            float m[4];
            load4(momentum, base + i * 4, kFloat32, valid, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                m[j] = new_momentum(m[j], v[j], all.keep);
                v[j] = update_of(m[j], v[j], all.nesterov);
            }
            store4(momentum, base + i * 4, kFloat32, valid, m);
        }
        sum += ((double)v[0] * v[0] + (double)v[1] * v[1]) + ((double)v[2] * v[2] + (double)v[3] * v[3]);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (threadIdx.x % 32 == 0) s_part[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kThreads / 32; ++i) sum += s_part[i];
        partial[z * gridDim.x + blockIdx.x] = sum;
    }
}

// X = G / max(|G|, eps) as pairs.  Norms whose inverse times 2^12 is no ordinary fp32 number take two factors, the first a power of two.
__global__ void __launch_bounds__(kThreads)
normalise_kernel(const Matrices all, int64_t rows, int64_t cols, const double *__restrict__ partial, int parts, double eps,
                 uint16_t *__restrict__ x, int64_t pitch, int64_t plane) {
    __shared__ float s_first, s_scale;
    grid_dependency_wait();
    grid_dependents_launch();
    const int64_t z = blockIdx.y, base = all.stride * z;
    const int entry = all.stride ? 0 : (int)z;
    const void *g = all.g[entry];
    const float *momentum = all.momentum[entry];
    if (threadIdx.x < 32) {
        double sum = 0;
        for (int i = threadIdx.x; i < parts; i += 32) sum += partial[z * parts + i];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const double norm = sqrt(sum), by = norm > eps ? norm : eps;
        if (threadIdx.x == 0) {
            s_first = by < 0x1p-64 ? 0x1p100f : by > 0x1p100 ? 0x1p-60f : 1.f;
            // a norm that is not finite (an infinite or undefined entry) makes the whole result undefined
            s_scale = norm <= 1.7e308 ? (float)((double)kPairScale / (by * s_first)) : __int_as_float(0x7fc00000);
        }
    }
    __syncthreads();
    const float first = s_first, scale = s_scale;
    const int64_t quads = (cols + 3) / 4, total = rows * quads;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t row = i / quads, col = (i - row * quads) * 4, at = base + row * cols + col;
        const int valid = (int)(cols - col < 4 ? cols - col : 4);
        float v[4];
        load4(g, at, all.type, valid, v);
        if (momentum != nullptr) {
            float m[4];
            load4(momentum, at, kFloat32, valid, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = update_of(m[j], v[j], all.nesterov);
        }
        uint2 hi, lo;
        split_two(v[0] * first * scale, v[1] * first * scale, hi.x, lo.x);
        split_two(v[2] * first * scale, v[3] * first * scale, hi.y, lo.y);
        uint16_t *to = x + 2 * z * plane + row * pitch + col;
        *reinterpret_cast<uint2 *>(to) = hi;
        *reinterpret_cast<uint2 *>(to + plane) = lo;
    }
}

// Results of the iteration as pairs: v = scale * sum (+ factor * the pair in `more`) (+ diagonal on the diagonal).  Of a symmetric result
// the blocks of 128 x 128 below the diagonal are stored on both sides, those above it not looked at.
struct PairEpilogue {
    static constexpr bool kWholeTiles = false;
    static constexpr int kColumns = 32;
    uint16_t *out;
    const uint16_t *more;      // null: none
    int64_t pitch, plane;      // of both; rows are padded to whole units, whose last values are written too and read by nothing
    float scale, factor, diagonal;
    bool symmetric;
    struct Place {
        int row, col, m, n;    // of the warp's first value
        int64_t matrix;
    };
    __device__ __forceinline__ Place begin(const Tile &t, const MatmulShape &s, int row, int col, int) const {
        return {row, col, s.m, s.n, 2 * t.matrix * plane};
    }
    // The slots' rows -- high and low halves -- to rows row .. of the result, columns col .., of which those below `rows`, `cols` are there.
    __device__ __forceinline__ void store(uint8_t *stage, int lane, const Place &p, int row, int col, int rows, int cols) const {
        const int r = row + lane / 4, c = col + lane % 4 * 8;
        uint16_t *to = out + p.matrix + r * pitch + c;
        uint4 hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = *slot_unit(stage, lane, i);
            lo[i] = *slot_unit(stage + kSlotBytes, lane, i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r + 8 * i >= rows || c >= cols) continue;
            *reinterpret_cast<uint4 *>(to + 8 * i * pitch) = hi[i];
            *reinterpret_cast<uint4 *>(to + 8 * i * pitch + plane) = lo[i];
        }
        __syncwarp();
    }
    struct Ahead {
        uint4 hi[4], lo[4];   // of `more`, as slot_unit's
    };
    __device__ __forceinline__ void fetch(const Place &p, int across, int lane, Ahead &a) const {
        if (more == nullptr) return;
        const int r = p.row + lane / 4, c = p.col + across + lane % 4 * 8;
        const uint16_t *from = more + p.matrix + r * pitch + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool there = r + 8 * i < p.m && c < p.n;
            a.hi[i] = there ? *reinterpret_cast<const uint4 *>(from + 8 * i * pitch) : make_uint4(0, 0, 0, 0);
            a.lo[i] = there ? *reinterpret_cast<const uint4 *>(from + 8 * i * pitch + plane) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void piece(const Place &p, int across, const float (&v)[kColumns], const Ahead &a, uint8_t *stage, int lane) const {
        const int col = p.col + across, below = p.row / kMatmulRows - col / kMatmulRows, row = p.row + lane;
        if (p.row >= p.m || (symmetric && below < 0)) return;
        uint32_t hi[16], lo[16];
        float w[kColumns];
#pragma unroll
        for (int j = 0; j < kColumns; ++j) w[j] = v[j] * scale;
        if (more != nullptr) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                *slot_unit(stage, lane, i) = a.hi[i];
                *slot_unit(stage + kSlotBytes, lane, i) = a.lo[i];
            }
            __syncwarp();
            uint4 h[4], l[4];
            slot_read_row(stage, lane, h);
            slot_read_row(stage + kSlotBytes, lane, l);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint32_t x[4] = {h[j / 4].x, h[j / 4].y, h[j / 4].z, h[j / 4].w}, y[4] = {l[j / 4].x, l[j / 4].y, l[j / 4].z, l[j / 4].w};
                const float2 up = __half22float2(*reinterpret_cast<const __half2 *>(&x[j % 4])), down = __half22float2(*reinterpret_cast<const __half2 *>(&y[j % 4]));
                w[2 * j] += factor * (up.x + down.x);
                w[2 * j + 1] += factor * (up.y + down.y);
            }
        }
        if (diagonal != 0.f && p.row < col + kColumns && col < p.row + 32) {
#pragma unroll
            for (int j = 0; j < kColumns; ++j)
                if (row == col + j) w[j] += diagonal;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) split_two(w[2 * j], w[2 * j + 1], hi[j], lo[j]);
        slot_row(stage, lane, hi);
        slot_row(stage + kSlotBytes, lane, lo);
        __syncwarp();
        store(stage, lane, p, p.row, col, p.m, p.n);
        if (symmetric && below > 0) {   // columns as rows
#pragma unroll
            for (int j = 0; j < kColumns; ++j) {
                slot_column(stage, lane, j, (uint16_t)(hi[j / 2] >> (j % 2 * 16)));
                slot_column(stage + kSlotBytes, lane, j, (uint16_t)(lo[j / 2] >> (j % 2 * 16)));
            }
            __syncwarp();
            store(stage, lane, p, col, p.row, p.n, p.m);
        }
    }
};

// The last product: the result itself, or the weights' update w <- decay w - rate v.
struct OrthogonalEpilogue {
    static constexpr bool kWholeTiles = false;
    static constexpr int kColumns = kPieceColumns;
    void *out;              // results behind each other; null: the weights of `all` are updated
    Matrices all;
    int64_t cols;           // values of a row
    const uint16_t *more;   // added, as in PairEpilogue
    int64_t pitch, plane;
    float scale, factor;
    float decay, rate;
    struct Place {
        int row, col, m, n;   // of the lane's first value
        int64_t at, matrix;
        float *weight;
    };
    __device__ __forceinline__ Place begin(const Tile &t, const MatmulShape &s, int row, int col, int lane) const {
        const int r = row + lane / 4, c = col + lane % 4 * 4;
        const int64_t at = r * cols + c;
        return {r, c, s.m, s.n, out == nullptr ? at : at + (int64_t)t.matrix * s.m * cols, 2 * t.matrix * plane, out == nullptr ? all.weight[t.matrix] : nullptr};
    }
    struct Ahead {
        ushort4 hi[4], lo[4];   // of `more`
        float w[4][4];          // of the weights
    };
    __device__ __forceinline__ void fetch(const Place &p, int across, int, Ahead &a) const {
        const int left = p.n - p.col - across;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p.row + 8 * i >= p.m || left <= 0) continue;
            if (p.weight != nullptr) load4(p.weight, p.at + across + 8 * i * cols, kFloat32, left < 4 ? left : 4, a.w[i]);
            if (more != nullptr) {
                const uint16_t *from = more + p.matrix + (p.row + 8 * i) * pitch + p.col + across;
                a.hi[i] = *reinterpret_cast<const ushort4 *>(from);
                a.lo[i] = *reinterpret_cast<const ushort4 *>(from + plane);
            }
        }
    }
    __device__ __forceinline__ void piece(const Place &p, int across, const float (&v)[kColumns], const Ahead &a, uint8_t *stage, int lane) const {
        float q[4][4];
        piece_quads(stage, lane, v, q);
        const int left = p.n - p.col - across;
        if (left <= 0) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p.row + 8 * i >= p.m) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) q[i][j] *= scale;
            if (more != nullptr) {
                const ushort4 hi = a.hi[i], lo = a.lo[i];
                q[i][0] += factor * join_pair(hi.x, lo.x);
                q[i][1] += factor * join_pair(hi.y, lo.y);
                q[i][2] += factor * join_pair(hi.z, lo.z);
                q[i][3] += factor * join_pair(hi.w, lo.w);
            }
            if (p.weight != nullptr) {
#pragma unroll
                for (int j = 0; j < 4; ++j) q[i][j] = a.w[i][j] * decay - rate * q[i][j];
                store4(p.weight, p.at + across + 8 * i * cols, kFloat32, left < 4 ? left : 4, q[i]);
            } else {
                store4(out, p.at + across + 8 * i * cols, all.type, left < 4 ? left : 4, q[i]);
            }
        }
    }
};

// The iterations multiply one plane or two.
template <class Epilogue>
static int launch_planes(const Product &p, const MatmulPlan &plan, const Epilogue &e, float *partial, int sms, cudaStream_t st, const char *what) {
    return p.planes == 1 ? launch_product<1>(p, plan, e, partial, sms, st, what) : launch_product<2>(p, plan, e, partial, sms, st, what);
}

struct OrthogonalLayout {
    int64_t side, x_pitch, x_plane, s_pitch, s_plane;   // side: the smaller one
    bool tall;
    int parts;
    MatmulPlan gram, square, product;
    int64_t x_bytes, s_bytes, norm_bytes, partial_bytes;
    int64_t total() const { return 2 * x_bytes + 2 * s_bytes + norm_bytes + partial_bytes; }
};

static OrthogonalLayout orthogonal_layout(int64_t batch, int64_t rows, int64_t cols, bool light, int sms, int choice) {
    OrthogonalLayout l = {};
    l.tall = rows >= cols;
    l.side = l.tall ? cols : rows;
    l.x_pitch = padded(cols);
    l.x_plane = rows * l.x_pitch;
    l.s_pitch = padded(l.side);
    l.s_plane = l.side * l.s_pitch;
    l.parts = (int)(ceil_div(rows * cols, 4 * kThreads * 4) < 2 * sms ? ceil_div(rows * cols, 4 * kThreads * 4) : 2 * sms);
    l.gram = plan_matmul(l.side, l.side, l.tall ? rows : cols, batch, light ? 1 : 2, true, sms, choice);
    l.square = plan_matmul(l.side, l.side, l.side, batch, 2, true, sms, choice);
    l.product = plan_matmul(rows, cols, l.side, batch, light ? 1 : 2, false, sms, choice);
    l.x_bytes = padded_bytes(batch * 2 * l.x_plane * 2);
    l.s_bytes = padded_bytes(batch * 2 * l.s_plane * 2);
    l.norm_bytes = padded_bytes(batch * l.parts * 8);
    l.partial_bytes = l.gram.partial_bytes;
    if (l.square.partial_bytes > l.partial_bytes) l.partial_bytes = l.square.partial_bytes;
    if (l.product.partial_bytes > l.partial_bytes) l.partial_bytes = l.product.partial_bytes;
    return l;
}

// How far a step's polynomials go.  Singular values of X start in [0, 1]; a step takes those of [0, reach] to |a s + b s^3 + c s^5|, which
// as a continuous image of an interval with 0 in it is the interval up to the largest one: at the end or where the derivative is zero.
static double largest_value(double a, double b, double c, double reach) {
    double most = fabs(reach * (a + reach * reach * (b + reach * reach * c)));
    const double root = 9 * b * b - 20 * a * c;
    if (root >= 0) {   // the roots of a + 3 b u + 5 c u^2, u = s^2, without a difference of near equals where c is small
        const double q = -(3 * b + copysign(sqrt(root), b)) / 2;
        for (const double u : {q / (5 * c), a / q})
            if (u > 0 && u < reach * reach) most = std::max(most, fabs(sqrt(u) * (a + u * (b + u * c))));
    }
    return most;
}
// The largest of |a + b u + c u^2| over the same values, u = s^2: the norm of M.
static double largest_factor(double a, double b, double c, double reach) {
    const double end = reach * reach, u = c != 0 ? -b / (2 * c) : 0;
    double most = std::max(fabs(a), fabs(a + end * (b + end * c)));
    if (u > 0 && u < end) most = std::max(most, fabs(a + u * (b + u * c)));
    return most;
}
constexpr double kMostReach = 8.01;   // X itself is kept times 2^12: fp16 ends at 16 of that
// Pairs of a matrix of this norm are kept as many times smaller, a power of two, so that its entries, no larger than the norm, stay below 16
// with some room for what is rounded on the way.  1 for coefficients that keep values near 1.
static float kept_smaller(double norm) {
    float by = 1.f;
    while (norm / by > 12) by *= 2;
    return by;
}

// steps times: S = X^T X (X X^T where X is wide), M = b S + c S^2, X = a X + X M (M X).  `last` takes the last product.
// b S is added up in the epilogue of c S^2, which reads S beside its products; S stored a second time with b / c on its diagonal, so that
// one product gave both, costs more in stores than it saves: 4 x 1024 x 1024 bf16 347 us for 304.
//
// Results of 22 bits (fp32, fp16): every product is one of pairs, and a X comes out of the product too, as the diagonal of M, since
// the pair of a X would have to be read again.  bf16 results have 8 bits, and the steps need no more than this: S from the first planes
// alone, which leaves the result 6e-4 off (relative, over random, low-rank and steeply falling spectra; rounding it to bf16 is
// 1.7e-3); S^2 from pairs; X M from the first planes, a X added as the pair that it is.  That last form matters: what is rounded away
// of X in a product with a I + b S + c S^2 grows by a factor of a in every step along directions of small singular values, 4e-2 in the
// end where X has few large ones; M alone is next to nothing along those.  All together 1.6e-3, half the products.
static int orthogonalise(const Matrices &all, int64_t batch, int64_t rows, int64_t cols, int steps, const float *coefficients, double eps,
                         const OrthogonalEpilogue &last, uint8_t *workspace, int sms, int choice, cudaStream_t st, const char *what) {
    const bool light = all.type == kBFloat16;
    const OrthogonalLayout l = orthogonal_layout(batch, rows, cols, light, sms, choice);
    uint8_t *at = workspace;
    const auto take = [&](int64_t bytes) {
        uint8_t *p = at;
        at += bytes;
        return p;
    };
    uint16_t *x = reinterpret_cast<uint16_t *>(take(l.x_bytes)), *next = reinterpret_cast<uint16_t *>(take(l.x_bytes));
    uint16_t *gram = reinterpret_cast<uint16_t *>(take(l.s_bytes)), *poly = reinterpret_cast<uint16_t *>(take(l.s_bytes));
    double *norms = reinterpret_cast<double *>(take(l.norm_bytes));
    float *partial = reinterpret_cast<float *>(at);
    int status;
    launch_dependent(true, square_sums_kernel, dim3((unsigned)l.parts, (unsigned)batch), dim3(kThreads), 0, st, all, rows * cols, norms);
    if ((status = launch_status(what)) != DL_OK) return status;
    int64_t blocks = ceil_div(rows * ceil_div(cols, 4), kThreads * 2);
    if (blocks > 16 * sms) blocks = 16 * sms;
    launch_dependent(true, normalise_kernel, dim3((unsigned)blocks, (unsigned)batch), dim3(kThreads), 0, st, all, rows, cols, (const double *)norms,
                     l.parts, eps, x, l.x_pitch, l.x_plane);
    if ((status = launch_status(what)) != DL_OK) return status;
    Product p = {};
    p.batch = batch;
    p.planes_z = 2;
    p.exact = !light;
    const float once = 1.f / kPairScale, twice = once * once;
    double reach = 1;
    for (int i = 0; i < steps; ++i) {
        const float a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
        const float gram_by = kept_smaller(reach * reach), poly_by = kept_smaller(largest_factor(light ? 0.f : a, b, c, reach));
        reach = largest_value(a, b, c, reach);
        p.a = p.b = {x, l.x_pitch, l.x_plane, l.tall};
        p.m = p.n = l.side;
        p.k = l.tall ? rows : cols;
        p.symmetric = true;
        p.planes = light ? 1 : 2;
        PairEpilogue e = {};
        e.pitch = l.s_pitch;
        e.plane = l.s_plane;
        e.scale = once / gram_by;
        e.symmetric = true;
        e.out = gram;
        if (c == 0.f) {   // the cubic iteration: M comes straight out of this product
            e.scale = b * once / poly_by;
            e.diagonal = light ? 0.f : a * kPairScale / poly_by;
        }
        if ((status = launch_planes(p, l.gram, e, partial, sms, st, what)) != DL_OK) return status;
        if (c != 0.f) {
            p.a = p.b = {gram, l.s_pitch, l.s_plane, false};
            p.k = l.side;
            p.planes = 2;
            e.out = poly;
            e.more = gram;
            e.factor = b * (gram_by / poly_by);
            e.scale = c * once * (gram_by * gram_by / poly_by);
            e.diagonal = light ? 0.f : a * kPairScale / poly_by;
            if ((status = launch_planes(p, l.square, e, partial, sms, st, what)) != DL_OK) return status;
        }
        const Operand m = {c != 0.f ? poly : gram, l.s_pitch, l.s_plane, false};
        p.k = l.side;
        p.a = l.tall ? Operand{x, l.x_pitch, l.x_plane, false} : m;
        p.b = l.tall ? m : Operand{x, l.x_pitch, l.x_plane, true};
        p.m = rows;
        p.n = cols;
        p.symmetric = false;
        p.planes = light ? 1 : 2;
        const uint16_t *more = light ? x : nullptr;
        if (i + 1 < steps) {
            PairEpilogue to_next = {};
            to_next.more = more;
            to_next.pitch = l.x_pitch;
            to_next.plane = l.x_plane;
            to_next.scale = once * poly_by;
            to_next.factor = a;
            to_next.out = next;
            status = launch_planes(p, l.product, to_next, partial, sms, st, what);
        } else {
            OrthogonalEpilogue to_end = last;
            to_end.all = all;
            to_end.cols = cols;
            to_end.more = more;
            to_end.pitch = l.x_pitch;
            to_end.plane = l.x_plane;
            to_end.scale = twice * poly_by;
            to_end.factor = a * once;
            status = launch_planes(p, l.product, to_end, partial, sms, st, what);
        }
        if (status != DL_OK) return status;
        uint16_t *done = x;
        x = next;
        next = done;
    }
    return DL_OK;
}

}  // namespace dl

using namespace dl;

// The smallest norm of a matrix that is not zero is 1.4e-45: any eps far below that is the same one, and the scales that it leads to, and
// their squares, are finite.
static double usable_eps(double eps) { return eps > 1e-60 ? eps : 1e-60; }

// Matrices of so few columns stay as they are: their Gram matrix is iterated instead (gram_steps.cu).
static bool few_columns(int64_t cols) { return cols <= kGramColumns; }

extern "C" DL_API int64_t dl_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int type) {
    const int choice = matmul_choice(&type);
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    if (few_columns(cols)) return gram_workspace_bytes(batch, batch * rows, current_sms());
    return orthogonal_layout(batch, rows, cols, type == kBFloat16, current_sms(), choice).total();
}

static int check_steps(int steps, const float *coefficients, double eps, const char *what) {
    DL_REQUIRE(steps >= 1 && steps <= kMostSteps && coefficients, DL_ERR_INVALID_ARG, "%s: needs 1 to %d steps and their coefficients", what, kMostSteps);
    DL_REQUIRE(eps > 0, DL_ERR_INVALID_ARG, "%s: eps must be positive", what);
    double reach = 1;
    for (int i = 0; i < steps; ++i) {
        const float *at = coefficients + 3 * i;
        for (int j = 0; j < 3; ++j) DL_REQUIRE(fabsf(at[j]) <= 64, DL_ERR_INVALID_ARG, "%s: a coefficient of more than 64", what);
        reach = largest_value(at[0], at[1], at[2], reach);
        DL_REQUIRE(reach <= kMostReach, DL_ERR_INVALID_ARG, "%s: with these coefficients singular values do not stay near 1", what);
    }
    return DL_OK;
}

extern "C" DL_API int dl_orthogonalize(const void *g, void *out, int64_t batch, int64_t rows, int64_t cols, int type, int steps,
                                       const float *coefficients, double eps, void *workspace, void *stream) {
    const char *what = "dl_orthogonalize";
    const int choice = matmul_choice(&type);
    DL_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0 && rows <= INT32_MAX / 2 && cols <= INT32_MAX / 2, DL_ERR_INVALID_ARG, "%s: bad size", what);
    DL_REQUIRE(batch <= 65535, DL_ERR_TOO_LARGE, "%s: more than 65535 matrices", what);
    DL_REQUIRE(type >= kFloat32 && type <= kFloat16, DL_ERR_INVALID_ARG, "%s: unknown type %d", what, type);
    int status = check_steps(steps, coefficients, eps, what);
    if (status != DL_OK) return status;
    if (batch == 0 || rows == 0 || cols == 0) return DL_OK;
    DL_REQUIRE(g && out && workspace, DL_ERR_INVALID_ARG, "%s: null pointer", what);
    DL_REQUIRE(aligned_to(workspace, 16), DL_ERR_INVALID_ARG, "%s: the workspace must be 16-byte aligned", what);
    if (few_columns(cols)) {
        GramJob job = {};
        job.count = 1;
        job.batch = batch;
        job.matrix[0] = {g, nullptr, out, rows, 0.f};
        job.cols = (int)cols;
        job.type = type;
        return launch_gram_steps(job, steps, coefficients, usable_eps(eps), reinterpret_cast<double *>(workspace), current_sms(), as_stream(stream), what);
    }
    Matrices all = {};
    all.g[0] = g;
    all.stride = rows * cols;
    all.type = type;
    OrthogonalEpilogue last = {};
    last.out = out;
    return orthogonalise(all, batch, rows, cols, steps, coefficients, usable_eps(eps), last, reinterpret_cast<uint8_t *>(workspace), current_sms(),
                         choice, as_stream(stream), what);
}

// One step: the matrices of few columns together, then those of one shape after the other.
namespace dl {

template <class Few, class Many>
static int over_muon_groups(const int64_t *table, int64_t count, const Few &few, const Many &many) {
    int status = DL_OK;
    for (int64_t i = 0; i < count && status == DL_OK; ++i) {   // every group at its first matrix
        const int64_t *at = table + 5 * i;
        GramJob job = {};
        if (few_columns(at[4])) {
            bool taken = false;   // by an earlier group of this number of columns
            for (int64_t j = 0; j < i; ++j) taken |= table[5 * j + 4] == at[4];
            if (!taken) {
                job.cols = (int)at[4];
                for (int64_t j = i; j < count && status == DL_OK; ++j) {
                    const int64_t *t = table + 5 * j;
                    if (t[4] != at[4] || t[3] == 0) continue;
                    job.matrix[job.count++] = {reinterpret_cast<const void *>(t[1]), reinterpret_cast<float *>(t[2]), reinterpret_cast<void *>(t[0]), t[3], 0.f};
                    if (job.count == GramJob::kMost) {
                        status = few(job);
                        job.count = 0;
                    }
                }
                if (job.count > 0 && status == DL_OK) status = few(job);
            }
        } else {
            bool taken = at[3] == 0;
            for (int64_t j = 0; j < i; ++j) taken |= table[5 * j + 3] == at[3] && table[5 * j + 4] == at[4];
            if (!taken) {
                Matrices all = {};
                int64_t batch = 0;
                for (int64_t j = i; j < count && status == DL_OK; ++j) {
                    const int64_t *t = table + 5 * j;
                    if (t[3] != at[3] || t[4] != at[4]) continue;
                    all.weight[batch] = reinterpret_cast<float *>(t[0]);
                    all.g[batch] = reinterpret_cast<const void *>(t[1]);
                    all.momentum[batch++] = reinterpret_cast<float *>(t[2]);
                    if (batch == Matrices::kMost) {
                        status = many(all, batch, at[3], at[4]);
                        batch = 0;
                    }
                }
                if (batch > 0 && status == DL_OK) status = many(all, batch, at[3], at[4]);
            }
        }
    }
    return status;
}

static int64_t rows_of(const GramJob &job) {
    int64_t rows = 0;
    for (int i = 0; i < job.count; ++i) rows += job.matrix[i].rows;
    return rows * job.batch;
}

// Whether what is written, weights and momenta, shares no memory with anything else of the table; gradients may share theirs.
static bool disjoint(const int64_t *table, int64_t count) {
    struct Range {
        int64_t first, last;
        bool written;
    };
    std::vector<Range> all;   // may throw
    all.reserve(3 * count);
    for (int64_t i = 0; i < count; ++i) {
        const int64_t *t = table + 5 * i, size = t[3] * t[4] * 4;
        if (size == 0) continue;
        for (int j = 0; j < 3; ++j) all.push_back({t[j], t[j] + size, j != 1});
    }
    std::sort(all.begin(), all.end(), [](const Range &a, const Range &b) { return a.first < b.first; });
    int64_t any = 0, written = 0;   // where what came so far ends
    for (const Range &r : all) {
        if (r.first < (r.written ? any : written)) return false;
        any = std::max(any, r.last);
        if (r.written) written = std::max(written, r.last);
    }
    return true;
}

}  // namespace dl

extern "C" DL_API int64_t dl_muon_workspace_bytes(const int64_t *table, int64_t count) {
    if (table == nullptr) return 0;
    const int sms = current_sms();
    int64_t most = 0;
    over_muon_groups(
        table, count,
        [&](GramJob &job) {
            job.batch = 1;
            const int64_t bytes = gram_workspace_bytes(job.count, rows_of(job), sms);
            if (bytes > most) most = bytes;
            return DL_OK;
        },
        [&](Matrices &, int64_t batch, int64_t rows, int64_t cols) {
            const int64_t bytes = orthogonal_layout(batch, rows, cols, false, sms, 0).total();
            if (bytes > most) most = bytes;
            return DL_OK;
        });
    return most;
}

extern "C" DL_API int dl_muon_step_f32(const int64_t *table, int64_t count, double lr, double momentum, int nesterov, double weight_decay, int steps,
                                       const float *coefficients, double eps, void *workspace, void *stream) {
    const char *what = "dl_muon_step_f32";
    DL_REQUIRE(count >= 0 && (table || count == 0), DL_ERR_INVALID_ARG, "%s: null pointer", what);
    int status = check_steps(steps, coefficients, eps, what);
    if (status != DL_OK) return status;
    for (int64_t i = 0; i < count; ++i) {
        const int64_t *t = table + 5 * i;
        DL_REQUIRE(t[3] >= 0 && t[4] > 0 && t[3] <= INT32_MAX / 2 && t[4] <= INT32_MAX / 2, DL_ERR_INVALID_ARG, "%s: bad size", what);
        DL_REQUIRE(t[3] == 0 || (t[0] && t[1] && t[2]), DL_ERR_INVALID_ARG, "%s: null pointer", what);
        DL_REQUIRE((t[0] | t[1] | t[2]) % 4 == 0, DL_ERR_INVALID_ARG, "%s: misaligned matrix", what);
    }
    if (count == 0) return DL_OK;
    try {
        DL_REQUIRE(disjoint(table, count), DL_ERR_INVALID_ARG, "%s: a weight or momentum shares memory with another matrix", what);
    } catch (const std::exception &) {
        return fail(DL_ERR_INVALID_ARG, "%s: no memory on the host for %lld matrices", what, (long long)count);
    }
    DL_REQUIRE(workspace && aligned_to(workspace, 16), DL_ERR_INVALID_ARG, "%s: the workspace is missing or not 16-byte aligned", what);
    const int sms = current_sms();
    cudaStream_t st = as_stream(stream);
    const auto rate = [&](int64_t rows, int64_t cols) { return (float)(lr * sqrt(rows > cols ? (double)rows / (double)cols : 1.0)); };
    const float keep = (float)(1.0 - momentum), toward = nesterov ? (float)momentum : 1.f, decay = (float)(1.0 - lr * weight_decay);
    return over_muon_groups(
        table, count,
        [&](GramJob &job) {
            job.batch = 1;
            job.type = kFloat32;
            job.update = true;
            job.keep = keep;
            job.nesterov = toward;
            job.decay = decay;
            for (int i = 0; i < job.count; ++i) job.matrix[i].rate = rate(job.matrix[i].rows, job.cols);
            return launch_gram_steps(job, steps, coefficients, usable_eps(eps), reinterpret_cast<double *>(workspace), sms, st, what);
        },
        [&](Matrices &all, int64_t batch, int64_t rows, int64_t cols) {
            all.type = kFloat32;
            all.keep = keep;
            all.nesterov = toward;
            OrthogonalEpilogue last = {};
            last.decay = decay;
            last.rate = rate(rows, cols);
            return orthogonalise(all, batch, rows, cols, steps, coefficients, usable_eps(eps), last, reinterpret_cast<uint8_t *>(workspace), sms, 0, st, what);
        });
}
