// Newton-Schulz steps on matrices of up to 16 columns: the gate weights of logic layers, thousands of rows of 16.
//
// A step X <- X (a I + b S + c S^2) with S = X^T X multiplies X from the right with a polynomial of S, and all of these commute:
//   X_n = X_0 P,  P = M_1 M_2 ... M_n,  M = a I + b S + c S^2,  S <- M S M.
// So the rows are read twice, once for S and once for X_0 P, and the steps themselves are products of 16 x 16.  What rounds S away
// grows by up to a^2 = 12 a step along directions of small singular values, 2e5 in five steps; S, the steps and P are held in 64 bits.
//
// First kernel: momentum and gradient of a matrix, the new momentum, and sums of S.  Second kernel: every block adds the sums up in their
// order and takes the steps for itself, while its first rows are on their way, then multiplies its rows with P.  Both on the
// 64-bit matrix instruction m8n8k4 (lane l holds A[l / 4][l % 4], B[l % 4][l / 4] and D[l / 4][2 (l % 4) .. + 1]).
#include "gram_steps.h"
#include "matmul_values.cuh"

namespace dl {

constexpr int kGramThreads = 256, kGramWarps = kGramThreads / 32;
constexpr int kGramSums = 3 * 64;        // three 8 x 8 blocks of S: even-even, even-odd and odd-odd columns
constexpr int kGramParts = 64;           // at most, of a matrix

struct GramBlocks {
    GramJob job;
    int64_t strip;                       // rows of a block, a multiple of 32
    int first[GramJob::kMost + 1];       // block of every matrix (batch: of the first one)
    double scale_eps;
    int steps;
    float coefficients[3 * kMostSteps];
};

__device__ __forceinline__ void multiply64(double (&d)[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}

struct GramPlace {
    int matrix, part, parts, sums;       // entry; strip of it, of how many; its first sum
    int64_t base, rows;                  // first value, rows
};
__device__ __forceinline__ GramPlace gram_place(const GramBlocks &g, int block) {
    GramPlace p;
    if (g.job.count == 1) {
        p.matrix = 0;
        p.parts = g.first[1];
        const int z = block / p.parts;
        p.part = block - z * p.parts;
        p.rows = g.job.matrix[0].rows;
        p.base = z * p.rows * g.job.cols;
        p.sums = z * p.parts;
    } else {
        p.matrix = 0;
        while (block >= g.first[p.matrix + 1]) ++p.matrix;
        p.parts = g.first[p.matrix + 1] - g.first[p.matrix];
        p.part = block - g.first[p.matrix];
        p.rows = g.job.matrix[p.matrix].rows;
        p.base = 0;
        p.sums = g.first[p.matrix];
    }
    return p;
}

// N neighbouring values of a row of `cols`; those behind its end are zero.
template <int N>
__device__ __forceinline__ void load_row(const void *p, int64_t row_at, int col, int cols, int type, bool there, float (&v)[N]) {
    if (there && type == kFloat32 && col + N <= cols && cols % N == 0 && (reinterpret_cast<uintptr_t>(p) & (4 * N - 1)) == 0) {
        const float *at = reinterpret_cast<const float *>(p) + row_at + col;
        if constexpr (N == 4) {
            const float4 f = *reinterpret_cast<const float4 *>(at);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            const float2 f = *reinterpret_cast<const float2 *>(at);
            v[0] = f.x; v[1] = f.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = there && col + j < cols ? load_as_float(p, row_at + col + j, type) : 0.f;
    }
}

__global__ void __launch_bounds__(kGramThreads)
gram_sums_kernel(const __grid_constant__ GramBlocks g, double *__restrict__ sums) {
    __shared__ double s_sum[kGramWarps][kGramSums];
    grid_dependency_wait();
    grid_dependents_launch();
    const GramPlace p = gram_place(g, blockIdx.x);
    const GramMatrix &m = g.job.matrix[p.matrix];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, cols = g.job.cols, type = g.job.type, col = lane / 4 * 2;
    const int64_t first = p.part * g.strip, last = first + g.strip < p.rows ? first + g.strip : p.rows;
    // lane l: row l % 4, columns 2 (l / 4) and the one after it, which makes its value both the A and the B of a block of S
    double even[2] = {0, 0}, mixed[2] = {0, 0}, odd[2] = {0, 0};
    constexpr int kAhead = 8;   // rows of four at a time
    for (int64_t row = first + warp * 4 * kAhead; row < last; row += kGramWarps * 4 * kAhead) {
        float v[kAhead][2], o[kAhead][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * 4 + lane % 4;
            load_row<2>(m.g, p.base + r * cols, col, cols, type, r < last, v[i]);
            if (m.momentum != nullptr) load_row<2>(m.momentum, p.base + r * cols, col, cols, kFloat32, r < last, o[i]);
        }
        if (m.momentum != nullptr) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int64_t r = row + i * 4 + lane % 4;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    o[i][j] = new_momentum(o[i][j], v[i][j], g.job.keep);
                    v[i][j] = update_of(o[i][j], v[i][j], g.job.nesterov);
                }
                float *to = m.momentum + p.base + r * cols + col;
                if (r < last) {
                    if (cols % 2 == 0 && col < cols && (reinterpret_cast<uintptr_t>(to) & 7) == 0) {
                        *reinterpret_cast<float2 *>(to) = make_float2(o[i][0], o[i][1]);
                    } else {
                        if (col < cols) to[0] = o[i][0];
                        if (col + 1 < cols) to[1] = o[i][1];
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const double a = v[i][0], b = v[i][1];
            multiply64(even, a, a);
            multiply64(mixed, a, b);
            multiply64(odd, b, b);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int at = lane / 4 * 8 + lane % 4 * 2 + j;
        s_sum[warp][at] = even[j];
        s_sum[warp][64 + at] = mixed[j];
        s_sum[warp][128 + at] = odd[j];
    }
    __syncthreads();
    if (threadIdx.x < kGramSums) {
        double r = 0;
#pragma unroll
        for (int w = 0; w < kGramWarps; ++w) r += s_sum[w][threadIdx.x];
        sums[(int64_t)blockIdx.x * kGramSums + threadIdx.x] = r;
    }
}

constexpr int kSquarePitch = 18;   // doubles of a row of a 16 x 16 matrix
using Square = double[kGramColumns][kSquarePitch];

// One 8 x 8 block of A B.
__device__ __forceinline__ void square_block(const Square &a, const Square &b, int block, int lane, double (&d)[2]) {
    const int down = block / 2 * 8, across = block % 2 * 8;
    d[0] = d[1] = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) multiply64(d, a[down + lane / 4][4 * k + lane % 4], b[4 * k + lane % 4][across + lane / 4]);
}

struct GramShared {
    double part[kGramWarps][kGramSums];
    Square s, m, product[2], moved;
    double scale;
};

// P of a matrix, in s.product[steps % 2], scaled to take the matrix as it is.
__device__ __forceinline__ const Square &take_steps(GramShared &s, const GramBlocks &g, const double *__restrict__ sums, int parts) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    {
        double r[kGramSums / 32] = {};
        for (int i = warp; i < parts; i += kGramWarps) {
#pragma unroll
            for (int j = 0; j < kGramSums / 64; ++j) {
                const double2 d = *reinterpret_cast<const double2 *>(sums + (int64_t)i * kGramSums + j * 64 + lane * 2);
                r[2 * j] += d.x;
                r[2 * j + 1] += d.y;
            }
        }
#pragma unroll
        for (int j = 0; j < kGramSums / 64; ++j) {
            s.part[warp][j * 64 + lane * 2] = r[2 * j];
            s.part[warp][j * 64 + lane * 2 + 1] = r[2 * j + 1];
        }
    }
    __syncthreads();
    if (threadIdx.x < kGramSums) {
        double r = 0;
#pragma unroll
        for (int w = 0; w < kGramWarps; ++w) r += s.part[w][threadIdx.x];
        const int kind = threadIdx.x / 64, i = threadIdx.x % 64 / 8, j = threadIdx.x % 8;
        if (kind == 0) s.s[2 * i][2 * j] = r;
        if (kind == 1) s.s[2 * i][2 * j + 1] = s.s[2 * j + 1][2 * i] = r;
        if (kind == 2) s.s[2 * i + 1][2 * j + 1] = r;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double trace = 0;
        for (int i = 0; i < kGramColumns; ++i) trace += s.s[i][i];
        const double norm = sqrt(trace);
        s.scale = norm > g.scale_eps || norm != norm ? 1 / norm : 1 / g.scale_eps;
    }
    __syncthreads();
    const double scale = s.scale;
    if (threadIdx.x < 256) s.s[threadIdx.x / 16][threadIdx.x % 16] *= scale * scale;
    __syncthreads();
    const int block = warp % 4, row = block / 2 * 8 + lane / 4, col = block % 2 * 8 + lane % 4 * 2;
    for (int i = 0; i < g.steps; ++i) {
        const double a = g.coefficients[3 * i], b = g.coefficients[3 * i + 1], c = g.coefficients[3 * i + 2];
        double d[2];
        if (warp < 4) {
            square_block(s.s, s.s, block, lane, d);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const double v = (row == col + j ? a : 0) + b * s.s[row][col + j] + c * d[j];
                s.m[row][col + j] = v;
                if (i == 0) s.product[1][row][col + j] = v * scale;
            }
        }
        __syncthreads();
        if (i > 0 && warp < 4) {
            square_block(s.product[i % 2], s.m, block, lane, d);
            s.product[(i + 1) % 2][row][col] = d[0];
            s.product[(i + 1) % 2][row][col + 1] = d[1];
        }
        if (i + 1 < g.steps) {
            if (warp >= 4) {
                square_block(s.s, s.m, block, lane, d);
                s.moved[row][col] = d[0];
                s.moved[row][col + 1] = d[1];
            }
            __syncthreads();
            if (warp < 4) {
                square_block(s.moved, s.m, block, lane, d);
                s.s[row][col] = d[0];
                s.s[row][col + 1] = d[1];
            }
        }
        __syncthreads();
    }
    return s.product[g.steps % 2];
}

__global__ void __launch_bounds__(kGramThreads)
gram_apply_kernel(const __grid_constant__ GramBlocks g, const double *__restrict__ sums) {
    __shared__ GramShared s;
    grid_dependency_wait();
    grid_dependents_launch();
    const GramPlace p = gram_place(g, blockIdx.x);
    const GramMatrix &m = g.job.matrix[p.matrix];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, cols = g.job.cols, type = g.job.type;
    const int64_t first = p.part * g.strip, last = first + g.strip < p.rows ? first + g.strip : p.rows;
    // a warp takes 8 rows at a time: lane l reads columns 4 (l % 4) .. + 3 of row l / 4 (which order the columns are summed in is
    // free) and has columns 2 (l % 4), + 1, + 8 and + 9 of the result
    constexpr int kAhead = 4;
    const int from = lane % 4 * 4, to = lane % 4 * 2;
    float v[kAhead][4], o[kAhead][4], w[kAhead][2][2];
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * 8 + lane / 4, at = p.base + r * cols;
            load_row<4>(m.g, at, from, cols, type, r < last, v[i]);
            if (m.momentum != nullptr) load_row<4>(m.momentum, at, from, cols, kFloat32, r < last, o[i]);
            if (g.job.update) {
                load_row<2>(m.out, at, to, cols, kFloat32, r < last, w[i][0]);
                load_row<2>(m.out, at, to + 8, cols, kFloat32, r < last, w[i][1]);
            }
        }
    };
    int64_t row = first + warp * 8 * kAhead;
    fetch(row);
    const Square &product = take_steps(s, g, sums + (int64_t)p.sums * kGramSums, p.parts);
    double factor[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) factor[h][k] = product[from + k][8 * h + lane / 4];
    for (; row < last; row += kGramWarps * 8 * kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * 8 + lane / 4, at = p.base + r * cols;
            double d[2][2] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double x = m.momentum != nullptr ? update_of(o[i][k], v[i][k], g.job.nesterov) : v[i][k];
                multiply64(d[0], x, factor[0][k]);
                multiply64(d[1], x, factor[1][k]);
            }
            if (r >= last) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float out[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) out[j] = g.job.update ? w[i][h][j] * g.job.decay - m.rate * (float)d[h][j] : (float)d[h][j];
                const int col = to + 8 * h;
                if (type == kFloat32) {
                    float *at_out = reinterpret_cast<float *>(m.out) + at + col;
                    if (cols % 2 == 0 && col < cols && (reinterpret_cast<uintptr_t>(at_out) & 7) == 0) {
                        *reinterpret_cast<float2 *>(at_out) = make_float2(out[0], out[1]);
                        continue;
                    }
                    if (col < cols) at_out[0] = out[0];
                    if (col + 1 < cols) at_out[1] = out[1];
                } else {
                    uint16_t *at_out = reinterpret_cast<uint16_t *>(m.out) + at + col;
                    if (col < cols) at_out[0] = to_16bit(out[0], type);
                    if (col + 1 < cols) at_out[1] = to_16bit(out[1], type);
                }
            }
        }
        const int64_t next = row + kGramWarps * 8 * kAhead;
        if (next < last) fetch(next);
    }
}

// Two blocks to an SM over all matrices, at most kGramParts to a matrix; a multiple of 32 rows each.
static int64_t gram_strip(int64_t rows, int64_t most_rows, int sms) {
    int64_t strip = ceil_div(rows, 2 * sms);
    if (strip < ceil_div(most_rows, kGramParts)) strip = ceil_div(most_rows, kGramParts);
    return ceil_div(strip < 1 ? 1 : strip, 32) * 32;
}

int64_t gram_workspace_bytes(int64_t matrices, int64_t rows, int sms) {
    // a strip is at least rows / (2 sms) of all rows: that many whole ones, and one more for each matrix
    return (2 * sms + matrices) * (int64_t)kGramSums * (int64_t)sizeof(double);
}

int launch_gram_steps(const GramJob &job, int steps, const float *coefficients, double eps, double *workspace, int sms, cudaStream_t st,
                      const char *what) {
    GramBlocks g = {};
    g.job = job;
    g.steps = steps;
    g.scale_eps = eps;
    for (int i = 0; i < 3 * steps; ++i) g.coefficients[i] = coefficients[i];
    int64_t rows = 0, most = 0;
    for (int i = 0; i < job.count; ++i) {
        rows += job.matrix[i].rows;
        if (job.matrix[i].rows > most) most = job.matrix[i].rows;
    }
    const int64_t batch = job.count == 1 ? job.batch : 1;
    g.strip = gram_strip(rows * batch, most, sms);
    for (int i = 0; i < job.count; ++i) g.first[i + 1] = g.first[i] + (int)ceil_div(job.matrix[i].rows, g.strip);
    const int64_t blocks = g.first[job.count] * batch;
    launch_dependent(true, gram_sums_kernel, dim3((unsigned)blocks), dim3(kGramThreads), 0, st, g, workspace);
    int status = launch_status(what);
    if (status != DL_OK) return status;
    launch_dependent(true, gram_apply_kernel, dim3((unsigned)blocks), dim3(kGramThreads), 0, st, g, (const double *)workspace);
    return launch_status(what);
}

}  // namespace dl
