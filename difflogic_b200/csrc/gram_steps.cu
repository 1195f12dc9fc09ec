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
//
// A step of four matrices of 128000 x 16: 42 us, 17 for the sums and 24 for the rest, 98 and 131 MB of reads and writes: 5.5 TB/s, HBM and
// L2 together (every byte of the operands once would be 164 MB and 25 us).  Five of 16000 x 16: 12 us, bound by latency: two launches, the
// sums of a matrix (2 us) and five steps one after the other (3 us).
#include "gram_steps.h"
#include "matmul_values.cuh"

namespace dl {

constexpr int kGramThreads = 512, kGramWarps = kGramThreads / 32;   // of a block that takes the steps
constexpr int kSumThreads = 256, kSumWarps = kSumThreads / 32;      // of one that adds S up
constexpr int kGramSums = 3 * 64;        // three 8 x 8 blocks of S: even-even, even-odd and odd-odd columns
constexpr int kGramParts = 128;          // at most, of a matrix

struct GramBlocks {
    GramJob job;
    struct {
        int64_t strip;                   // rows of a block
        int first[GramJob::kMost + 1];   // block of every matrix (batch: of the first one)
    } sums, rows;
    double scale_eps;
    int steps;
    float coefficients[3 * kMostSteps];
};

__device__ __forceinline__ void multiply64(double (&d)[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}

struct GramPlace {
    int matrix, sums, parts;             // entry; its first sum, and how many
    int64_t base, first, last;           // first value; rows of the block
};
template <class Cut>
__device__ __forceinline__ GramPlace gram_place(const GramBlocks &g, const Cut &cut, int block) {
    GramPlace p;
    p.matrix = 0;
    p.base = 0;
    p.sums = 0;
    if (g.job.count == 1) {
        const int z = block / cut.first[1];
        block -= z * cut.first[1];
        p.base = z * g.job.matrix[0].rows * g.job.cols;
        p.sums = z * g.sums.first[1];
    } else {
        while (block >= cut.first[p.matrix + 1]) ++p.matrix;
        block -= cut.first[p.matrix];
        p.sums = g.sums.first[p.matrix];
    }
    p.parts = g.sums.first[p.matrix + 1] - g.sums.first[p.matrix];
    const int64_t rows = g.job.matrix[p.matrix].rows;
    p.first = block * cut.strip;
    p.last = p.first + cut.strip < rows ? p.first + cut.strip : rows;
    return p;
}

// N neighbouring values of row `row` of `cols`; a row that is not there reads as the last one.  WHOLE: rows of 16 fp32 values on 16-byte
// units, else values one by one, zeros behind the end of a row.
template <bool WHOLE, int N>
__device__ __forceinline__ void load_row(const void *p, int64_t base, int64_t row, int64_t last, int col, int cols, int type, float (&v)[N]) {
    const int64_t at = base + (row < last ? row : last - 1) * (WHOLE ? kGramColumns : cols) + col;
    if constexpr (WHOLE && N == 4) {
        const float4 f = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + at);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else if constexpr (WHOLE) {
        const float2 f = *reinterpret_cast<const float2 *>(reinterpret_cast<const float *>(p) + at);
        v[0] = f.x; v[1] = f.y;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = col + j < cols ? load_as_float(p, at + j, type) : 0.f;
    }
}
template <bool WHOLE>
__device__ __forceinline__ void store_two(void *p, int64_t at, int col, int cols, int type, float a, float b) {
    if constexpr (WHOLE) {
        *reinterpret_cast<float2 *>(reinterpret_cast<float *>(p) + at) = make_float2(a, b);
    } else if (type == kFloat32) {
        if (col < cols) reinterpret_cast<float *>(p)[at] = a;
        if (col + 1 < cols) reinterpret_cast<float *>(p)[at + 1] = b;
    } else {
        if (col < cols) reinterpret_cast<uint16_t *>(p)[at] = to_16bit(a, type);
        if (col + 1 < cols) reinterpret_cast<uint16_t *>(p)[at + 1] = to_16bit(b, type);
    }
}

// UPDATE: of momenta, of weights.
template <bool WHOLE, bool UPDATE>
__global__ void __launch_bounds__(kSumThreads, 3)
gram_sums_kernel(const __grid_constant__ GramBlocks g, double *__restrict__ sums) {
    __shared__ double s_sum[kSumWarps][kGramSums];
    grid_dependency_wait();
    grid_dependents_launch();
    const GramPlace p = gram_place(g, g.sums, blockIdx.x);
    const GramMatrix &m = g.job.matrix[p.matrix];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, cols = g.job.cols, type = g.job.type, col = lane / 4 * 2;
    const int64_t first = p.first, last = p.last;
    // lane l: row l % 4, columns 2 (l / 4) and the one after it, which makes its value both the A and the B of a block of S
    double even[2] = {0, 0}, mixed[2] = {0, 0}, odd[2] = {0, 0};
    constexpr int kAhead = 8;   // rows of four at a time
    for (int64_t row = first + warp * 4 * kAhead; row < last; row += kSumWarps * 4 * kAhead) {
        float v[kAhead][2], o[kAhead][2];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * 4 + lane % 4;
            load_row<WHOLE>(m.g, p.base, r, last, col, cols, type, v[i]);
            if (UPDATE) load_row<WHOLE>(m.momentum, p.base, r, last, col, cols, kFloat32, o[i]);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * 4 + lane % 4;
            const bool there = r < last;
            if (UPDATE) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    o[i][j] = new_momentum(o[i][j], v[i][j], g.job.keep);
                    v[i][j] = update_of(o[i][j], v[i][j], g.job.nesterov);
                }
                if (there) store_two<WHOLE>(m.momentum, p.base + r * (WHOLE ? kGramColumns : cols) + col, col, cols, kFloat32, o[i][0], o[i][1]);
            }
            const double a = there ? v[i][0] : 0.f, b = there ? v[i][1] : 0.f;
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
        for (int w = 0; w < kSumWarps; ++w) r += s_sum[w][threadIdx.x];
        sums[(int64_t)blockIdx.x * kGramSums + threadIdx.x] = r;
    }
}

constexpr int kSquarePitch = 18;   // doubles of a row of a 16 x 16 matrix
using Square = double[kGramColumns][kSquarePitch];

// One 8 x 8 block of A B, in two chains: an instruction takes about 30 clocks until its sum can be added to.
__device__ __forceinline__ void square_block(const Square &a, const Square &b, int block, int lane, double (&d)[2]) {
    const int down = block / 2 * 8, across = block % 2 * 8;
    double e[2] = {0, 0};
    d[0] = d[1] = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        multiply64(d, a[down + lane / 4][4 * k + lane % 4], b[4 * k + lane % 4][across + lane / 4]);
        multiply64(e, a[down + lane / 4][4 * k + 8 + lane % 4], b[4 * k + 8 + lane % 4][across + lane / 4]);
    }
    d[0] += e[0];
    d[1] += e[1];
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
        constexpr int kMost = kGramParts / kGramWarps;   // of a warp, all asked for at a time
        double2 d[kMost][kGramSums / 64];
#pragma unroll
        for (int i = 0; i < kMost; ++i)
#pragma unroll
            for (int j = 0; j < kGramSums / 64; ++j) {
                const int part = warp + i * kGramWarps;
                d[i][j] = part < parts ? *reinterpret_cast<const double2 *>(sums + (int64_t)part * kGramSums + j * 64 + lane * 2) : make_double2(0, 0);
            }
#pragma unroll
        for (int i = 0; i < kMost; ++i)
#pragma unroll
            for (int j = 0; j < kGramSums / 64; ++j) {
                r[2 * j] += d[i][j].x;
                r[2 * j + 1] += d[i][j].y;
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
    if (warp == 0) {
        double trace = lane < kGramColumns ? s.s[lane][lane] : 0;
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) trace += __shfl_xor_sync(0xffffffffu, trace, off);
        if (lane == 0) {
            const double norm = sqrt(trace);
            s.scale = norm > g.scale_eps || norm != norm ? 1 / norm : 1 / g.scale_eps;
        }
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
            if (warp >= 4 && warp < 8) {
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

template <bool WHOLE, bool UPDATE>
__global__ void __launch_bounds__(kGramThreads, 1)
gram_apply_kernel(const __grid_constant__ GramBlocks g, const double *__restrict__ sums) {
    __shared__ GramShared s;
    grid_dependency_wait();
    grid_dependents_launch();
    const GramPlace p = gram_place(g, g.rows, blockIdx.x);
    const GramMatrix &m = g.job.matrix[p.matrix];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, cols = g.job.cols, type = g.job.type;
    const int64_t first = p.first, last = p.last;
    // a warp takes 8 rows at a time: lane l reads columns 4 (l % 4) .. + 3 of row l / 4 (which order the columns are summed in is
    // free) and has columns 2 (l % 4), + 1, + 8 and + 9 of the result
    constexpr int kAhead = 2;
    const int from = lane % 4 * 4, to = lane % 4 * 2;
    struct Rows {
        float v[kAhead][4], o[kAhead][4], w[kAhead][2][2];
    };
    const auto fetch = [&](Rows &b, int64_t row) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * 8 + lane / 4;
            load_row<WHOLE>(m.g, p.base, r, last, from, cols, type, b.v[i]);
            if (UPDATE) {
                load_row<WHOLE>(m.momentum, p.base, r, last, from, cols, kFloat32, b.o[i]);
                load_row<WHOLE>(m.out, p.base, r, last, to, cols, kFloat32, b.w[i][0]);
                load_row<WHOLE>(m.out, p.base, r, last, to + 8, cols, kFloat32, b.w[i][1]);
            }
        }
    };
    constexpr int kStride = kGramWarps * 8 * kAhead;
    Rows one, two;   // while one is worked on, the other is on its way
    int64_t row = first + warp * 8 * kAhead;
    fetch(one, row);
    fetch(two, row + kStride);
    const Square &product = take_steps(s, g, sums + (int64_t)p.sums * kGramSums, p.parts);
    double factor[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) factor[h][k] = product[from + k][8 * h + lane / 4];
    const auto apply = [&](const Rows &b, int64_t row) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t r = row + i * 8 + lane / 4;
            double d[2][2] = {};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double x = UPDATE ? update_of(b.o[i][k], b.v[i][k], g.job.nesterov) : b.v[i][k];
                multiply64(d[0], x, factor[0][k]);
                multiply64(d[1], x, factor[1][k]);
            }
            if (r >= last) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float out[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) out[j] = UPDATE ? b.w[i][h][j] * g.job.decay - m.rate * (float)d[h][j] : (float)d[h][j];
                const int col = to + 8 * h;
                store_two<WHOLE>(m.out, p.base + r * (WHOLE ? kGramColumns : cols) + col, col, cols, UPDATE ? kFloat32 : type, out[0], out[1]);
            }
        }
        __syncwarp();
    };
    for (; row < last; row += 2 * kStride) {
        apply(one, row);
        if (row + 2 * kStride < last) fetch(one, row + 2 * kStride);
        if (row + kStride >= last) break;
        apply(two, row + kStride);
        if (row + 3 * kStride < last) fetch(two, row + 3 * kStride);
    }
}

// Sums: three blocks to an SM over all matrices, 256 rows at a time, at most kGramParts to a matrix.
static int64_t sum_strip(int64_t rows, int64_t most_rows, int sms) {
    const int64_t each = ceil_div(rows, 3 * sms), least = ceil_div(most_rows, kGramParts);
    return ceil_div(each > least ? each : least, 256) * 256;
}

int64_t gram_workspace_bytes(int64_t matrices, int64_t rows, int sms) {
    // a strip has at least rows / (3 sms) of all rows: that many whole ones, and one more for each matrix
    return (3 * sms + matrices) * (int64_t)kGramSums * (int64_t)sizeof(double);
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
    g.sums.strip = sum_strip(rows * batch, most, sms);
    // a block to an SM, as each takes the steps; not one more than there are, which would run alone
    const auto blocks_of = [&](int64_t strip) {
        int64_t n = 0;
        for (int i = 0; i < job.count; ++i) n += ceil_div(job.matrix[i].rows, strip);
        return n * batch;
    };
    g.rows.strip = ceil_div(ceil_div(rows * batch, sms), 32) * 32;
    while (blocks_of(g.rows.strip) > sms && g.rows.strip < most) g.rows.strip += 32;
    for (int i = 0; i < job.count; ++i) {
        g.sums.first[i + 1] = g.sums.first[i] + (int)ceil_div(job.matrix[i].rows, g.sums.strip);
        g.rows.first[i + 1] = g.rows.first[i] + (int)ceil_div(job.matrix[i].rows, g.rows.strip);
    }
    bool whole = job.cols == kGramColumns && job.type == kFloat32;
    for (int i = 0; i < job.count; ++i)
        whole = whole && aligned_to(job.matrix[i].g, 16) && aligned_to(job.matrix[i].momentum, 16) && aligned_to(job.matrix[i].out, 16);
    const dim3 sums((unsigned)(g.sums.first[job.count] * batch)), blocks((unsigned)(g.rows.first[job.count] * batch));
    const auto launch = [&](auto sums_kernel, auto apply_kernel) {
        launch_dependent(true, sums_kernel, sums, dim3(kSumThreads), 0, st, g, workspace);
        launch_dependent(true, apply_kernel, blocks, dim3(kGramThreads), 0, st, g, (const double *)workspace);
    };
    if (whole && job.update) launch(gram_sums_kernel<true, true>, gram_apply_kernel<true, true>);
    else if (whole) launch(gram_sums_kernel<true, false>, gram_apply_kernel<true, false>);
    else if (job.update) launch(gram_sums_kernel<false, true>, gram_apply_kernel<false, true>);
    else launch(gram_sums_kernel<false, false>, gram_apply_kernel<false, false>);
    return launch_status(what);
}

}  // namespace dl
