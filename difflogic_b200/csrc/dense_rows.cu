// Dense layers of few samples: y[b][f] = sum_k x[b][k] w[f][k], bound by reading w once.
//
// A block takes 16 or 32 outputs for all samples; its eight warps take every eighth piece of k each and add their sums up in shared
// memory.  The products go to the warp-wide matrix instructions (16 outputs x 8 samples), which take their operands from registers, so
// that w goes from memory straight into them: fp32 values are split there, where the tensor cores' tiles would have them laid out in three planes
// in memory first, four times the bytes of w; and no tile of 64 columns waits for samples that are not there.
// 4096 -> 16000, 8 samples, fp32: 51 us, 5.2 TB/s; 784 -> 16000: 15 us, 3.4 TB/s, bound by the latency of reads of which a block has 4
// a thread under way; 2048 -> 2048, one sample, bf16: 5 us, a launch and two waits for memory.
// The order in which k is summed is free: a lane reads 16 neighbouring bytes of its rows of w and of x, and what the instruction calls
// columns t and t + 4 (fp32) are neighbours in memory.
//
// fp32: hi + lo, hi the nearest value of 11 bits (the instruction reads no more), lo the rest, of which it reads 11 bits: lo hi + hi lo, then
// hi hi, in sums that are taken out every two pieces, since the instruction cuts off what is below its last bit.  lo has 12 bits and
// either sign, so that its cut-off bit (2^-23 of the value at most, a quarter of the values) and lo lo (2^-24, at worst 2^-22, of the
// product) average out over a sum.  (hi cut off in place of rounded: all of them of the product's sign.)  Off by, over the results' root mean
// square, for 784 positive operands 1.2e-7 on average and 1.3e-7 in all, a library's 32-bit product 4e-9 and 4.2e-7; hi cut off, and sums taken
// out every four pieces, 4.6e-7 both.
#include "dense_epilogue.cuh"

namespace dl {

constexpr int kRowsThreads = 256, kRowsWarps = kRowsThreads / 32;

struct RowsJob {
    const void *x, *w;
    int64_t x_row, x_col;    // values to the next sample, to the next input
    int64_t inner, outer;
    int batch, type;
    bool x_whole;            // rows of x can be read 16 bytes at a time
};

__device__ __forceinline__ uint4 load_once(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// 16 bytes' worth of values from input k on, zeros behind the last one.
template <bool FULL>
__device__ __forceinline__ uint4 load_piece(const void *row, int64_t step, int64_t k, int64_t inner, bool whole, bool streamed) {
    constexpr int kValues = FULL ? 4 : 8;
    if (whole) {
        if (k >= inner) return make_uint4(0, 0, 0, 0);
        const void *at = reinterpret_cast<const char *>(row) + k * (FULL ? 4 : 2);
        return streamed ? load_once(at) : __ldg(reinterpret_cast<const uint4 *>(at));
    }
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kValues; ++j) {
        if (k + j >= inner) continue;
        if (FULL) v[j] = reinterpret_cast<const uint32_t *>(row)[(k + j) * step];
        else v[j / 2] |= (uint32_t) reinterpret_cast<const uint16_t *>(row)[(k + j) * step] << (j % 2 * 16);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ void multiply_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void multiply_16bit(float (&d)[4], bool bfloat, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (bfloat)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four values become the nearest ones of 11 bits; returns what that leaves.  (Values that round to infinity, the last 2^-12 of fp32's range,
// make results that are not finite, which product_once_more sees to.)
__device__ __forceinline__ uint4 split_piece(uint4 &v) {
    uint32_t *u[4] = {&v.x, &v.y, &v.z, &v.w}, lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t hi = (*u[j] + 0x1000u) & 0xffffe000u;
        lo[j] = __float_as_uint(__uint_as_float(*u[j]) - __uint_as_float(hi));
        *u[j] = hi;
    }
    return make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// A whole warp's: one result of fp32 operands in 64 bits, for sums that are not finite.  Infinities and NaN have their way then, and what
// passed fp32's range on the way alone is back in it.
__device__ __noinline__ float product_once_more(const RowsJob &j, int64_t output, int sample) {
    const float *w = reinterpret_cast<const float *>(j.w) + output * j.inner, *x = reinterpret_cast<const float *>(j.x) + sample * j.x_row;
    double sum = 0;
    for (int64_t k = threadIdx.x % 32; k < j.inner; k += 32) sum += (double)x[k * j.x_col] * w[k];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    return (float)sum;
}

// MT groups of 16 outputs, NT of 8 samples; FULL: fp32; WHOLE: rows of w can be read 16 bytes at a time.
template <int MT, int NT, bool FULL, bool WHOLE>
__global__ void __launch_bounds__(kRowsThreads, MT * NT == 1 ? 3 : 2)
dense_rows_kernel(const __grid_constant__ RowsJob j, const DenseOutput output) {
    constexpr int kPiece = FULL ? 16 : 32;   // values of k that a warp's four lanes of a row read at a time
    constexpr int kAhead = NT == 1 ? 4 : 2;
    constexpr int kOutputs = 16 * MT, kSamples = 8 * NT;
    __shared__ float s_sum[kRowsWarps][kOutputs][kSamples + 1];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
    const int64_t base = (int64_t)blockIdx.x * kOutputs;
    const char *rows[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t f = base + m * 16 + h * 8 + g;   // outputs behind the last one: its row once more
            rows[m][h] = reinterpret_cast<const char *>(j.w) + (f < j.outer ? f : j.outer - 1) * j.inner * (FULL ? 4 : 2);
        }
    float sum[MT][NT][4] = {};
    grid_dependency_wait();
    grid_dependents_launch();
    for (int64_t first = (int64_t)warp * kPiece; first < j.inner; first += (int64_t)kAhead * kRowsWarps * kPiece) {
        uint4 w[kAhead][MT][2], x[kAhead][NT];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t k = first + (int64_t)i * kRowsWarps * kPiece + t * (kPiece / 4);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) w[i][m][h] = load_piece<FULL>(rows[m][h], 1, k, j.inner, WHOLE, true);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int b = n * 8 + g;
                x[i][n] = make_uint4(0, 0, 0, 0);
                if (b < j.batch)
                    x[i][n] = load_piece<FULL>(reinterpret_cast<const char *>(j.x) + b * j.x_row * (FULL ? 4 : 2), j.x_col, k, j.inner, j.x_whole, false);
            }
        }
        float part[MT][NT][4] = {};
        if constexpr (FULL) {
            // the small products of all pieces, then the large ones, in sums of their own: lo may have either sign, and beside it a large sum near
            // fp32's end would pass it
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                uint4 rest[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) rest[n] = split_piece(x[i][n]);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint4 c = split_piece(w[i][m][0]), d = split_piece(w[i][m][1]);
                    const uint4 &up = w[i][m][0], &down = w[i][m][1];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        multiply_tf32(part[m][n], c.x, d.x, c.y, d.y, x[i][n].x, x[i][n].y);
                        multiply_tf32(part[m][n], up.x, down.x, up.y, down.y, rest[n].x, rest[n].y);
                        multiply_tf32(part[m][n], c.z, d.z, c.w, d.w, x[i][n].z, x[i][n].w);
                        multiply_tf32(part[m][n], up.z, down.z, up.w, down.w, rest[n].z, rest[n].w);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        sum[m][n][q] += part[m][n][q];
                        part[m][n][q] = 0.f;
                    }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 &up = w[i][m][0], &down = w[i][m][1];
                        if (i % 2 == 0 && i > 0) {   // every two pieces
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                sum[m][n][q] += part[m][n][q];
                                part[m][n][q] = 0.f;
                            }
                        }
                        multiply_tf32(part[m][n], up.x, down.x, up.y, down.y, x[i][n].x, x[i][n].y);
                        multiply_tf32(part[m][n], up.z, down.z, up.w, down.w, x[i][n].z, x[i][n].w);
                    }
        } else {
            const bool bfloat = j.type == kBFloat16;
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 &a = w[i][m][0], &c = w[i][m][1], &b = x[i][n];
                        multiply_16bit(part[m][n], bfloat, a.x, c.x, a.y, c.y, b.x, b.y);
                        multiply_16bit(part[m][n], bfloat, a.z, c.z, a.w, c.w, b.z, b.w);
                    }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[m][n][i] += part[m][n][i];
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_sum[warp][m * 16 + i / 2 * 8 + g][n * 8 + t * 2 + i % 2] = sum[m][n][i];
    __syncthreads();
    for (int first = warp * 32; first < kOutputs * j.batch; first += kRowsThreads) {
        const int i = first + lane, f = output.feature_major ? i / j.batch : i % kOutputs, b = output.feature_major ? i % j.batch : i / kOutputs;
        const bool there = i < kOutputs * j.batch && base + f < j.outer;
        float r = 0.f;
        if (there) {
#pragma unroll
            for (int v = 0; v < kRowsWarps; ++v) r += s_sum[v][f][b];
        }
        if constexpr (FULL) {
            for (uint32_t again = __ballot_sync(0xffffffffu, !(fabsf(r) <= 3.402823466e38f)); again != 0; again &= again - 1) {
                const int whose = __ffs(again) - 1;
                const float v = product_once_more(j, base + __shfl_sync(0xffffffffu, f, whose), __shfl_sync(0xffffffffu, b, whose));
                if (lane == whose) r = v;
            }
        }
        if (there) output.one((int)(base + f), b, r);
    }
}

// This way / the tensor cores' way (one sample more), us: fp32 784 -> 16000, 16 samples: 18 / 51, 32: 32 / 51; 2048 -> 2048: 12 / 25, 15 / 25;
// 784 -> 256, 32: 6.5 / 14; bf16 784 -> 16000, 8: 9.0 / 11, 16: 12.3 / 10.5; 2048 -> 2048, 16: 7.0 / 9.6; rows off the 16-byte units, 783 -> 2001,
// 16: 8.2 / 14.  Not so where few outputs and a long sum leave most SMs without a block, which the rule does not look at: fp32 16000 -> 10,
// 8: 30 / 23, 32: 80 / 23; 4096 -> 100, 8: 12 / 17, 32: 26 / 17.
bool dense_rows_applicable(int64_t batch, int type) { return batch <= (type == kFloat32 ? 32 : 16); }

template <int NT, bool FULL, bool WHOLE>
static void launch_outputs(const RowsJob &j, const DenseOutput &e, int sms, cudaStream_t st) {
    // 32 outputs to a block read x half as often as 16, where there are blocks for all SMs all the same (and registers: NT < 4)
    if constexpr (NT < 4)
        if (j.outer >= 32 * 2 * sms) {
            launch_dependent(true, dense_rows_kernel<2, NT, FULL, WHOLE>, dim3((unsigned)ceil_div(j.outer, 32)), dim3(kRowsThreads), 0, st, j, e);
            return;
        }
    launch_dependent(true, dense_rows_kernel<1, NT, FULL, WHOLE>, dim3((unsigned)ceil_div(j.outer, 16)), dim3(kRowsThreads), 0, st, j, e);
}

template <int NT>
static void launch_samples(const RowsJob &j, const DenseOutput &e, bool whole, int sms, cudaStream_t st) {
    if constexpr (NT == 4) whole ? launch_outputs<NT, true, true>(j, e, sms, st) : launch_outputs<NT, true, false>(j, e, sms, st);   // fp32 alone
    else if (j.type == kFloat32) whole ? launch_outputs<NT, true, true>(j, e, sms, st) : launch_outputs<NT, true, false>(j, e, sms, st);
    else whole ? launch_outputs<NT, false, true>(j, e, sms, st) : launch_outputs<NT, false, false>(j, e, sms, st);
}

int launch_dense_rows(const void *x, int64_t x_pitch, bool x_feature_major, const void *w, const DenseOutput &output, int64_t batch,
                      int64_t inner, int64_t outer, int type, int sms, cudaStream_t st) {
    const int values = type == kFloat32 ? 4 : 8;
    const bool x_whole = !x_feature_major && aligned_to(x, 16) && inner % values == 0 && (batch == 1 || x_pitch % values == 0);
    const RowsJob j = {x, w, x_feature_major ? 1 : x_pitch, x_feature_major ? x_pitch : 1, inner, outer, (int)batch, type, x_whole};
    const bool whole = aligned_to(w, 16) && inner % values == 0;
    if (batch <= 8) launch_samples<1>(j, output, whole, sms, st);
    else if (batch <= 16) launch_samples<2>(j, output, whole, sms, st);
    else launch_samples<4>(j, output, whole, sms, st);
    return launch_status("dl_dense_forward");
}

}  // namespace dl
