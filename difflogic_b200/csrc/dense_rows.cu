// Dense layers of few samples: y[b][f] = sum_k x[b][k] w[f][k], bound by reading w once.
//
// A warp takes R outputs at a time for all samples: its lanes read 16 bytes each of R rows of w (single values where rows are off the
// 16-byte units), multiply them with the samples, which lie in shared memory as fp32, and add up R x B sums of their own; then the lanes
// share out the sums, halving them five times.  The ordinary FMA units do: at B samples they have B products for every value of w, 90
// of 128 a clock for 16 fp32 or 8 bf16 samples at the rate at which memory delivers w.  fp32 values stay as they are here, where the
// tensor cores would have them laid out in three planes first, four times the bytes of w.
//
// Samples are a chunk of at most 64 KB at a time, so that two blocks fit an SM.
#include "dense_epilogue.cuh"

namespace dl {

constexpr int kRowsThreads = 256, kRowsWarps = kRowsThreads / 32;
constexpr int kRowsBytes = 65536;

struct RowsJob {
    const void *x, *w;
    int64_t x_row, x_col;    // values to the next sample, to the next input
    int64_t inner, outer;
    int batch, type;
    int chunk;               // inputs in shared memory at a time
};

template <int WIDTH>
__device__ __forceinline__ void load_weights(const void *w, int64_t at, int type, float (&v)[WIDTH]) {
    if constexpr (WIDTH == 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(w) + at));
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else if constexpr (WIDTH == 8) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(w) + at));
        const uint32_t p[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (type == kBFloat16) {
                v[2 * j] = __uint_as_float(p[j] << 16);
                v[2 * j + 1] = __uint_as_float(p[j] & 0xffff0000u);
            } else {
                const __half2 h = *reinterpret_cast<const __half2 *>(&p[j]);
                v[2 * j] = __low2float(h);
                v[2 * j + 1] = __high2float(h);
            }
        }
    } else {
        v[0] = load_as_float(w, at, type);
    }
}

// Where input k of a chunk lies in shared memory.  Lanes read 8 neighbouring ones as two quads: the first and the second quads of all
// lanes lie apart, so that 8 lanes meet no bank twice.
template <int WIDTH>
__device__ __forceinline__ int place_of(int k, int chunk) {
    return WIDTH == 8 ? k / 8 * 4 + k % 4 + (k % 8 / 4) * (chunk / 2) : k;
}

template <int B, int R, int WIDTH>
__global__ void __launch_bounds__(kRowsThreads)
dense_rows_kernel(const RowsJob j, const DenseEpilogue epilogue) {
    extern __shared__ float s_x[];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    constexpr int kAll = R * B;
    grid_dependency_wait();
    grid_dependents_launch();
    for (int64_t group = (int64_t)blockIdx.x * kRowsWarps * R; group < j.outer; group += (int64_t)gridDim.x * kRowsWarps * R) {
        const int64_t feature = group + warp * R;
        float sum[kAll];
#pragma unroll
        for (int i = 0; i < kAll; ++i) sum[i] = 0.f;
        for (int64_t from = 0; from < j.inner; from += j.chunk) {
            const int count = (int)(j.inner - from < j.chunk ? j.inner - from : j.chunk);
            if (j.inner > j.chunk || group == (int64_t)blockIdx.x * kRowsWarps * R) {
                __syncthreads();
                for (int i = threadIdx.x; i < B * j.chunk; i += kRowsThreads) {   // zeros behind the last sample and input
                    const int b = i / j.chunk, k = i - b * j.chunk;
                    s_x[b * j.chunk + place_of<WIDTH>(k, j.chunk)] =
                        b < j.batch && k < count ? load_as_float(j.x, b * j.x_row + (from + k) * j.x_col, j.type) : 0.f;
                }
                __syncthreads();
            }
            if (feature >= j.outer) continue;
            // WIDTH divides j.inner where it is not 1: whole vectors only
#pragma unroll 4
            for (int k = lane * WIDTH; k < count; k += 32 * WIDTH) {
                float w[R][WIDTH];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const int64_t f = feature + r < j.outer ? feature + r : j.outer - 1;
                    load_weights<WIDTH>(j.w, f * j.inner + from + k, j.type, w[r]);
                }
#pragma unroll
                for (int b = 0; b < B; ++b) {
                    float x[WIDTH];
                    if constexpr (WIDTH == 1) {
                        x[0] = s_x[b * j.chunk + k];
                    } else {
#pragma unroll
                        for (int q = 0; q < WIDTH / 4; ++q) {
                            const float4 f = *reinterpret_cast<const float4 *>(s_x + b * j.chunk + place_of<WIDTH>(k + 4 * q, j.chunk));
                            x[4 * q] = f.x; x[4 * q + 1] = f.y; x[4 * q + 2] = f.z; x[4 * q + 3] = f.w;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r)
#pragma unroll
                        for (int i = 0; i < WIDTH; ++i) sum[r * B + b] = fmaf(w[r][i], x[i], sum[r * B + b]);
                }
            }
        }
        if (feature >= j.outer) continue;
        // halve the sums as long as there are two: a lane with the bit set keeps the upper half
        int index = 0;
#pragma unroll
        for (int off = 16, left = kAll; off > 0; off >>= 1) {
            if (left > 1) {
                left /= 2;
                const bool upper = lane & off;
#pragma unroll
                for (int i = 0; i < kAll / 2; ++i) {
                    if (i >= left) break;
                    const float give = upper ? sum[i] : sum[i + left], keep = upper ? sum[i + left] : sum[i];
                    sum[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
                }
                index += upper ? left : 0;
            } else {
                sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], off);
            }
        }
        constexpr int kLeft = kAll > 32 ? kAll / 32 : 1, kShared = kAll < 32 ? 32 / kAll : 1;   // sums of a lane; lanes with the same one
        if (lane % kShared != 0) continue;
#pragma unroll
        for (int i = 0; i < kLeft; ++i) {
            const int at = index + i, r = at / B, b = at % B;
            if (feature + r < j.outer && b < j.batch) epilogue.one((int)(feature + r), b, sum[i]);
        }
    }
}

// fp32: the tensor cores' way reads w, writes it in planes and reads those.  16-bit types: a tile of 64 columns is empty but for the
// samples there, but costs no more than the FMA units from here on.
bool dense_rows_applicable(int64_t batch, int64_t inner, int64_t outer, int type) {
    (void)inner;
    (void)outer;
    return batch <= (type == kFloat32 ? 16 : 4);
}

template <int B, int R, int WIDTH>
static void launch_rows(const RowsJob &job, const DenseEpilogue &epilogue, int sms, cudaStream_t st) {
    RowsJob j = job;
    int64_t chunk = kRowsBytes / (4 * B);
    if (chunk > ceil_div(j.inner, 8) * 8) chunk = ceil_div(j.inner, 8) * 8;   // a multiple of 8
    j.chunk = (int)chunk;
    const size_t shared = (size_t)B * chunk * 4;
    int64_t blocks = ceil_div(j.outer, kRowsWarps * R);
    const int64_t most = (int64_t)sms * (shared > 32768 ? 2 : 4);
    if (blocks > most) blocks = most;
    cudaFuncSetAttribute(dense_rows_kernel<B, R, WIDTH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsBytes);
    launch_dependent(true, dense_rows_kernel<B, R, WIDTH>, dim3((unsigned)blocks), dim3(kRowsThreads), shared, st, j, epilogue);
}

template <int B>
static void launch_batch(const RowsJob &j, const DenseEpilogue &e, bool whole, int sms, cudaStream_t st) {
    // one output to a warp where four would leave warps without any
    const bool four = j.outer >= (int64_t)4 * kRowsWarps * 2 * sms || B > 4;
    if (!whole) four ? launch_rows<B, 4, 1>(j, e, sms, st) : launch_rows<B, 1, 1>(j, e, sms, st);
    else if (j.type == kFloat32) four ? launch_rows<B, 4, 4>(j, e, sms, st) : launch_rows<B, 1, 4>(j, e, sms, st);
    else four ? launch_rows<B, 4, 8>(j, e, sms, st) : launch_rows<B, 1, 8>(j, e, sms, st);
}

int launch_dense_rows(const void *x, int64_t x_pitch, bool x_feature_major, const void *w, const DenseEpilogue &epilogue, int64_t batch,
                      int64_t inner, int64_t outer, int type, int sms, cudaStream_t st) {
    const RowsJob j = {x, w, x_feature_major ? 1 : x_pitch, x_feature_major ? x_pitch : 1, inner, outer, (int)batch, type, 0};
    const bool whole = aligned_to(w, 16) && inner % (type == kFloat32 ? 4 : 8) == 0;
    if (batch <= 1) launch_batch<1>(j, epilogue, whole, sms, st);
    else if (batch <= 2) launch_batch<2>(j, epilogue, whole, sms, st);
    else if (batch <= 4) launch_batch<4>(j, epilogue, whole, sms, st);
    else if (batch <= 8) launch_batch<8>(j, epilogue, whole, sms, st);
    else launch_batch<16>(j, epilogue, whole, sms, st);
    return launch_status("dl_dense_forward");
}

}  // namespace dl
