// Dense layers and the orthogonalisation of matrices: the matrix products of matmul.cuh with their epilogues, what lays out their
// operands, and the entry points.
#include <math.h>

#include "dense_epilogue.cuh"
#include "gram_steps.h"
#include "matmul.cuh"
#include "matmul_plan.h"

namespace dl {

int matmul_async_error() {
    int flag = 0;
    if (cudaMemcpyFromSymbol(&flag, g_matmul_async_error, sizeof(int)) != cudaSuccess) {
        cudaGetLastError();
        return -1;
    }
    return flag;
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                 const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

bool make_tile_map(CUtensorMap *map, const void *base, bool bfloat, int64_t inner, int64_t rows, int64_t planes, int64_t row_bytes,
                   int64_t plane_bytes) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    if (planes == 1) plane_bytes = row_bytes * rows;   // not used, but looked at
    const cuuint64_t sizes[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t pitches[2] = {(cuuint64_t)row_bytes, (cuuint64_t)plane_bytes};
    const cuuint32_t box[3] = {kChunk, kChunk, 1}, steps[3] = {1, 1, 1};
    return encode(map, bfloat ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), sizes,
                  pitches, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// -- launching a product --------------------------------------------------------------------------------------------------------

struct Product {
    Operand a, b;
    int64_t m, n, k, batch;
    int planes, planes_z;   // multiplied; per matrix in memory
    bool bfloat, symmetric;
    bool exact;   // sums are taken out of tensor memory every so often
};

static bool map_operand(CUtensorMap *map, const Operand &o, const Product &p, int64_t rows) {
    const int64_t inner = o.mn ? rows : p.k, outer = o.mn ? p.k : rows;
    return make_tile_map(map, o.base, p.bfloat, inner, outer, p.planes_z * p.batch, o.pitch * 2, o.plane * 2);
}

template <int PLANES, int COLUMNS, bool PAIR, class Epilogue>
static int launch_tiles(const MatmulShape &shape, const CUtensorMap &a, const CUtensorMap &b, const Epilogue &epilogue, int sms,
                        cudaStream_t st, const char *what) {
    using Config = MatmulConfig<PLANES, COLUMNS, PAIR>;
    auto kernel = matmul_kernel<PLANES, COLUMNS, PAIR, Epilogue>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Config::kSharedBytes) != cudaSuccess) return launch_status(what);
    const int64_t ctas = PAIR ? 2 * (int64_t)shape.tiles : shape.tiles, most = PAIR ? sms / 2 * 2 : sms;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ctas < most ? ctas : most));
    cfg.blockDim = dim3(Config::kThreadsAll);
    cfg.dynamicSmemBytes = Config::kSharedBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = PAIR ? 2 : 1;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, a, b, shape, epilogue);
    return launch_status(what);
}

template <int PLANES, class Epilogue>
static int launch_columns(const Product &p, const MatmulPlan &plan, const Epilogue &epilogue, int sms, cudaStream_t st, const char *what) {
    CUtensorMap a, b;
    if (!map_operand(&a, p.a, p, p.m) || !map_operand(&b, p.b, p, p.n))
        return fail(DL_ERR_CUDA, "%s: the driver refuses the map of an operand", what);
    const int rows = plan.pair ? 2 * kMatmulRows : kMatmulRows;
    MatmulShape s = {};
    s.m = (int32_t)p.m;
    s.n = (int32_t)p.n;
    s.batch = (int32_t)p.batch;
    s.planes_z = p.planes_z;
    s.tiles_m = (int32_t)ceil_div(p.m, rows);
    s.tiles_n = (int32_t)ceil_div(p.n, plan.columns);
    s.splits = plan.splits;
    s.k_steps = (int32_t)ceil_div(p.k, kChunk);
    s.steps_per_split = plan.steps_per_split;
    // one plane: nothing adds blocks up; wide tiles have one sum for large and small products
    s.steps_per_sum = PLANES > 1 && p.exact ? (plan.columns == 256 ? 1 : 2) : s.k_steps;
    s.symmetric = p.symmetric;
    const int64_t per_matrix = tiles_of(p.m, p.n, rows, plan.columns, p.symmetric), tiles = per_matrix * s.splits * p.batch;
    if (tiles > INT32_MAX / 2) return fail(DL_ERR_TOO_LARGE, "%s: too many tiles", what);
    s.per_matrix = (int32_t)per_matrix;
    s.tiles = (int32_t)tiles;
    s.a_mn = p.a.mn;
    s.b_mn = p.b.mn;
    s.instruction = instruction_descriptor(p.bfloat, p.a.mn, p.b.mn, rows, plan.columns);
    if (plan.pair) return launch_tiles<PLANES, 256, true>(s, a, b, epilogue, sms, st, what);
    if (plan.columns == 64) return launch_tiles<PLANES, 64, false>(s, a, b, epilogue, sms, st, what);
    if (plan.columns == 128) return launch_tiles<PLANES, 128, false>(s, a, b, epilogue, sms, st, what);
    return fail(DL_ERR_INVALID_ARG, "%s: no such tile", what);
}

// One product with its epilogue; `partial`: plan.partial_bytes.
template <int PLANES, class Epilogue>
static int launch_product(const Product &p, const MatmulPlan &plan, const Epilogue &epilogue, float *partial, int sms, cudaStream_t st,
                          const char *what) {
    if (plan.splits == 1) return launch_columns<PLANES>(p, plan, epilogue, sms, st, what);
    const int status = launch_columns<PLANES>(p, plan, StorePartial{partial, p.n, p.m * p.n}, sms, st, what);
    if (status != DL_OK) return status;
    const int64_t quads = ceil_div(p.n, 4) * p.m * p.batch;
    int64_t blocks = ceil_div(quads, kThreads);
    if (blocks > 8 * sms) blocks = 8 * sms;
    launch_dependent(true, matmul_join_kernel<Epilogue>, dim3((unsigned)blocks), dim3(kThreads), 0, st, (const float *)partial, plan.splits,
                     (int)p.batch, (int)p.m, (int)p.n, (int)p.symmetric, epilogue);
    return launch_status(what);
}

// Dense layers multiply one plane or three, the iterations one or two.
template <class Epilogue>
static int launch_planes(const Product &p, const MatmulPlan &plan, const Epilogue &e, float *partial, int sms, cudaStream_t st, const char *what) {
    constexpr int kMore = Epilogue::kPlanes;
    return p.planes == 1 ? launch_product<1>(p, plan, e, partial, sms, st, what) : launch_product<kMore>(p, plan, e, partial, sms, st, what);
}

// Values of a row of planes that the library lays out: whole units of 16 bytes.
static int64_t padded(int64_t n) { return ceil_div(n, 8) * 8; }
static int64_t padded_bytes(int64_t n) { return ceil_div(n, 256) * 256; }

// ============================================================== dense layers ====================================================

// Gradients: the sums as they are, in the layer's type.
struct PlainEpilogue {
    static constexpr int kPlanes = 3;
    void *out;
    int64_t pitch;
    int type;
    __device__ __forceinline__ bool by_column(int, int) const { return false; }
    __device__ __forceinline__ bool by_row(int, int) const { return true; }
    template <int N>
    __device__ __forceinline__ void down(int, int, int, const float (&)[N], int, int) const {}
    template <int N, int STEP>
    __device__ __forceinline__ void across(int, int row, int col, const float (&sum)[N][4], int m, int valid) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (row + i * STEP < m) store4(out, (row + i * STEP) * pitch + col, type, valid, sum[i]);
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

// The layer's outputs are the rows of the product where that leaves fewer of a tile's 128 rows and 64 columns empty.
static bool features_as_rows(int64_t batch, int64_t outer) { return batch < outer && batch < 256; }

static MatmulPlan plan_forward(int64_t batch, int64_t inner, int64_t outer, int planes, int sms) {
    return features_as_rows(batch, outer) ? plan_matmul(outer, batch, inner, 1, planes, false, sms) : plan_matmul(batch, outer, inner, 1, planes, false, sms);
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
                                             int64_t outer, int type, int64_t *sizes) {
    sizes[0] = sizes[1] = sizes[2] = 0;
    if (batch <= 0 || inner <= 0 || outer <= 0 || dense_rows_applicable(batch, type)) return;
    const DenseLayout l = dense_layout(batch, inner, outer, x_pitch, x_feature_major != 0, type, x, w);
    sizes[0] = l.x_bytes;
    sizes[1] = l.w_bytes;
    sizes[2] = plan_forward(batch, inner, outer, l.planes, current_sms()).partial_bytes;
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
        const DenseEpilogue e = {y, bias, residual, slope, y_feature_major ? batch : outer, residual_feature, residual_batch, type, act, true,
                                 y_feature_major != 0};
        return launch_dense_rows(x, x_pitch, x_feature_major != 0, w, e, batch, inner, outer, type, sms, st);
    }
    const MatmulPlan plan = plan_forward(batch, inner, outer, l.planes, sms);
    DL_REQUIRE((!l.lay_x || x_planes) && (!l.lay_w || w_planes) && (plan.partial_bytes == 0 || workspace), DL_ERR_INVALID_ARG,
               "%s: a workspace is missing", what);
    DL_REQUIRE(aligned_to(x_planes, 16) && aligned_to(w_planes, 16) && aligned_to(workspace, 16), DL_ERR_INVALID_ARG,
               "%s: workspaces must be 16-byte aligned", what);
    if (l.lay_x && (status = lay_out(x, l.x_rows, l.x_cols, x_pitch, type, x_planes, l.x_plane_pitch, l.x_plane, sms, st, what)) != DL_OK) return status;
    if (l.lay_w && (status = lay_out(w, outer, inner, inner, type, w_planes, l.w_plane_pitch, l.w_plane, sms, st, what)) != DL_OK) return status;
    const Operand ox = {l.lay_x ? x_planes : x, l.lay_x ? l.x_plane_pitch : x_pitch, l.x_plane, x_feature_major != 0};
    const Operand ow = {l.lay_w ? w_planes : w, l.lay_w ? l.w_plane_pitch : inner, l.w_plane, false};
    const bool rows_are_features = features_as_rows(batch, outer);
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
    const DenseEpilogue e = {y, bias, residual, slope, y_feature_major ? batch : outer, rows_are_features ? residual_feature : residual_batch,
                             rows_are_features ? residual_batch : residual_feature, type, act, rows_are_features, y_feature_major != 0};
    return launch_planes(p, plan, e, reinterpret_cast<float *>(workspace), sms, st, what);
}

namespace dl {

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
        if ((status = launch_planes(p, b.to_x, PlainEpilogue{gx, inner, type}, partial, sms, st, what)) != DL_OK) return status;
    }
    if (gw) {   // gz^T x, summed over the batch
        p.a = g;
        p.a.mn = g_feature_major == 0;
        p.b = {l.lay_x ? x_planes : x, l.lay_x ? l.x_plane_pitch : x_pitch, l.x_plane, x_feature_major == 0};
        p.m = outer;
        p.n = inner;
        p.k = batch;
        if ((status = launch_planes(p, b.to_w, PlainEpilogue{gw, inner, type}, partial, sms, st, what)) != DL_OK) return status;
    }
    return DL_OK;
}

// =============================================================== orthogonalisation ==============================================

namespace dl {

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

// X = G / max(|G|, eps) as pairs.
__global__ void __launch_bounds__(kThreads)
normalise_kernel(const Matrices all, int64_t rows, int64_t cols, const double *__restrict__ partial, int parts, double eps,
                 uint16_t *__restrict__ x, int64_t pitch, int64_t plane) {
    __shared__ float s_scale;
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
        const double norm = sqrt(sum);
        // a norm that is not finite (an infinite or undefined entry) makes the whole result undefined
        if (threadIdx.x == 0) s_scale = norm <= 1.7e308 ? (float)((double)kPairScale / (norm > eps ? norm : eps)) : __int_as_float(0x7fc00000);
    }
    __syncthreads();
    const float scale = s_scale;
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
        uint16_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_pair(v[j] * scale, hi[j], lo[j]);
        uint16_t *to = x + 2 * z * plane + row * pitch + col;
        *reinterpret_cast<ushort4 *>(to) = make_ushort4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<ushort4 *>(to + plane) = make_ushort4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// Results of the iteration as pairs: v = scale * sum (+ factor * the pair in `more`) (+ diagonal on the diagonal).
struct PairEpilogue {
    static constexpr int kPlanes = 2;
    uint16_t *out;
    const uint16_t *more;   // laid out as `out`; null: none
    int64_t pitch, plane;
    float scale, factor, diagonal;
    bool symmetric;

    __device__ __forceinline__ bool by_column(int row, int col) const { return symmetric && col / kMatmulRows < row / kMatmulRows; }
    __device__ __forceinline__ bool by_row(int row, int col) const { return !symmetric || col / kMatmulRows <= row / kMatmulRows; }
    template <int N>
    __device__ __forceinline__ void down(int z, int row, int col, const float (&sum)[N], int m, int valid) const {   // the mirrored values
        if (row >= m) return;
        const int64_t first = 2 * z * plane + (int64_t)col * pitch + row;
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = sum[j] * scale;
        if (more != nullptr) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j < valid) v[j] += factor * join_pair(more[first + j * pitch], more[first + j * pitch + plane]);
        }
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < valid) split_pair(v[j], out[first + j * pitch], out[first + j * pitch + plane]);
    }
    template <int N, int STEP>
    __device__ __forceinline__ void across(int z, int row, int col, const float (&sum)[N][4], int m, int) const {
        // rows are padded to whole units: the values behind the last one are written too, and read by nothing
        const int64_t first = 2 * z * plane + (int64_t)row * pitch + col;
        float v[N][4];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = sum[i][j] * scale + (row + i * STEP == col + j ? diagonal : 0.f);
        if (more != nullptr) {
            ushort4 hi[N], lo[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (row + i * STEP >= m) continue;
                hi[i] = *reinterpret_cast<const ushort4 *>(more + first + i * STEP * pitch);
                lo[i] = *reinterpret_cast<const ushort4 *>(more + first + i * STEP * pitch + plane);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (row + i * STEP >= m) continue;
                v[i][0] += factor * join_pair(hi[i].x, lo[i].x);
                v[i][1] += factor * join_pair(hi[i].y, lo[i].y);
                v[i][2] += factor * join_pair(hi[i].z, lo[i].z);
                v[i][3] += factor * join_pair(hi[i].w, lo[i].w);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (row + i * STEP >= m) continue;
            uint16_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) split_pair(v[i][j], hi[j], lo[j]);
            *reinterpret_cast<ushort4 *>(out + first + i * STEP * pitch) = make_ushort4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<ushort4 *>(out + first + i * STEP * pitch + plane) = make_ushort4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
};

// The last product: the result itself, or the weights' update w <- decay w - rate v.
struct OrthogonalEpilogue {
    static constexpr int kPlanes = 2;
    void *out;              // results behind each other; null: the weights of `all` are updated
    Matrices all;
    int64_t cols, matrix;   // values of a row, of a matrix
    const uint16_t *more;   // added, as in PairEpilogue
    int64_t pitch, plane;
    float scale, factor;
    float decay, rate;
    __device__ __forceinline__ bool by_column(int, int) const { return false; }
    __device__ __forceinline__ bool by_row(int, int) const { return true; }
    template <int N>
    __device__ __forceinline__ void down(int, int, int, const float (&)[N], int, int) const {}
    template <int N, int STEP>
    __device__ __forceinline__ void across(int z, int row, int col, const float (&sum)[N][4], int m, int valid) const {
        float *weight = out == nullptr ? all.weight[z] : nullptr;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row + i * STEP;
            if (r >= m) break;
            const int64_t at = r * cols + col;
            float v[4], w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = sum[i][j] * scale;
            if (more != nullptr) {
                const int64_t from = 2 * z * plane + r * pitch + col;
                const ushort4 hi = *reinterpret_cast<const ushort4 *>(more + from), lo = *reinterpret_cast<const ushort4 *>(more + from + plane);
                v[0] += factor * join_pair(hi.x, lo.x);
                v[1] += factor * join_pair(hi.y, lo.y);
                v[2] += factor * join_pair(hi.z, lo.z);
                v[3] += factor * join_pair(hi.w, lo.w);
            }
            if (weight != nullptr) {
                load4(weight, at, kFloat32, valid, w);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = w[j] * decay - rate * v[j];
                store4(weight, at, kFloat32, valid, v);
            } else {
                store4(out, z * matrix + at, all.type, valid, v);
            }
        }
    }
};

struct OrthogonalLayout {
    int64_t side, x_pitch, x_plane, s_pitch, s_plane;   // side: the smaller one
    bool tall;
    int parts;
    MatmulPlan gram, square, product;
    int64_t x_bytes, s_bytes, norm_bytes, partial_bytes;
    int64_t total() const { return 2 * x_bytes + 2 * s_bytes + norm_bytes + partial_bytes; }
};

static OrthogonalLayout orthogonal_layout(int64_t batch, int64_t rows, int64_t cols, bool light, int sms) {
    OrthogonalLayout l = {};
    l.tall = rows >= cols;
    l.side = l.tall ? cols : rows;
    l.x_pitch = padded(cols);
    l.x_plane = rows * l.x_pitch;
    l.s_pitch = padded(l.side);
    l.s_plane = l.side * l.s_pitch;
    l.parts = (int)(ceil_div(rows * cols, 4 * kThreads * 4) < 2 * sms ? ceil_div(rows * cols, 4 * kThreads * 4) : 2 * sms);
    l.gram = plan_matmul(l.side, l.side, l.tall ? rows : cols, batch, light ? 1 : 2, true, sms);
    l.square = plan_matmul(l.side, l.side, l.side, batch, 2, true, sms);
    l.product = plan_matmul(rows, cols, l.side, batch, light ? 1 : 2, false, sms);
    l.x_bytes = padded_bytes(batch * 2 * l.x_plane * 2);
    l.s_bytes = padded_bytes(batch * 2 * l.s_plane * 2);
    l.norm_bytes = padded_bytes(batch * l.parts * 8);
    l.partial_bytes = l.gram.partial_bytes;
    if (l.square.partial_bytes > l.partial_bytes) l.partial_bytes = l.square.partial_bytes;
    if (l.product.partial_bytes > l.partial_bytes) l.partial_bytes = l.product.partial_bytes;
    return l;
}

// steps times: S = X^T X (X X^T where X is wide), M = b S + c S^2, X = a X + X M (M X).  `last` takes the last product.
//
// Results of 22 bits (fp32, fp16): every product is one of pairs, and a X comes out of the product too, as the diagonal of M, since
// the pair of a X would have to be read again.  bf16 results have 8 bits, and the steps need no more than this: S from the first planes
// alone, which leaves the result 6e-4 off (relative, over random, low-rank and steeply falling spectra; rounding it to bf16 is
// 1.7e-3); S^2 from pairs; X M from the first planes, a X added as the pair that it is.  That last form matters: what is rounded away
// of X in a product with a I + b S + c S^2 grows by a factor of a in every step along directions of small singular values, 4e-2 in the
// end where X has few large ones; M alone is next to nothing along those.  All together 1.6e-3, half the products.
static int orthogonalise(const Matrices &all, int64_t batch, int64_t rows, int64_t cols, int steps, const float *coefficients, double eps,
                         const OrthogonalEpilogue &last, uint8_t *workspace, int sms, cudaStream_t st, const char *what) {
    const bool light = all.type == kBFloat16;
    const OrthogonalLayout l = orthogonal_layout(batch, rows, cols, light, sms);
    uint16_t *x = reinterpret_cast<uint16_t *>(workspace), *next = reinterpret_cast<uint16_t *>(workspace + l.x_bytes);
    uint16_t *gram = reinterpret_cast<uint16_t *>(workspace + 2 * l.x_bytes), *poly = reinterpret_cast<uint16_t *>(workspace + 2 * l.x_bytes + l.s_bytes);
    double *norms = reinterpret_cast<double *>(workspace + 2 * l.x_bytes + 2 * l.s_bytes);
    float *partial = reinterpret_cast<float *>(workspace + 2 * l.x_bytes + 2 * l.s_bytes + l.norm_bytes);
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
    for (int i = 0; i < steps; ++i) {
        const float a = coefficients[3 * i], b = coefficients[3 * i + 1], c = coefficients[3 * i + 2];
        p.a = p.b = {x, l.x_pitch, l.x_plane, l.tall};
        p.m = p.n = l.side;
        p.k = l.tall ? rows : cols;
        p.symmetric = true;
        p.planes = light ? 1 : 2;
        const PairEpilogue to_gram = {gram, nullptr, l.s_pitch, l.s_plane, once, 0.f, 0.f, true};
        if ((status = launch_planes(p, l.gram, to_gram, partial, sms, st, what)) != DL_OK) return status;
        p.a = p.b = {gram, l.s_pitch, l.s_plane, false};
        p.k = l.side;
        p.planes = 2;
        const PairEpilogue to_poly = {poly, gram, l.s_pitch, l.s_plane, c * once, b, light ? 0.f : a * kPairScale, true};
        if ((status = launch_planes(p, l.square, to_poly, partial, sms, st, what)) != DL_OK) return status;
        const Operand m = {poly, l.s_pitch, l.s_plane, false};
        p.a = l.tall ? Operand{x, l.x_pitch, l.x_plane, false} : m;
        p.b = l.tall ? m : Operand{x, l.x_pitch, l.x_plane, true};
        p.m = rows;
        p.n = cols;
        p.symmetric = false;
        p.planes = light ? 1 : 2;
        const uint16_t *more = light ? x : nullptr;
        if (i + 1 < steps) {
            const PairEpilogue to_next = {next, more, l.x_pitch, l.x_plane, once, a, 0.f, false};
            status = launch_planes(p, l.product, to_next, partial, sms, st, what);
        } else {
            OrthogonalEpilogue e = last;
            e.all = all;
            e.cols = cols;
            e.matrix = rows * cols;
            e.more = more;
            e.pitch = l.x_pitch;
            e.plane = l.x_plane;
            e.scale = twice;
            e.factor = a * once;
            status = launch_planes(p, l.product, e, partial, sms, st, what);
        }
        if (status != DL_OK) return status;
        uint16_t *done = x;
        x = next;
        next = done;
    }
    return DL_OK;
}

}  // namespace dl

// Matrices of so few columns stay as they are: their Gram matrix is iterated instead (gram_steps.cu).
static bool few_columns(int64_t cols) { return cols <= kGramColumns; }

extern "C" DL_API int64_t dl_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int type) {
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    if (few_columns(cols)) return gram_workspace_bytes(batch, batch * rows, current_sms());
    return orthogonal_layout(batch, rows, cols, type == kBFloat16, current_sms()).total();
}

static int check_steps(int steps, const float *coefficients, double eps, const char *what) {
    DL_REQUIRE(steps >= 1 && steps <= kMostSteps && coefficients, DL_ERR_INVALID_ARG, "%s: needs 1 to %d steps and their coefficients", what, kMostSteps);
    DL_REQUIRE(eps > 0, DL_ERR_INVALID_ARG, "%s: eps must be positive", what);
    return DL_OK;
}

extern "C" DL_API int dl_orthogonalize(const void *g, void *out, int64_t batch, int64_t rows, int64_t cols, int type, int steps,
                                       const float *coefficients, double eps, void *workspace, void *stream) {
    const char *what = "dl_orthogonalize";
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
        return launch_gram_steps(job, steps, coefficients, eps, reinterpret_cast<double *>(workspace), current_sms(), as_stream(stream), what);
    }
    Matrices all = {};
    all.g[0] = g;
    all.stride = rows * cols;
    all.type = type;
    OrthogonalEpilogue last = {};
    last.out = out;
    return orthogonalise(all, batch, rows, cols, steps, coefficients, eps, last, reinterpret_cast<uint8_t *>(workspace), current_sms(),
                         as_stream(stream), what);
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
            const int64_t bytes = orthogonal_layout(batch, rows, cols, false, sms).total();
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
            return launch_gram_steps(job, steps, coefficients, eps, reinterpret_cast<double *>(workspace), sms, st, what);
        },
        [&](Matrices &all, int64_t batch, int64_t rows, int64_t cols) {
            all.type = kFloat32;
            all.keep = keep;
            all.nesterov = toward;
            OrthogonalEpilogue last = {};
            last.decay = decay;
            last.rate = rate(rows, cols);
            return orthogonalise(all, batch, rows, cols, steps, coefficients, eps, last, reinterpret_cast<uint8_t *>(workspace), sms, st, what);
        });
}
