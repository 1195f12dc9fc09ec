// Launching the matrix products of matmul.cuh.
#pragma once

#include <atomic>

#include "matmul.cuh"
#include "matmul_plan.h"

namespace dl {

static int matmul_error_flag() {
    int flag = 0;
    if (cudaMemcpyFromSymbol(&flag, g_matmul_async_error, sizeof(int)) != cudaSuccess) {
        cudaGetLastError();
        return -1;
    }
    return flag;
}

struct Product {
    Operand a, b;
    int64_t m, n, k, batch;
    int planes, planes_z;   // multiplied; per matrix in memory
    bool bfloat, symmetric;
    bool exact;   // sums are taken out of tensor memory every so often
};

// `own`: rows of it that a CTA copies for a tile, at once where they are K-major.
static bool map_operand(CUtensorMap *map, const Operand &o, const Product &p, int64_t rows, int own) {
    const int64_t inner = o.mn ? rows : p.k, outer = o.mn ? p.k : rows;
    return make_tile_map(map, o.base, p.bfloat, inner, outer, p.planes_z * p.batch, o.pitch * 2, o.plane * 2, o.mn ? kChunk : own);
}

template <int PLANES, int COLUMNS, bool PAIR, class Epilogue>
static int launch_tiles(const MatmulShape &shape, const CUtensorMap &a, const CUtensorMap &b, const Epilogue &epilogue, int sms,
                        cudaStream_t st, const char *what) {
    using Config = MatmulConfig<PLANES, COLUMNS, PAIR>;
    auto kernel = matmul_kernel<PLANES, COLUMNS, PAIR, Epilogue>;
    // once for each kernel and device: the call takes the host longer than the rest of a launch
    static std::atomic<uint64_t> allowed{0};
    int device = 0;
    cudaGetDevice(&device);
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if ((allowed.load(std::memory_order_relaxed) & bit) == 0) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Config::kSharedBytes) != cudaSuccess) return launch_status(what);
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
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

template <int PLANES, int COLUMNS, bool PAIR, class Epilogue>
static int launch_splits(const MatmulShape &s, const CUtensorMap &a, const CUtensorMap &b, const Epilogue &epilogue, float *partial, int sms,
                         cudaStream_t st, const char *what) {
    if (s.splits == 1) return launch_tiles<PLANES, COLUMNS, PAIR>(s, a, b, epilogue, sms, st, what);
    constexpr int kRows = PAIR ? 2 * kMatmulRows : kMatmulRows;
    const int status = launch_tiles<PLANES, COLUMNS, PAIR>(s, a, b, StorePartial{partial, kRows, COLUMNS}, sms, st, what);
    if (status != DL_OK) return status;
    int64_t blocks = ceil_div((int64_t)s.per_matrix * s.batch * (kRows / 32) * (COLUMNS / kPieceColumns), kThreads / 32);
    if (blocks > 8 * sms) blocks = 8 * sms;
    launch_dependent(true, matmul_join_kernel<kRows, COLUMNS, Epilogue>, dim3((unsigned)blocks), dim3(kThreads), 0, st, (const float *)partial, s,
                     epilogue);
    return launch_status(what);
}

// One product with its epilogue; `partial`: plan.partial_bytes.
template <int PLANES, class Epilogue>
static int launch_product(const Product &p, const MatmulPlan &plan, const Epilogue &epilogue, float *partial, int sms, cudaStream_t st,
                          const char *what) {
    CUtensorMap a, b;
    if (!map_operand(&a, p.a, p, p.m, kMatmulRows) || !map_operand(&b, p.b, p, p.n, plan.pair ? plan.columns / 2 : plan.columns))
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
    s.steps_per_sum = PLANES > 1 && p.exact ? 2 : s.k_steps;   // one plane: nothing adds blocks up
    s.symmetric = p.symmetric;
    const int64_t per_matrix = tiles_of(p.m, p.n, rows, plan.columns, p.symmetric), tiles = per_matrix * s.splits * p.batch;
    if (tiles > INT32_MAX / 2) return fail(DL_ERR_TOO_LARGE, "%s: too many tiles", what);
    s.per_matrix = (int32_t)per_matrix;
    s.tiles = (int32_t)tiles;
    s.a_mn = p.a.mn;
    s.b_mn = p.b.mn;
    s.instruction = instruction_descriptor(p.bfloat, p.a.mn, p.b.mn, rows, plan.columns);
    if (plan.pair) return launch_splits<PLANES, 256, true>(s, a, b, epilogue, partial, sms, st, what);
    if (plan.columns == 64) return launch_splits<PLANES, 64, false>(s, a, b, epilogue, partial, sms, st, what);
    if (plan.columns == 128) return launch_splits<PLANES, 128, false>(s, a, b, epilogue, partial, sms, st, what);
    return fail(DL_ERR_INVALID_ARG, "%s: no such tile", what);
}

// Values of a row of planes that the library lays out: whole units of 16 bytes.
static inline int64_t padded(int64_t n) { return ceil_div(n, 8) * 8; }
static inline int64_t padded_bytes(int64_t n) { return ceil_div(n, 256) * 256; }

}  // namespace dl
