// Matrix products on the tensor cores with an epilogue: D[m][n] = sum_k A[m][k] B[n][k], per matrix of a batch.
//
// Operands are one to three planes of 16-bit values whose sum is the operand, so that results can be as exact as 32-bit arithmetic:
//   1 plane   fp16 or bf16 values as they are;
//   2 planes  fp16 pairs hi + lo, 22 bits: hi hi + (hi lo + lo hi), 3 products; for operands of known size (the value is kept
//             times 2^12, so that lo is no subnormal for values above 2^-14);
//   3 planes  bf16 triples, all 24 bits of an fp32 in its whole range: 6 products, those below 2^-24 left out.
// A running sum in the tensor cores cuts off what is below its last bit, always towards zero: an error of about 1e-8 for every 16 values
// (measured: 6e-7 after 800, 1.2e-6 after 2000, where 32-bit sums of rounded steps have 2e-7 and 4e-7).  So the sums of planes are
// taken out of tensor memory every steps_per_sum steps and added up in the epilogue's registers, and the small products have a sum
// of their own.
//
// What bounds it.  Large products: the tensor cores.  8192 x 4096 x 4096 bf16 with the epilogue of a dense layer 207 us, 1330 TFLOP/s (a
// library's plain product, 4096 values a side and more, has 1627 in a burst); 4096 x 4096 x 4096 of pairs 336 us, three products each:
// 1230 TFLOP/s.  Pairs of SMs share a tile of 256 x 256 there, since a step's copies of 128 x 128 take as long as its products (60 bytes
// a clock and SM).  Products of a few tiles per SM: their latency, about 5 us until the sums of the first steps are there and 5 to 10 us
// of epilogue that no next tile hides; 1024 x 1024 x 1024 of pairs 20 us.
#pragma once

#include "matmul_values.cuh"
#include "tensor_core.cuh"

namespace dl {

struct Operand {       // rows x k, or k x rows where mn: the rows of the result are contiguous
    const void *base;
    int64_t pitch, plane;  // in values: between rows in memory, planes
    bool mn;
};

struct MatmulShape {
    int32_t m, n, batch, planes_z;        // planes_z: planes per matrix in the maps
    int32_t tiles_m, tiles_n, splits, k_steps, steps_per_split, steps_per_sum;
    int32_t per_matrix;                   // tiles of a matrix (one split)
    int32_t tiles;                        // of all matrices and splits
    uint32_t a_mn, b_mn, instruction;
    int32_t symmetric;                    // only tiles that reach to or below the diagonal are computed
};

#ifdef __CUDACC__
// -- 16-bit planes --------------------------------------------------------------------------------------------------------------

constexpr float kPairScale = 4096.f;

// Two values as pairs, packed: conversions of two values at a time run at several times the rate of single ones.  An infinite value
// leaves an undefined lower half (inf - inf), which is what the products would give.
__device__ __forceinline__ void split_two(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 back = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - back.x, b - back.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ float join_pair(uint16_t hi, uint16_t lo) { return __half2float(__ushort_as_half(hi)) + __half2float(__ushort_as_half(lo)); }

// The nearest bf16 at each step: exact for every fp32 from 2^-110 on.  Infinities and NaN go into the first plane alone; values that would round to
// infinity are cut off.
__device__ __forceinline__ void split_triple(float x, uint16_t &hi, uint16_t &mid, uint16_t &lo) {
    const uint32_t bits = __float_as_uint(x);
    if ((bits & 0x7f800000u) == 0x7f800000u) {
        hi = (uint16_t)(bits >> 16) | (uint16_t)((bits & 0x007fffffu) ? 0x40 : 0);
        mid = lo = 0;
        return;
    }
    __nv_bfloat16 h = __float2bfloat16_rn(x);
    hi = __bfloat16_as_ushort(h);
    if ((hi & 0x7f80u) == 0x7f80u) hi = (uint16_t)(bits >> 16);
    const float rest = x - __uint_as_float((uint32_t)hi << 16);
    h = __float2bfloat16_rn(rest);
    mid = __bfloat16_as_ushort(h);
    lo = __bfloat16_as_ushort(__float2bfloat16_rn(rest - __bfloat162float(h)));
}

// -- the kernel -----------------------------------------------------------------------------------------------------------------

constexpr int kMatmulRows = 128;     // of a tile
constexpr int kPieceColumns = 16;    // columns of which sums are kept together where a product is split
constexpr int kSlotBytes = 2048;     // 32 rows of 64 bytes
constexpr int kStageBytes = 2 * kSlotBytes;   // shared memory of an epilogue warp

struct NothingAhead {};

// An epilogue takes pieces of 32 rows (lane = row) and kColumns columns from registers: `begin` says where the first piece of a warp's
// share of a tile lies (row, col: of its first value), `piece` takes the one `across` columns further.  What it has to read for that
// `fetch` asks for beforehand -- the first one's while the products are still running, the others' a piece ahead: a read takes 3000
// clocks when all SMs read at a time.
//
// Results leave by way of shared memory in tiles of 32 rows of 64 bytes, a slot each: written as the lanes have them, rows or columns as
// rows, and read back with 8 rows of four lanes at a time, so that a warp's store is of eight whole 64-byte rows.  The swizzle puts the
// 16-byte unit j of row r at j ^ (r / 2 % 4): 8 lanes meet no bank twice either way.  (Tiled copies out of the slots instead made the
// 4096 x 4096 iteration 5.8 ms for 4.0: the unit that does them has the operands' copies to do, 60 bytes a clock of them.)
__device__ __forceinline__ void slot_row(uint8_t *slot, int lane, const uint32_t (&v)[16]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4 *>(slot + lane * 64 + ((j ^ (lane / 2 % 4)) << 4)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
__device__ __forceinline__ void slot_read_row(const uint8_t *slot, int lane, uint4 (&u)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = *reinterpret_cast<const uint4 *>(slot + lane * 64 + ((j ^ (lane / 2 % 4)) << 4));
}
__device__ __forceinline__ void slot_column(uint8_t *slot, int lane, int column, uint16_t v) {
    *reinterpret_cast<uint16_t *>(slot + column * 64 + ((lane / 8 ^ (column / 2 % 4)) << 4) + lane % 8 * 2) = v;
}
// Unit lane % 4 of row lane / 4 + 8 i.
__device__ __forceinline__ uint4 *slot_unit(uint8_t *slot, int lane, int i) {
    const int row = lane / 4 + 8 * i;
    return reinterpret_cast<uint4 *>(slot + row * 64 + ((lane % 4 ^ (row / 2 % 4)) << 4));
}

// Where a result cannot be stored that way: 32 rows of 16 columns turned into quads, lane l having rows l / 4 + 8 i and columns
// 4 (l % 4) .. + 3.
constexpr int kPiecePitch = kPieceColumns + 4;   // floats: 16-byte rows, 8 lanes on 8 banks
static_assert(32 * kPiecePitch * 4 <= kStageBytes, "a piece fits");
__device__ __forceinline__ void piece_quads(uint8_t *shared, int lane, const float (&v)[kPieceColumns], float (&q)[4][4]) {
    float *stage = reinterpret_cast<float *>(shared);
#pragma unroll
    for (int c = 0; c < kPieceColumns; c += 4)
        *reinterpret_cast<float4 *>(stage + lane * kPiecePitch + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 f = *reinterpret_cast<const float4 *>(stage + (lane / 4 + 8 * i) * kPiecePitch + lane % 4 * 4);
        q[i][0] = f.x; q[i][1] = f.y; q[i][2] = f.z; q[i][3] = f.w;
    }
    __syncwarp();
}

// Warps 0 .. 7: epilogue, one lane per row, two warps to the same rows; then one for the copies, one for the products, two idle: the
// registers that the epilogue does not leave to the others are handed out in groups of four warps.
template <int PLANES, int COLUMNS, bool PAIR>
struct MatmulConfig {
    static constexpr int kWarps = 8;
    static constexpr int kThreadsAll = (kWarps + 4) * 32;   // 384
    static constexpr int kTileRows = PAIR ? 2 * kMatmulRows : kMatmulRows;
    static constexpr int kOwnColumns = PAIR ? COLUMNS / 2 : COLUMNS;           // rows of B that a CTA copies
    static constexpr int kShare = COLUMNS / (kWarps / 4);                      // columns of an epilogue warp
    static constexpr int kStepBytes = PLANES * (kMatmulRows + kOwnColumns) * kChunk * 2;   // of a CTA
    static constexpr int kStagingBytes = kWarps * kStageBytes;
    static constexpr int kFit = (232448 - 1024 - 256 - kStagingBytes) / kStepBytes;
    static constexpr int kStages = kFit < 6 ? kFit : 6;
    static constexpr int kSums = PLANES > 1 && COLUMNS <= 128 ? 2 : 1;         // accumulators: of the large products, of the small ones
    static constexpr int kTensorColumns = 2 * kSums * COLUMNS;                 // two of each: one is filled while the other is read
    static constexpr int kSharedBytes = kStages * kStepBytes + kStagingBytes + 1024 + 256;
    static_assert(kStages >= 2, "the ring does not fit");
    static_assert((kTensorColumns & (kTensorColumns - 1)) == 0 && kTensorColumns >= 32 && kTensorColumns <= 512, "tensor memory");
};

struct Tile {
    int matrix, split, index;     // of the matrix' tiles
    int row, col;                 // first ones
};

template <int ROWS, int COLUMNS>
__device__ __forceinline__ Tile tile_of(int id, const MatmulShape &s) {
    Tile t;
    const int all = s.per_matrix * s.splits;
    t.matrix = id / all;
    id -= t.matrix * all;
    t.split = id / s.per_matrix;
    id -= t.split * s.per_matrix;
    t.index = id;
    int mi, ni;
    if (s.symmetric) {
        mi = 0;
        for (;;) {
            const int across = min(s.tiles_n, ((mi + 1) * ROWS + COLUMNS - 1) / COLUMNS);
            if (id < across) break;
            id -= across;
            ++mi;
        }
        ni = id;
    } else {
        // bands of 8 tiles down, so that the tiles that run at a time share operands in L2
        const int band = 8 * s.tiles_n, first = id / band * 8, high = min(8, s.tiles_m - first), in_band = id - id / band * band;
        mi = first + in_band % high;
        ni = in_band / high;
    }
    t.row = mi * ROWS;
    t.col = ni * COLUMNS;
    return t;
}

static __device__ int g_matmul_async_error = 0;   // set when a bounded wait ran out; read by matmul_async_error()

// Persistent: every CTA takes tiles blockIdx.x, blockIdx.x + gridDim.x, ...; the copies run ahead across tiles, and the epilogue of a
// tile runs beside the products of the next where tensor memory holds two.  All waits are bounded; when one runs out, the error flag is
// raised and every role leaves, the copies that are in flight waited for.
template <int PLANES, int COLUMNS, bool PAIR, class Epilogue>
__global__ void __launch_bounds__(MatmulConfig<PLANES, COLUMNS, PAIR>::kThreadsAll, 1)
matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const MatmulShape s, const __grid_constant__ Epilogue epilogue) {
    using Config = MatmulConfig<PLANES, COLUMNS, PAIR>;
    constexpr int kStages = Config::kStages;
    constexpr int kPlaneA = kMatmulRows * kChunk * 2, kPlaneB = Config::kOwnColumns * kChunk * 2;
    extern __shared__ uint8_t s_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *staging = ring + kStages * Config::kStepBytes;
    uint64_t *full = reinterpret_cast<uint64_t *>(staging + Config::kStagingBytes), *empty = full + kStages, *sums_full = empty + kStages,
             *sums_empty = sums_full + 2, *drained = sums_empty + 2;
    uint32_t *s_tensor = reinterpret_cast<uint32_t *>(drained + 1);
    volatile uint32_t *s_failed = s_tensor + 1;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const int first_tile = PAIR ? blockIdx.x / 2 : blockIdx.x, tile_step = PAIR ? gridDim.x / 2 : gridDim.x;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(sums_full + i, 1);
            mbar_init(sums_empty + i, PAIR ? 2 * Config::kWarps : Config::kWarps);
        }
        mbar_init(drained, 1);
        *s_failed = 0;
        mbar_fence_init();
    }
    if (warp == Config::kWarps + 1) tensor_alloc<PAIR>(s_tensor, Config::kTensorColumns);
    if (warp == Config::kWarps && lane == 0) {
        map_prefetch(&map_a);
        map_prefetch(&map_b);
    }
    tensor_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();   // the other one's barriers are there
    tensor_fence_after();
    const uint32_t tensor = *s_tensor;
    grid_dependency_wait();
    grid_dependents_launch();

    // 168 registers a thread at the launch, 384 threads: 216 for the epilogue's 256 and 72 for the other 128 are as many
    if (warp >= Config::kWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == Config::kWarps && lane == 0) {
            int stage = 0, used = 0;   // used: stages with a copy issued
            uint32_t phase = 0;
            bool ok = true;
            for (int id = first_tile; id < s.tiles && ok; id += tile_step) {
                const Tile t = tile_of<Config::kTileRows, COLUMNS>(id, s);
                const int first = t.split * s.steps_per_split, last = min(s.k_steps, first + s.steps_per_split);
                for (int step = first; step < last; ++step) {
                    ok = mbar_wait(empty + stage, phase ^ 1) && !*s_failed;
                    if (!ok) break;
                    if (rank == 0) mbar_arrive_expect_tx(full + stage, PAIR ? 2 * Config::kStepBytes : Config::kStepBytes);
                    const uint32_t bar = PAIR ? cluster_address(full + stage, 0) : smem_addr(full + stage);
                    uint8_t *at = ring + stage * Config::kStepBytes;
                    const int k = step * kChunk;
#pragma unroll 1
                    for (int p = 0; p < PLANES; ++p) {
                        const int z = t.matrix * s.planes_z + p;
                        const int row = t.row + (int)rank * kMatmulRows;
                        if (!s.a_mn) {
                            tile_load<PAIR>(at, &map_a, k, row, z, bar);
                        } else {
#pragma unroll
                            for (int c = 0; c < kMatmulRows / kChunk; ++c) tile_load<PAIR>(at + c * kChunkBytes, &map_a, row + c * kChunk, k, z, bar);
                        }
                        at += kPlaneA;
                    }
#pragma unroll 1
                    for (int p = 0; p < PLANES; ++p) {
                        const int z = t.matrix * s.planes_z + p;
                        const int col = t.col + (int)rank * Config::kOwnColumns;
                        if (!s.b_mn) {
                            tile_load<PAIR>(at, &map_b, k, col, z, bar);
                        } else {
#pragma unroll
                            for (int c = 0; c < Config::kOwnColumns / kChunk; ++c) tile_load<PAIR>(at + c * kChunkBytes, &map_b, col + c * kChunk, k, z, bar);
                        }
                        at += kPlaneB;
                    }
                    used = max(used, stage + 1);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok) {
                *s_failed = 1;
                g_matmul_async_error = 1;
            }
            // nothing of a CTA's copies is in flight when it ends: the latest copy into each stage (in a pair the first CTA's barriers
            // count both's, and the second CTA does not end before the first)
            if (rank == 0)
                for (int i = 0; i < used; ++i) mbar_wait(full + i, i < stage ? phase : phase ^ 1);
            else if (!ok)   // the first CTA may have given up before it counted these: they land within microseconds
                for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        }
        if (warp == Config::kWarps + 1 && lane == 0 && rank == 0) {
            int stage = 0, buffer = 0;
            uint32_t phase = 0, buffer_phase = 0;
            bool ok = true;
            const uint32_t a_step = s.a_mn ? 2048 >> 4 : 32 >> 4, b_step = s.b_mn ? 2048 >> 4 : 32 >> 4;
            for (int id = first_tile; id < s.tiles && ok; id += tile_step) {
                const Tile t = tile_of<Config::kTileRows, COLUMNS>(id, s);
                const int first = t.split * s.steps_per_split, last = min(s.k_steps, first + s.steps_per_split);
                for (int block = first; block < last && ok; block += s.steps_per_sum) {
                    ok = mbar_wait(sums_empty + buffer, buffer_phase ^ 1) && !*s_failed;
                    if (!ok) break;
                    tensor_fence_after();
                    const uint32_t large = tensor + buffer * Config::kSums * COLUMNS, small = large + (Config::kSums - 1) * COLUMNS;
                    const int end = min(last, block + s.steps_per_sum);
                    for (int step = block; step < end; ++step) {
                        ok = mbar_wait(full + stage, phase) && !*s_failed;
                        if (!ok) break;
                        tensor_fence_after();
                        const uint32_t at = smem_addr(ring + stage * Config::kStepBytes);
                        const uint64_t a = operand_descriptor(at), b = operand_descriptor(at + PLANES * kPlaneA);
                        const auto product = [&](int pa, int pb, uint32_t sum, bool fresh) {
                            const uint64_t from_a = a + pa * (kPlaneA >> 4), from_b = b + pb * (kPlaneB >> 4);
#pragma unroll
                            for (int k = 0; k < kChunk / 16; ++k)
                                tensor_multiply<PAIR>(sum, from_a + k * a_step, from_b + k * b_step, s.instruction, !(fresh && k == 0));
                        };
                        const bool fresh = step == block;
                        // the smallest products first: where they share a sum with the large ones, it cuts off little of them
                        if (PLANES > 2) {
                            product(1, 1, small, fresh);
                            product(0, 2, small, false);
                            product(2, 0, small, false);
                        }
                        if (PLANES > 1) {
                            product(0, 1, small, fresh && PLANES == 2);
                            product(1, 0, small, false);
                        }
                        product(0, 0, large, fresh && (PLANES == 1 || Config::kSums == 2));
                        tensor_commit<PAIR>(empty + stage);
                        if (++stage == kStages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                    if (!ok) break;
                    tensor_commit<PAIR>(sums_full + buffer);
                    buffer ^= 1;
                    buffer_phase ^= buffer == 0;
                }
            }
            if (!ok) {
                *s_failed = 1;
                g_matmul_async_error = 1;
                tensor_commit<PAIR>(drained);   // tensor memory is given back when nothing writes it any more
                mbar_wait(drained, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        constexpr int kSpan = Epilogue::kColumns, kShare = Config::kShare;
        constexpr bool kKeep = PLANES > 1;   // sums of several blocks, added up in registers
        uint8_t *mine = staging + warp * kStageBytes;
        const int quarter = warp % 4, from = warp / 4 * kShare;   // a warp reads the lanes of its number modulo 4
        int buffer = 0;
        uint32_t buffer_phase = 0;
        bool ok = true;
        for (int id = first_tile; id < s.tiles && ok; id += tile_step) {
            const Tile t = tile_of<Config::kTileRows, COLUMNS>(id, s);
            const int first = t.split * s.steps_per_split, last = min(s.k_steps, first + s.steps_per_split);
            const int row0 = t.row + (int)rank * kMatmulRows + quarter * 32;
            const auto place = epilogue.begin(t, s, row0, t.col + from, lane);
            typename Epilogue::Ahead ahead;
            epilogue.fetch(place, 0, lane, ahead);
            const auto finish = [&](const float (&v)[kSpan], int across) {
                if (t.col + from + across >= s.n && !Epilogue::kWholeTiles) return;
                const typename Epilogue::Ahead now = ahead;
                if (across + kSpan < kShare) epilogue.fetch(place, across + kSpan, lane, ahead);
                epilogue.piece(place, across, v, now, mine, lane);
            };
            float kept[kKeep ? kShare : 1];
#pragma unroll
            for (int c = 0; c < (kKeep ? kShare : 1); ++c) kept[c] = 0.f;
            for (int block = first; block < last; block += s.steps_per_sum) {
                ok = mbar_wait(sums_full + buffer, buffer_phase) && !*s_failed;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tensor_fence_after();
                const uint32_t sums = tensor + buffer * Config::kSums * COLUMNS + from + ((uint32_t)quarter * 32 << 16);
                if constexpr (kKeep) {
                    // 64 values on their way at a time
                    constexpr int kTake = Config::kSums == 2 ? 32 : kShare < 64 ? kShare : 64;
#pragma unroll
                    for (int c0 = 0; c0 < kShare; c0 += kTake) {
                        uint32_t one[32], other[32];
                        tensor_read32(sums + c0, one);
                        if (Config::kSums == 2) tensor_read32(sums + COLUMNS + c0, other);
                        else if (kTake == 64) tensor_read32(sums + c0 + 32, other);
                        tensor_read_wait();
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (Config::kSums == 2) {
                                kept[c0 + c] += __uint_as_float(one[c]) + __uint_as_float(other[c]);
                            } else {
                                kept[c0 + c] += __uint_as_float(one[c]);
                                if (kTake == 64) kept[c0 + 32 + c] += __uint_as_float(other[c]);
                            }
                        }
                    }
                } else {
                    // the next 32 columns are on their way while these are worked on
                    uint32_t bits[32];
                    tensor_read32(sums, bits);
                    tensor_read_wait();
#pragma unroll 1
                    for (int c0 = 0; c0 < kShare && (t.col + from + c0 < s.n || Epilogue::kWholeTiles); c0 += 32) {
                        float v[32 / kSpan][kSpan];
#pragma unroll
                        for (int c = 0; c < 32; ++c) v[c / kSpan][c % kSpan] = __uint_as_float(bits[c]);
                        if (c0 + 32 < kShare) tensor_read32(sums + c0 + 32, bits);
#pragma unroll
                        for (int h = 0; h < 32 / kSpan; ++h) finish(v[h], c0 + h * kSpan);
                        tensor_read_wait();
                    }
                }
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_in_cluster(cluster_address(sums_empty + buffer, 0));
                    else mbar_arrive(sums_empty + buffer);
                }
                buffer ^= 1;
                buffer_phase ^= buffer == 0;
            }
            if constexpr (kKeep) {
                if (ok) {
#pragma unroll(kSpan == 32 ? 4 : 1)
                    for (int c0 = 0; c0 < kShare; c0 += kSpan) {
                        float v[kSpan];
#pragma unroll
                        for (int c = 0; c < kSpan; ++c) v[c] = kept[kSpan == 32 ? c0 + c : c];
                        if (kSpan != 32) {   // the registers move up: one copy of the epilogue's code
#pragma unroll
                            for (int c = 0; c + kSpan < kShare; ++c) kept[c] = kept[c + kSpan];
                        }
                        finish(v, c0);
                    }
                }
            }
        }
        if (!ok) {
            *s_failed = 1;
            g_matmul_async_error = 1;
        }
    }
    __syncwarp();
    tensor_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();   // neither frees or leaves what the other one still uses
    if (warp == Config::kWarps + 1) tensor_free<PAIR>(tensor, Config::kTensorColumns);
}

// Sums of a product that was split along k, whole tiles of them, each piece as its lanes have it; matmul_join_kernel adds them up in the
// order of the splits.
struct StorePartial {
    static constexpr bool kWholeTiles = true;
    static constexpr int kColumns = kPieceColumns;
    float *out;
    int tile_rows, columns;
    struct Place {
        float4 *to;
    };
    // pieces of a tile, down and then across
    __device__ __forceinline__ Place begin(const Tile &t, const MatmulShape &s, int row, int col, int lane) const {
        const int64_t tile = (int64_t)(t.split * s.batch + t.matrix) * s.per_matrix + t.index;
        const int piece = (row - t.row) / 32 + (col - t.col) / kPieceColumns * (tile_rows / 32);
        return {reinterpret_cast<float4 *>(out + tile * tile_rows * columns) + piece * (8 * kPieceColumns) + lane};
    }
    using Ahead = NothingAhead;
    __device__ __forceinline__ void fetch(const Place &, int, int, Ahead &) const {}
    __device__ __forceinline__ void piece(const Place &p, int across, const float (&v)[kColumns], const Ahead &, uint8_t *, int) const {
        float4 *to = p.to + across / kPieceColumns * (tile_rows / 32) * (8 * kPieceColumns);
#pragma unroll
        for (int c = 0; c < kPieceColumns; c += 4) to[c * 8] = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
    }
};

template <int ROWS, int COLUMNS, class Epilogue>
__global__ void __launch_bounds__(kThreads)
matmul_join_kernel(const float *__restrict__ partial, const MatmulShape s, const __grid_constant__ Epilogue epilogue) {
    __shared__ __align__(1024) uint8_t s_stage[kThreads / 32][kStageBytes];
    grid_dependency_wait();
    grid_dependents_launch();
    constexpr int kDown = ROWS / 32, kTake = Epilogue::kColumns, kPieces = kDown * COLUMNS / kTake;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t tiles = (int64_t)s.per_matrix * s.batch;
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + warp; i < tiles * kPieces; i += (int64_t)gridDim.x * (kThreads / 32)) {
        const int64_t tile = i / kPieces;
        const int piece = (int)(i - tile * kPieces), matrix = (int)(tile / s.per_matrix);
        const Tile t = tile_of<ROWS, COLUMNS>((int)(tile - (int64_t)matrix * s.per_matrix) + matrix * s.per_matrix * s.splits, s);
        const int row = t.row + piece % kDown * 32, col = t.col + piece / kDown * kTake;
        if (row >= s.m || col >= s.n) continue;
        const float4 *from = reinterpret_cast<const float4 *>(partial + tile * ROWS * COLUMNS) +
                             (piece % kDown + piece / kDown * (kTake / kPieceColumns) * kDown) * (8 * kPieceColumns) + lane;
        const int64_t split = tiles * ROWS * COLUMNS / 4;
        const auto place = epilogue.begin(t, s, row, col, lane);
        typename Epilogue::Ahead ahead;
        epilogue.fetch(place, 0, lane, ahead);
        float v[kTake] = {};
        for (int sp = 0; sp < s.splits; ++sp, from += split) {
#pragma unroll
            for (int c = 0; c < kTake; c += 4) {
                const float4 f = from[(c % kPieceColumns) * 8 + c / kPieceColumns * (kDown * 8 * kPieceColumns)];
                v[c] += f.x; v[c + 1] += f.y; v[c + 2] += f.z; v[c + 3] += f.w;
            }
        }
        epilogue.piece(place, 0, v, ahead, s_stage[warp], lane);
    }
}
#endif  // __CUDACC__

}  // namespace dl
