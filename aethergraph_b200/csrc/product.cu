// Product of 8-bit rows (e4m3, a scale per 128 columns of a row) with 8-bit weights (a scale per
// 128 x 128 block), the rows in order or by id: the gather of a feature store that multiplies
// what it reads.  No counterpart in the reference.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "internal.h"

namespace ag {

namespace {

__device__ uint32_t g_rows_error;  // sticky error bits of this device's products that are no store's (ag_rows_check)

struct ProductArgs {
    const uint8_t *codes, *weight;
    const float *scales, *weight_scales;
    const void *ids;
    const float *bias;
    void *out;
    uint32_t *error;  // the store's sticky error bits, or null
    uint64_t rows, held, code_stride, weight_stride, out_stride;
    uint32_t dim, out_dim, blocks;  // blocks: of 128 columns
    int ids64, out_dtype;
};

__device__ __forceinline__ void raise(const ProductArgs &a, uint32_t bits) { atomicOr(a.error ? a.error : &g_rows_error, bits); }

// Row of the codes that output row m takes; `held` where its id names none.
__device__ __forceinline__ uint64_t source_row(const ProductArgs &a, uint64_t m) {
    if (!a.ids) return m;
    const uint64_t id = a.ids64 ? (uint64_t)((const int64_t *)a.ids)[m] : (uint64_t)((const uint32_t *)a.ids)[m];
    if (id < a.held) return id;
    raise(a, kErrBadId);
    return a.held;
}

__device__ __forceinline__ void store_out(const ProductArgs &a, uint64_t m, uint32_t n, float v) {
    if (a.out_dtype == AG_F32) ((float *)a.out)[m * a.out_stride + n] = v;
    else if (a.out_dtype == AG_F16) ((__half *)a.out)[m * a.out_stride + n] = __float2half_rn(v);
    else ((__nv_bfloat16 *)a.out)[m * a.out_stride + n] = __float2bfloat16_rn(v);
}

// 16 codes of a row from column c on, a multiple of 16; columns past `dim` are zeros.
__device__ __forceinline__ void load_codes(const uint8_t *row, uint32_t c, uint32_t dim, float v[16]) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (c + 16 <= dim) {
        const uint4 q = *(const uint4 *)(row + c);
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {  // the last row's memory may end with its last column
        for (uint32_t i = 0; c + i < dim; ++i) w[i >> 2] |= (uint32_t)row[c + i] << (8 * (i & 3));
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i >> 2] >> (8 * (i & 3))), __NV_E4M3);
        const float2 f = __half22float2(__half2(h));
        v[i] = f.x;
        v[i + 1] = f.y;
    }
}

constexpr int kDotThreads = 256;
// Beyond this many rows the tensor-core tiles are faster: 1024 x 1024 1, 2, 4, 8 rows 3.6, 4.2, 5.3, 5.8 us this way,
// 5.1, 5.1, 5.0, 5.2 the other; 2048 x 1024 4.8, 5.8, 7.8, 8.2 and 6.5, 6.5, 6.8, 6.8; 256 x 256 3.1, 3.2, 3.9, 3.8 and 4.0, 3.8, 3.8, 4.1.
constexpr int kFewRows = 3;

// Few rows: a warp per column of the output, a lane 16 codes a turn, which lie in one scale
// block.  The weights are all there is to read; 1 x 1024 x 1024: 3.6 us, of which launch and one dependent load are most.
__global__ void __launch_bounds__(kDotThreads)
k_product_dot(ProductArgs a) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t n = blockIdx.x * (kDotThreads / 32) + (threadIdx.x >> 5);
    if (n >= a.out_dim) return;
    uint64_t src[kFewRows];
    float acc[kFewRows];
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
        src[r] = r < a.rows ? source_row(a, r) : a.held;
        acc[r] = 0.f;
    }
    for (uint32_t c = lane * 16; c < a.dim; c += 512) {
        float w[16];
        load_codes(a.weight + (uint64_t)n * a.weight_stride, c, a.dim, w);
        const float ws = a.weight_scales[(uint64_t)(n / kF8Block) * a.blocks + c / kF8Block];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            if (src[r] == a.held) continue;
            float v[16], dot = 0.f;
            load_codes(a.codes + src[r] * a.code_stride, c, a.dim, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) dot += v[i] * w[i];
            acc[r] += dot * (a.scales[src[r] * a.blocks + c / kF8Block] * ws);
        }
    }
#pragma unroll
    for (int r = 0; r < kFewRows; ++r) {
        for (int o = 16; o > 0; o /= 2) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (lane == 0 && r < a.rows) store_out(a, r, n, src[r] == a.held ? 0.f : acc[r] + (a.bias ? a.bias[n] : 0.f));
    }
}

// ------------------------------------------------------ tensor-core tiles --
// A tile of 128 rows x BN output columns per turn of a persistent block, K in steps of 128 bytes,
// which is one scale block: the tensor cores add up the 128 products of a step in f32 in TMEM, and
// the epilogue warps fold each step into their sums in registers, times the row's and the weights'
// scale.  Roles: warp 0 loads by TMA, and rows by id come through warps 0 and 2 with cp.async (38 411 rows of
// 256 by id: 25 us with the gather form of the TMA load, 20 so); one thread each of warps 1 and 3 issues
// tcgen05.mma (K = 32 each) and the commits; warps 4 - 11 read TMEM (a warp can reach only the 32 lanes
// of its number mod 4, so two warps share a quarter of the rows and split the columns).  Each
// epilogue thread loads its own row's scales, four steps at a time, four steps ahead and across tiles.
//
// Measured: 131 072 x 2048 x 1024 to bf16 305 us alone, 313 - 325 back to back, up to 373 for a second and more under the
// power cap (1.8 - 1.5 PFLOP/s; 1.1 - 0.9 of the measured bf16 rate of the library's product).  Without the epilogue's work 230 us: a step's 32 KB pass through shared memory twice, on their
// way in and as operands, 512 clocks at 128 bytes where its multiplications take 256.  The rest is
// TMEM reads and sums that do not hide behind them.  38 411 x 256 x 256 without ids 11.8 us, of them
// about 4 the launch and the first tile's chain, then 1.6 us a round of 148 tiles: 4.5 TB/s, rows from L2.  By id 12.9 us
// with the same ids in every call (rows in L2), 14.3 with others each time (rows of 2 M, from HBM).
//
// Every wait is bounded.  A role whose wait runs out marks the block dead and the sticky error
// word (the store's, or the device's); all roles then leave their loops, copies and multiplications in flight are waited for
// (bounded too) and TMEM is freed.
constexpr int kBM = 128, kBK = 128, kAccStages = 4, kTileThreads = 384;
constexpr long long kWaitLimit = 4000000000ll;  // clocks, two seconds

constexpr int load_stages(int bn, int elem) { return bn < 128 ? 7 : elem == 2 ? 5 : 4; }
constexpr int stage_bytes(int bn) { return (kBM + bn) * kBK; }
constexpr int out_bytes(int bn, int elem) { return 8 * 32 * (bn / 2) * elem; }  // the epilogue warps' rows on their way out
constexpr int tile_shared(int bn, int elem) { return load_stages(bn, elem) * stage_bytes(bn) + out_bytes(bn, elem) + 1024 + 256 + kBM * 4; }
// Bytes of a row that leave together: a box of the output's tensor map is 32 rows of so many, and is its swizzle.
constexpr int box_bytes(int bn, int elem) { return bn / 2 * elem < 128 ? bn / 2 * elem : 128; }

struct TileArgs {
    ProductArgs p;
    uint32_t m_tiles, n_tiles;
    uint32_t tma_out;      // the output's rows start on multiples of 16 bytes
    uint32_t scale_align;  // scales of a row that one load may take: 4, 2 or 1
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// The same without the wait that try_wait may spend on it.
__device__ __forceinline__ bool mbar_try_once(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Waits for the barrier's phase; false when the block is dead or the time ran out (which marks it dead).
// The clock is looked at now and then only.
__device__ __forceinline__ bool mbar_wait(const ProductArgs &a, uint32_t bar, uint32_t parity, volatile uint32_t *dead) {
    if (mbar_try(bar, parity)) return true;
    const long long since = clock64();
    for (uint32_t i = 1;; ++i) {
        if (mbar_try(bar, parity)) return true;
        if (i % 64) continue;
        if (*dead) return false;
        if (clock64() - since > kWaitLimit) {
            *dead = 1;
            raise(a, kErrSpinTimeout);
            return false;
        }
    }
}
// The same for what is already in flight when a dead block ends.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
    const long long since = clock64();
    while (!mbar_try(bar, parity) && clock64() - since < kWaitLimit) {}
}
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap *map, uint32_t bar, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(is));
    return is != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// Shared-memory matrix descriptor: rows of 128 bytes, 128-byte swizzle, eight rows (1024 bytes) to the next group.
__device__ __forceinline__ uint64_t matrix_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// 32 columns of this warp's 32 TMEM lanes, a lane a thread.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
                   "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
                   "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
}

// Waits for this thread's TMEM loads.  The registers pass through, so that no use of theirs moves ahead of it.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]) :: "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
    uint32_t (&lo)[16] = *(uint32_t (*)[16])&v[0];
    uint32_t (&hi)[16] = *(uint32_t (*)[16])&v[16];
    tmem_wait(lo);
    tmem_wait(hi);
}

template <typename T> __device__ __forceinline__ T round_to(float v);
template <> __device__ __forceinline__ float round_to<float>(float v) { return v; }
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// What an epilogue warp holds of its tile, 32 rows x COLS columns, a row a thread, leaves through
// shared memory, so that rows go out one beside the other in whole sectors: by TMA, which also leaves out what
// lies past the output's edges and works while the warp goes on, where the output's rows start on 16 bytes; else
// in units of eight bytes, or one by one.  16-byte piece j of a row is swizzled as the tensor map has it, which also
// spreads neighbouring threads' pieces over the banks.
template <typename T, int COLS>
__device__ __forceinline__ void store_rows(const TileArgs &t, const CUtensorMap *map, uint32_t m0, uint32_t n0, const float (&acc)[COLS], bool valid,
                                           uint8_t *out, uint32_t lane) {
    constexpr uint32_t kBox = COLS * sizeof(T) < 128 ? COLS * sizeof(T) : 128, kPer = 16 / sizeof(T), kBoxCols = kBox / sizeof(T), kPieces = kBox / 16;
    const ProductArgs &a = t.p;
    auto at = [&](uint32_t part, uint32_t r, uint32_t j) { return out + part * 32 * kBox + r * kBox + ((j ^ ((r * kBox / 128) % kPieces)) * 16); };
    if (t.tma_out && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();  // the last tile's rows have been read
#pragma unroll
    for (uint32_t part = 0; part < COLS / kBoxCols; ++part)
#pragma unroll
        for (uint32_t j = 0; j < kPieces; ++j) {
            T e[kPer];
#pragma unroll
            for (uint32_t i = 0; i < kPer; ++i) e[i] = round_to<T>(valid ? acc[part * kBoxCols + j * kPer + i] : 0.f);
            uint4 q;
            memcpy(&q, e, 16);
            *(uint4 *)at(part, lane, j) = q;
        }
    if (t.tma_out) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
#pragma unroll
            for (uint32_t part = 0; part < COLS / kBoxCols; ++part)
                if (n0 + part * kBoxCols < a.out_dim)
                    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                                 :: "l"(map), "r"(smem_u32(out + part * 32 * kBox)), "r"(n0 + part * kBoxCols), "r"(m0) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        return;
    }
    __syncwarp();
    const uint32_t rows = (uint32_t)min((uint64_t)32, a.rows - m0), cols = min((uint32_t)COLS, a.out_dim - n0);
    T *to = (T *)a.out + (uint64_t)m0 * a.out_stride + n0;
    auto copy = [&](auto unit, uint32_t from, uint32_t end) {  // columns [from, end) of the rows, a unit a lane
        using U = decltype(unit);
        constexpr uint32_t kUnit = sizeof(U) / sizeof(T), kLanes = COLS / kUnit < 32 ? COLS / kUnit : 32;  // lanes a row
        for (uint32_t c = from + lane % kLanes * kUnit; c < end; c += kLanes * kUnit) {
            const uint32_t in = c % kBoxCols;
            for (uint32_t r = lane / kLanes; r < rows; r += 32 / kLanes)
                *(U *)(to + (uint64_t)r * a.out_stride + c) = *(const U *)(at(c / kBoxCols, r, in / kPer) + in % kPer * sizeof(T));
        }
    };
    constexpr uint32_t kPerUnit = 8 / sizeof(T);
    const uint32_t whole = a.out_stride % kPerUnit == 0 && (uintptr_t)a.out % 8 == 0 ? cols / kPerUnit * kPerUnit : 0;
    if (whole) copy(uint2(), 0, whole);
    if (whole < cols) copy(T(), whole, cols);
}

// acc += scale * v for two columns at once.
__device__ __forceinline__ void fma2(float &a0, float &a1, float s, uint32_t v0, uint32_t v1) {
    uint64_t a, v, ss;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(a0), "f"(a1));
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
    asm("mov.b64 %0, {%1, %1};" : "=l"(ss) : "f"(s));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(v), "l"(ss));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(a));
}

// The held row that output row m takes; `held` or more where there is none.
template <bool IDS> __device__ __forceinline__ uint64_t id_of(const ProductArgs &a, uint64_t m) {
    if (m >= a.rows) return a.held;
    return !IDS ? m : a.ids64 ? (uint64_t)__ldg((const long long *)a.ids + m) : (uint64_t)__ldg((const uint32_t *)a.ids + m);
}

template <int BN, bool IDS, typename T>
__global__ void __launch_bounds__(kTileThreads, 1)
k_product_tile(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out,
               const __grid_constant__ TileArgs t) {
    constexpr int kStages = load_stages(BN, sizeof(T)), kHalf = BN / 2;
    // A wait by parity knows a phase from the next but not from the one after: a warp that issues step n may look for
    // it in stage n % kStages only when step n - kStages is known to have landed.  What shows that is its
    // accumulator, drained of step n - kAccStages: steps are loaded and drained in order.
    static_assert(kStages >= kAccStages, "the drained accumulator is of a step no older than the stage's last");
    extern __shared__ uint8_t raw_shared[];
    uint8_t *shared = (uint8_t *)(((uintptr_t)raw_shared + 1023) & ~(uintptr_t)1023);  // the swizzle's period
    uint64_t *bars = (uint64_t *)(shared + kStages * stage_bytes(BN) + out_bytes(BN, sizeof(T)));
    const uint32_t full = smem_u32(bars), empty = full + 8 * kStages, acc_full = empty + 8 * kStages, acc_empty = acc_full + 8 * kAccStages,
                   done = acc_empty + 8 * kAccStages;
    uint32_t *words = (uint32_t *)(bars + 2 * kStages + 2 * kAccStages + 2);
    uint8_t *out_shared = shared + kStages * stage_bytes(BN);  // 1024-byte aligned, as the swizzle wants it
    volatile uint32_t *dead = words + 1;
    uint32_t *row_ids = words + 4;  // of a tile's rows
    const ProductArgs &a = t.p;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // the shuffles tell that all lanes agree
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(full + 8 * i, IDS ? 3 : 1); mbar_init(empty + 8 * i, 1); }
        for (int i = 0; i < kAccStages; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_empty + 8 * i, 8); }
        mbar_init(done, 1);
        mbar_init(done + 8, 1);
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(words)), "r"(kAccStages * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(0xffffffffu, *(volatile uint32_t *)words, 0), shared_at = smem_u32(shared);
    const uint32_t tiles = t.m_tiles * t.n_tiles, steps = a.blocks;

    if (IDS ? warp == 0 || warp == 2 : warp == 0) {
        uint32_t issued = 0, landed = 0;
        bool alive = true;
        uint64_t id[2];  // rows half + lane and half + lane + 32 of the tile
        const uint32_t first = warp * 32, piece = lane % 8;
        auto load_ids = [&](uint32_t tile) {
#pragma unroll
            for (int i = 0; i < 2; ++i) id[i] = tile < tiles ? id_of<IDS>(a, (uint64_t)(tile / t.n_tiles) * kBM + first + lane + i * 32) : a.held;
        };
        // This warp's copies of step `landed` are there: made visible to the tensor core, then reported.
        auto report = [&] {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * (landed % kStages));
            ++landed;
        };
        if (IDS) load_ids(blockIdx.x);
        for (uint32_t tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
            const uint32_t m0 = tile / t.n_tiles * kBM, n0 = tile % t.n_tiles * BN;
            uint32_t *mine = row_ids + first;
            const uint8_t *rows[16];  // rows lane / 8, lane / 8 + 4, ... of this warp's half
            if (IDS) {  // rows without one, and ids outside, load row 0: the epilogue leaves its zeros
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mine[lane + i * 32] = id[i] < a.held ? (uint32_t)id[i] : 0;
                    if (id[i] >= a.held && m0 + first + lane + i * 32 < a.rows) raise(a, kErrBadId);
                }
                __syncwarp();
                load_ids(tile + gridDim.x);  // a tile ahead
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) rows[i] = a.codes + (uint64_t)mine[lane / 8 + i * 4] * (uint32_t)a.code_stride;
            }
            for (uint32_t k = 0; k < steps; ++k, ++issued) {
                const uint32_t s = issued % kStages;
                alive = __all_sync(0xffffffffu, mbar_wait(a, empty + 8 * s, (issued / kStages & 1) ^ 1, dead));
                if (!alive) break;
                const uint32_t at = shared_at + s * stage_bytes(BN);
                if (warp == 0 && elect_one()) {
                    mbar_expect(full + 8 * s, IDS ? BN * kBK : stage_bytes(BN));
                    if (!IDS) tma_tile(at, &map_a, full + 8 * s, k * kBK, m0);
                    tma_tile(at + kBM * kBK, &map_w, full + 8 * s, k * kBK, n0);
                }
                if (IDS) {  // eight lanes a row, 16 bytes each, swizzled as the tensor maps do; zeros past the row's end
                    const uint32_t c = k * kBK + piece * 16, bytes = c < a.dim ? min(a.dim - c, 16u) : 0, from = bytes ? c : 0;
                    const uint32_t even = at + (first + lane / 8) * kBK + ((piece ^ (lane / 8)) * 16), odd = even ^ 64;  // rows 4 apart
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                     :: "r"((i & 1 ? odd : even) + i * 4 * kBK), "l"(rows[i] + from), "r"(bytes) : "memory");
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (issued - landed >= kStages - 2) {
                        asm volatile("cp.async.wait_group %0;" :: "n"(kStages - 2) : "memory");
                        report();
                    }
                }
            }
        }
        if (IDS) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            while (landed < issued) report();  // of a dead block too: the loads' barriers end
        }
        // What arrives on the block's barriers by itself does so before the block ends: the last stages' commits or, where
        // a wait has run out (here or in the warps that multiply), the loads.
        if (warp == 0)
            for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                alive = alive && mbar_wait(a, empty + 8 * (i % kStages), i / kStages & 1, dead);
                if (!alive) mbar_drain(full + 8 * (i % kStages), i / kStages & 1);
            }
    } else if (warp & 1 && warp < 4) {
        // The whole warp walks the loop, so that addresses stay in uniform registers, and one lane issues.
        constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);  // e4m3 x e4m3 -> f32
        // Two warps issue in turn: every step has accumulators and operands of its own, and a warp's
        // overhead from one step to the next (barriers, descriptors, commits: 340 clocks) is longer than the 256
        // that a step's multiplications take.  Each tries its next step's barriers between this one's multiplications.
        const uint32_t total = blockIdx.x < tiles ? ((tiles - 1 - blockIdx.x) / gridDim.x + 1) * steps : 0;
        bool alive = true, ready = false;
        for (uint32_t n = warp >> 1; n < total; n += 2) {
            const uint32_t s = n % kStages, c = n % kAccStages;
            if (!__all_sync(0xffffffffu, ready)) {
                alive = __all_sync(0xffffffffu, mbar_wait(a, acc_empty + 8 * c, (n / kAccStages & 1) ^ 1, dead) && mbar_wait(a, full + 8 * s, n / kStages & 1, dead));
                if (!alive) break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t at = shared_at + s * stage_bytes(BN), d = tmem + c * BN;
            const uint64_t da = matrix_desc(at), db = matrix_desc(at + kBM * kBK);
            const bool leads = elect_one();
            if (leads) {
                mma_f8(d, da, db, kIdesc, false);
                mma_f8(d, da + 2, db + 2, kIdesc, true);
            }
            __syncwarp();
            const uint32_t next = n + 2, s2 = next % kStages, c2 = next % kAccStages;
            ready = next < total && mbar_try_once(acc_empty + 8 * c2, (next / kAccStages & 1) ^ 1) && mbar_try_once(full + 8 * s2, next / kStages & 1);
            if (leads) {
                mma_f8(d, da + 4, db + 4, kIdesc, true);
                mma_f8(d, da + 6, db + 6, kIdesc, true);
                mma_commit(empty + 8 * s);
                mma_commit(acc_full + 8 * c);
            }
            __syncwarp();
        }
        if (!alive) {
            if (elect_one()) mma_commit(done + 8 * (warp >> 1));
            __syncwarp();
            mbar_drain(done + 8 * (warp >> 1), 0);
        }
    } else if (warp >= 4) {
        const uint32_t quarter = warp & 3, half = (warp - 4) / 4;
        constexpr int kLoad = kHalf >= 32 ? 32 : 16, kParts = kHalf / kLoad;
        uint8_t *out = out_shared + (warp - 4) * 32 * kHalf * sizeof(T);
        uint32_t n = 0;
        bool alive = true, ready = false;
        auto id_at = [&](uint32_t tile) { return tile < tiles ? id_of<IDS>(a, (uint64_t)(tile / t.n_tiles) * kBM + quarter * 32 + lane) : a.held; };
        uint64_t id = id_at(blockIdx.x);
        float next[4];  // the row's scales of four steps
        auto fetch = [&](const float *row, uint32_t k) {
            const uint32_t left = steps - k;
            if (t.scale_align == 4) {
                const float4 f = __ldg((const float4 *)(row + k));
                next[0] = f.x; next[1] = f.y; next[2] = f.z; next[3] = f.w;
            } else if (t.scale_align == 2) {
                const float2 lo = __ldg((const float2 *)(row + k)), hi = left > 2 ? __ldg((const float2 *)(row + k + 2)) : make_float2(0.f, 0.f);
                next[0] = lo.x; next[1] = lo.y; next[2] = hi.x; next[3] = hi.y;
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) next[j] = j < left ? __ldg(row + k + j) : 0.f;
            }
        };
        bool valid = id < a.held;
        const float *row = a.scales + (valid ? id : 0) * steps;
        fetch(row, 0);
        for (uint32_t tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
            const uint32_t m0 = tile / t.n_tiles * kBM + quarter * 32, nt = tile % t.n_tiles, n0 = nt * BN + half * kHalf;
            const float *weights = a.weight_scales + (uint64_t)(nt * BN / kF8Block) * steps;
            float weight = lane < steps ? __ldg(weights + lane) : 0.f;  // 32 steps' in the lanes
            id = id_at(tile + gridDim.x);
            float acc[kHalf];
            if (a.bias && n0 + kHalf <= a.out_dim && (uintptr_t)a.bias % 16 == 0) {  // the sums start from it: one branch here, not one for each value that is stored
#pragma unroll
                for (int i = 0; i < kHalf; i += 4) {
                    const float4 f = __ldg((const float4 *)(a.bias + n0 + i));
                    acc[i] = f.x; acc[i + 1] = f.y; acc[i + 2] = f.z; acc[i + 3] = f.w;
                }
            } else if (a.bias) {
#pragma unroll
                for (int i = 0; i < kHalf; ++i) acc[i] = n0 + i < a.out_dim ? __ldg(a.bias + n0 + i) : 0.f;
            } else {
#pragma unroll
                for (int i = 0; i < kHalf; ++i) acc[i] = 0.f;
            }
            for (uint32_t k0 = 0; k0 < steps && alive; k0 += 4) {
                float scale[4];
                if (k0 && k0 % 32 == 0) weight = k0 + lane < steps ? __ldg(weights + k0 + lane) : 0.f;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) scale[j] = next[j] * __shfl_sync(0xffffffffu, weight, k0 % 32 + j);
                if (k0 + 4 < steps) fetch(row, k0 + 4);
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    if (k0 + j >= steps) break;
                    const uint32_t c = n % kAccStages;
                    if (!__all_sync(0xffffffffu, ready)) {
                        alive = __all_sync(0xffffffffu, mbar_wait(a, acc_full + 8 * c, n / kAccStages & 1, dead));
                        if (!alive) break;
                    }
                    ++n;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t from = tmem + c * BN + half * kHalf + (quarter << 21);
                    uint32_t v[kParts][kLoad];
#pragma unroll
                    for (int q = 0; q < kParts; ++q) {
                        if constexpr (kLoad == 32) tmem_load32(from + q * 32, v[q]);
                        else tmem_load16(from, v[q]);
                    }
#pragma unroll
                    for (int q = 0; q < kParts; ++q) tmem_wait(v[q]);
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    if (lane == 0) mbar_arrive(acc_empty + 8 * c);
                    ready = mbar_try_once(acc_full + 8 * (n % kAccStages), n / kAccStages & 1);  // the answer comes beside the sums
#pragma unroll
                    for (int i = 0; i < kHalf; i += 2) fma2(acc[i], acc[i + 1], scale[j], v[i / kLoad][i % kLoad], v[i / kLoad][i % kLoad + 1]);
                }
            }
            const bool keep = valid;
            valid = id < a.held;
            row = a.scales + (valid ? id : 0) * steps;
            if (tile + gridDim.x < tiles) fetch(row, 0);
            if (alive && m0 < a.rows && n0 < a.out_dim) store_rows<T, kHalf>(t, &map_out, m0, n0, acc, keep, out, lane);
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(kAccStages * BN));
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                 const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static EncodeTiled fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult status;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &status) == cudaSuccess && status == cudaDriverEntryPointSuccess)
            fn = (EncodeTiled)p;
        else cudaGetLastError();
    });
    return fn;
}

// Rows of elements of `elem` bytes as a tensor map of boxes `box_cols` x `box_rows`, swizzled over a box's
// bytes (128, 64 or 32).  What lies outside reads as zeros and is not written.
int32_t rows_map(CUtensorMap *map, const void *base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t elem, uint32_t box_cols, uint32_t box_rows) {
    if (!encode_tiled()) return fail(AG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
    const cuuint32_t boxes[2] = {box_cols, box_rows}, steps[2] = {1, 1};
    const uint32_t bytes = box_cols * elem;
    const CUresult r = encode_tiled()(map, elem == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32,
                                      2, const_cast<void *>(base), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                      bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(AG_ERR_CUDA, "cannot describe %llu rows of %llu elements at a pitch of %llu bytes (driver error %d)", (unsigned long long)rows,
                    (unsigned long long)cols, (unsigned long long)pitch, (int)r);
    return AG_OK;
}

template <int BN, bool IDS, typename T>
int32_t launch_tile(const ProductArgs &a, cudaStream_t st) {
    const uint64_t pitch = a.out_stride * sizeof(T);
    TileArgs t{a, (uint32_t)((a.rows + kBM - 1) / kBM), (a.out_dim + BN - 1) / BN, pitch % 16 == 0 && (uintptr_t)a.out % 16 == 0 && pitch < (1ull << 40),
               a.blocks % 4 == 0 && (uintptr_t)a.scales % 16 == 0 ? 4u : a.blocks % 2 == 0 && (uintptr_t)a.scales % 8 == 0 ? 2u : 1u};
    CUtensorMap map_a{}, map_w, map_out{};
    if (!IDS) AG_TRY(rows_map(&map_a, a.codes, a.rows, a.dim, a.code_stride, 1, kBK, kBM));
    AG_TRY(rows_map(&map_w, a.weight, a.out_dim, a.dim, a.weight_stride, 1, kBK, BN));
    if (t.tma_out) AG_TRY(rows_map(&map_out, a.out, a.rows, a.out_dim, pitch, sizeof(T), box_bytes(BN, sizeof(T)) / sizeof(T), 32));
    AG_CUDA(cudaFuncSetAttribute(k_product_tile<BN, IDS, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, tile_shared(BN, sizeof(T))));
    const uint64_t tiles = (uint64_t)t.m_tiles * t.n_tiles;
    if (tiles > 0x7FFFFFFFull) return fail(AG_ERR_VALUE, "ag_rows_product: the output is too large");
    k_product_tile<BN, IDS, T><<<(uint32_t)std::min<uint64_t>(tiles, kSMs), kTileThreads, tile_shared(BN, sizeof(T)), st>>>(map_a, map_w, map_out, t);
    return AG_OK;
}

template <bool IDS, typename T> int32_t launch_tile(const ProductArgs &a, cudaStream_t st) {
    // Width by the rounds of tiles that it makes and what a round costs: 1.56, 1.10 and 0.98 us for 128, 64 and 32
    // columns at dim 256.  2000 x 512 x 512: 5.7, 4.9 and 5.8 us (1, 1 and 2 rounds); 38 411 x 256 x 256: 11.8, 13.9
    // and 20.7 (5, 9 and 17); 20 000 x 256 x 64: 6.3, 5.5, 6.3 (2, 2, 3).
    const uint64_t m_tiles = (a.rows + kBM - 1) / kBM;
    auto cost = [&](uint32_t width, uint32_t each) { return (m_tiles * ((a.out_dim + width - 1) / width) + kSMs - 1) / kSMs * each; };
    const uint64_t c128 = cost(128, 156), c64 = cost(64, 110), c32 = cost(32, 98);
    const uint32_t bn = c128 <= c64 && c128 <= c32 ? 128 : c64 <= c32 ? 64 : 32;
    if (bn == 128) return launch_tile<128, IDS, T>(a, st);
    if (bn == 64) return launch_tile<64, IDS, T>(a, st);
    return launch_tile<32, IDS, T>(a, st);
}

template <typename T> int32_t launch_tile(const ProductArgs &a, cudaStream_t st) {
    return a.ids ? launch_tile<true, T>(a, st) : launch_tile<false, T>(a, st);
}

}  // namespace

}  // namespace ag

using namespace ag;

extern "C" int32_t ag_rows_product(const ag_product *call, int32_t device, void *stream) {
    if (!call) return fail(AG_ERR_VALUE, "ag_rows_product: null argument");
    ag_product own = *call;
    ag_product *p = &own;
    if (const ag_features *f = p->store) {
        if (f->dtype != AG_F8) return fail(AG_ERR_VALUE, "ag_rows_product: the store does not hold 8-bit float rows");
        if (f->device != device) return fail(AG_ERR_VALUE, "ag_rows_product: the store is on device %d, the call on %d", f->device, device);
        if (p->codes || p->scales) return fail(AG_ERR_VALUE, "ag_rows_product: either a store or rows");
        p->codes = f->payload; p->scales = f->scales; p->held = f->rows; p->code_stride = f->pitch;
        if (f->dim != p->dim) return fail(AG_ERR_VALUE, "ag_rows_product: rows of %llu columns, weights of %llu", (unsigned long long)f->dim, (unsigned long long)p->dim);
    }
    if (p->out_dtype < AG_F32 || p->out_dtype > AG_BF16) return fail(AG_ERR_VALUE, "ag_rows_product: the output is f32, f16 or bf16, got dtype tag %d", p->out_dtype);
    if (p->dim == 0 || p->dim > 0x7FFFFF00ull || p->code_stride > 0xFFFFFFF0ull || p->out_dim == 0 || p->out_dim >= (1ull << 31) || p->held >= (1ull << 31) || p->rows >= (1ull << 31))
        return fail(AG_ERR_VALUE, "ag_rows_product: %llu rows of %llu x %llu from %llu held rows are out of range", (unsigned long long)p->rows,
                    (unsigned long long)p->dim, (unsigned long long)p->out_dim, (unsigned long long)p->held);
    if (p->rows == 0) return AG_OK;
    if (!p->codes || !p->scales || !p->weight || !p->weight_scales || !p->out) return fail(AG_ERR_VALUE, "ag_rows_product: null argument");
    if (p->held == 0) return fail(AG_ERR_VALUE, "ag_rows_product: no rows are held");
    if (!p->ids && p->held < p->rows) return fail(AG_ERR_VALUE, "ag_rows_product: %llu rows of %llu held", (unsigned long long)p->rows, (unsigned long long)p->held);
    if (p->code_stride % 16 || p->weight_stride % 16 || p->code_stride < p->dim || p->weight_stride < p->dim || (uintptr_t)p->codes % 16 ||
        (uintptr_t)p->weight % 16)
        return fail(AG_ERR_VALUE, "ag_rows_product: 8-bit rows start on multiples of 16 bytes and do not overlap");
    if (p->out_stride < p->out_dim) return fail(AG_ERR_VALUE, "ag_rows_product: rows of the output overlap");
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    ProductArgs a{};
    a.codes = (const uint8_t *)p->codes; a.weight = (const uint8_t *)p->weight; a.scales = p->scales; a.weight_scales = p->weight_scales;
    a.ids = p->ids; a.bias = p->bias; a.out = p->out; a.error = p->store ? p->store->err : nullptr; a.rows = p->rows; a.held = p->ids ? p->held : (1ull << 31);
    a.code_stride = p->code_stride; a.weight_stride = p->weight_stride; a.out_stride = p->out_stride;
    a.dim = (uint32_t)p->dim; a.out_dim = (uint32_t)p->out_dim; a.blocks = (uint32_t)((p->dim + kF8Block - 1) / kF8Block);
    a.ids64 = p->ids_are_i64; a.out_dtype = p->out_dtype;
    cudaStream_t st = (cudaStream_t)stream;
    if (a.rows <= kFewRows) {
        k_product_dot<<<(a.out_dim + kDotThreads / 32 - 1) / (kDotThreads / 32), kDotThreads, 0, st>>>(a);
    } else if (a.out_dtype == AG_F32) {
        AG_TRY(launch_tile<float>(a, st));
    } else if (a.out_dtype == AG_F16) {
        AG_TRY(launch_tile<__half>(a, st));
    } else {
        AG_TRY(launch_tile<__nv_bfloat16>(a, st));
    }
    AG_CUDA(cudaGetLastError());
    return AG_OK;
}

namespace ag {
namespace {
__global__ void k_clear_bits(uint32_t *word, uint32_t bits) { atomicAnd(word, ~bits); }
}  // namespace

// A run-out wait comes first and alone, the rest stays for the next call; only what is reported is cleared, so that
// what other streams raise meanwhile is kept.
int32_t take_error(uint32_t *word, uint32_t *bits) {
    AG_CUDA(cudaDeviceSynchronize());
    AG_CUDA(cudaMemcpy(bits, word, 4, cudaMemcpyDeviceToHost));
    if (*bits & kErrSpinTimeout) *bits = kErrSpinTimeout;
    if (*bits) {
        k_clear_bits<<<1, 1>>>(word, *bits);
        AG_CUDA(cudaGetLastError());
        AG_CUDA(cudaStreamSynchronize(nullptr));
    }
    return AG_OK;
}
}  // namespace ag

extern "C" int32_t ag_rows_check(int32_t device) {
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    uint32_t *word = nullptr, bits = 0;
    AG_CUDA(cudaGetSymbolAddress((void **)&word, g_rows_error));
    AG_TRY(take_error(word, &bits));
    if (bits == kErrSpinTimeout) return fail(AG_ERR_CUDA, "a product gave up waiting for its loads or multiplications; its output is incomplete");
    return bits ? fail(AG_ERR_VALUE, "a row id of a product is out of bounds") : AG_OK;
}
