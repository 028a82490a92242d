// Product of 8-bit rows (e4m3, a scale per 128 columns of a row) with 8-bit weights (a scale per
// 128 x 128 block), the rows in order or by id: the gather of a feature store that multiplies
// what it reads.  No counterpart in the reference.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace ag {

namespace {

__device__ uint32_t g_rows_error;  // sticky error bits of this device's products (ag_rows_check)

struct ProductArgs {
    const uint8_t *codes, *weight;
    const float *scales, *weight_scales;
    const void *ids;
    const float *bias;
    void *out;
    uint64_t rows, held, code_stride, weight_stride, out_stride;
    uint32_t dim, out_dim, blocks;  // blocks: of 128 columns
    int ids64, out_dtype;
};

// Row of the codes that output row m takes; `held` where its id names none.
__device__ __forceinline__ uint64_t source_row(const ProductArgs &a, uint64_t m) {
    if (!a.ids) return m;
    const uint64_t id = a.ids64 ? (uint64_t)((const int64_t *)a.ids)[m] : (uint64_t)((const uint32_t *)a.ids)[m];
    if (id < a.held) return id;
    atomicOr(&g_rows_error, kErrBadId);
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

constexpr int kDotThreads = 256, kDotRows = 4;

// Few rows: a warp per column of the output and up to kDotRows rows.
__global__ void __launch_bounds__(kDotThreads)
k_product_dot(ProductArgs a) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t n = blockIdx.x * (kDotThreads / 32) + (threadIdx.x >> 5);
    const uint64_t m0 = (uint64_t)blockIdx.y * kDotRows;
    if (n >= a.out_dim) return;
    uint64_t src[kDotRows];
    float acc[kDotRows];
#pragma unroll
    for (int r = 0; r < kDotRows; ++r) {
        src[r] = m0 + r < a.rows ? source_row(a, m0 + r) : a.held;
        acc[r] = 0.f;
    }
    for (uint32_t c = lane * 16; c < a.dim; c += 512) {
        float w[16];
        load_codes(a.weight + (uint64_t)n * a.weight_stride, c, a.dim, w);
        const float ws = a.weight_scales[(uint64_t)(n / kF8Block) * a.blocks + c / kF8Block];
#pragma unroll
        for (int r = 0; r < kDotRows; ++r) {
            if (src[r] == a.held) continue;
            float v[16], dot = 0.f;
            load_codes(a.codes + src[r] * a.code_stride, c, a.dim, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) dot += v[i] * w[i];
            acc[r] += dot * (a.scales[src[r] * a.blocks + c / kF8Block] * ws);
        }
    }
#pragma unroll
    for (int r = 0; r < kDotRows; ++r) {
        for (int o = 16; o > 0; o /= 2) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (lane == 0 && m0 + r < a.rows) store_out(a, m0 + r, n, src[r] == a.held ? 0.f : acc[r] + (a.bias ? a.bias[n] : 0.f));
    }
}

}  // namespace

}  // namespace ag

using namespace ag;

extern "C" int32_t ag_rows_product(const ag_product *p, int32_t device, void *stream) {
    if (!p) return fail(AG_ERR_VALUE, "ag_rows_product: null argument");
    if (p->out_dtype < AG_F32 || p->out_dtype > AG_BF16) return fail(AG_ERR_VALUE, "ag_rows_product: the output is f32, f16 or bf16, got dtype tag %d", p->out_dtype);
    if (p->dim == 0 || p->dim > 0x7FFFFF00ull || p->out_dim == 0 || p->out_dim >= (1ull << 31) || p->held >= (1ull << 31) || p->rows >= (1ull << 31))
        return fail(AG_ERR_VALUE, "ag_rows_product: %llu rows of %llu x %llu from %llu held rows are out of range", (unsigned long long)p->rows,
                    (unsigned long long)p->dim, (unsigned long long)p->out_dim, (unsigned long long)p->held);
    if (p->rows == 0) return AG_OK;
    if (!p->codes || !p->scales || !p->weight || !p->weight_scales || !p->out) return fail(AG_ERR_VALUE, "ag_rows_product: null argument");
    if (!p->ids && p->held < p->rows) return fail(AG_ERR_VALUE, "ag_rows_product: %llu rows of %llu held", (unsigned long long)p->rows, (unsigned long long)p->held);
    if (p->code_stride % 16 || p->weight_stride % 16 || p->code_stride < p->dim || p->weight_stride < p->dim || (uintptr_t)p->codes % 16 ||
        (uintptr_t)p->weight % 16)
        return fail(AG_ERR_VALUE, "ag_rows_product: 8-bit rows start on multiples of 16 bytes and do not overlap");
    if (p->out_stride < p->out_dim) return fail(AG_ERR_VALUE, "ag_rows_product: rows of the output overlap");
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    ProductArgs a{};
    a.codes = (const uint8_t *)p->codes; a.weight = (const uint8_t *)p->weight; a.scales = p->scales; a.weight_scales = p->weight_scales;
    a.ids = p->ids; a.bias = p->bias; a.out = p->out; a.rows = p->rows; a.held = p->ids ? p->held : (1ull << 31);
    a.code_stride = p->code_stride; a.weight_stride = p->weight_stride; a.out_stride = p->out_stride;
    a.dim = (uint32_t)p->dim; a.out_dim = (uint32_t)p->out_dim; a.blocks = (uint32_t)((p->dim + kF8Block - 1) / kF8Block);
    a.ids64 = p->ids_are_i64; a.out_dtype = p->out_dtype;
    cudaStream_t st = (cudaStream_t)stream;
    const uint64_t slabs = (a.rows + kDotRows - 1) / kDotRows;
    for (uint64_t s0 = 0; s0 < slabs; s0 += 65535) {  // the grid's y ends there
        ProductArgs b = a;
        b.rows = std::min<uint64_t>(a.rows - s0 * kDotRows, 65535ull * kDotRows);
        if (a.ids) b.ids = (const uint8_t *)a.ids + s0 * kDotRows * (a.ids64 ? 8 : 4);
        else { b.codes += s0 * kDotRows * a.code_stride; b.scales += s0 * kDotRows * a.blocks; }
        b.out = (uint8_t *)a.out + s0 * kDotRows * a.out_stride * elem_size(a.out_dtype);
        const uint32_t y = (uint32_t)std::min<uint64_t>(slabs - s0, 65535);
        k_product_dot<<<dim3((a.out_dim + kDotThreads / 32 - 1) / (kDotThreads / 32), y), kDotThreads, 0, st>>>(b);
    }
    AG_CUDA(cudaGetLastError());
    return AG_OK;
}

extern "C" int32_t ag_rows_check(int32_t device) {
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    uint32_t h = 0;
    AG_CUDA(cudaDeviceSynchronize());
    AG_CUDA(cudaMemcpyFromSymbol(&h, g_rows_error, 4));
    if (!h) return AG_OK;
    const uint32_t zero = 0;
    AG_CUDA(cudaMemcpyToSymbol(g_rows_error, &zero, 4));
    return fail(AG_ERR_VALUE, "a row id of a product is out of bounds");
}
