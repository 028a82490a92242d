// Row operators of a layer over a batch's feature rows: dropout, the root-mean-square norm
// with the residual's addition (forward and backward), rows and weights in 8-bit floats.
// No counterpart in the reference, which hands its rows to PyTorch.
//
// A row is cut into chunks of eight consecutive columns.  A thread owns a chunk: 16 bytes of
// f16 / bf16 or 32 bytes of f32 in one load, and exactly the eight 16-bit lots of one Philox4x32-10
// call, whose counter is (chunk, row, offset) — so a mask is a function of (seed, offset, row,
// column) alone, whatever the row pitch, launch shape or type, and is made again wherever it is
// needed instead of being stored.  All sums, statistics and products are held in f32; the one
// rounding to the rows' type is the store's.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>

#include "common.cuh"
#include "internal.h"

namespace ag {

namespace {

constexpr uint32_t kChunk = 8;
constexpr float kE4M3Max = 448.0f;
constexpr uint32_t kMaxNormDim = 16384;  // 512 threads x 4 chunks

// Division of 32-bit numbers by a divisor that the host knows: one high product instead of a division
// (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994, figure 4.1).
struct Divide {
    uint32_t by = 1, m = 1, s1 = 0, s2 = 0;
    explicit Divide(uint32_t d) : by(d) {
        uint32_t l = 0;
        while (l < 32 && (1ull << l) < d) ++l;
        m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
        s1 = l < 1 ? l : 1;
        s2 = l ? l - 1 : 0;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        const uint32_t t = __umulhi(m, n);
        return (t + ((n - t) >> s1)) >> s2;
    }
    // Quotient and remainder of what may pass 32 bits.
    __device__ __forceinline__ uint64_t operator()(uint64_t n, uint32_t &rest) const {
        const uint64_t q = n <= 0xFFFFFFFFull ? (*this)((uint32_t)n) : n / by;
        rest = (uint32_t)(n - q * by);
        return q;
    }
};

// ------------------------------------------------------------ row access --
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight stored elements, before conversion.
template <typename T> struct Raw { uint32_t w[sizeof(T) * 2]; };

// Plain loads: an in-place call writes what it has read.
__device__ __forceinline__ void load_words(Raw<float> &r, const void *p) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
                 : "l"(p) : "memory");
}
template <typename T> __device__ __forceinline__ void load_words(Raw<T> &r, const void *p) {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(p) : "memory");
}
__device__ __forceinline__ void store_words(const Raw<float> &r, void *p) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" :: "l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]),
                 "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7]) : "memory");
}
template <typename T> __device__ __forceinline__ void store_words(const Raw<T> &r, void *p) {
    asm volatile("st.global.v4.b32 [%0], {%1,%2,%3,%4};" :: "l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]) : "memory");
}

// Which eight columns of a row a thread holds in its step j.  Whole chunks where every row starts on a
// multiple of eight elements' bytes and is so many chunks long (or RAGGED says otherwise): one vector load.  Elsewhere the
// lanes of a group take neighbouring columns, so that a group's loads are coalesced and it still covers whole
// chunks together: pairs of 16-bit elements where rows start on four bytes and are even, else single elements.
constexpr int kSingle = 0, kWhole = 1, kPair = 2;
template <int MODE> struct Columns {
    uint32_t first, stride;  // stride: from one of its loads to the next, in units
    __device__ __forceinline__ Columns(uint32_t lane, uint32_t lanes, uint32_t step_chunk) {  // lanes: of the group, at most 32
        stride = MODE == kWhole ? 1 : lanes;
        first = MODE == kWhole ? (step_chunk + lane) * kChunk : step_chunk * kChunk + (MODE == kPair ? 2 * lane : lane);
    }
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return MODE == kPair ? first + i / 2 * 2 * stride + i % 2 : first + i * stride; }
    __device__ __forceinline__ bool whole(uint32_t dim) const { return at(kChunk - 1) < dim; }  // one test for all of them
};

// A thread's eight columns; what lies past the row's end reads as zeros.
template <typename T, int MODE, bool RAGGED = false> __device__ __forceinline__ Raw<T> load_chunk(const T *row, const Columns<MODE> &c, uint32_t dim) {
    Raw<T> r;
    if (MODE == kWhole && (!RAGGED || c.first + kChunk <= dim)) {
        load_words(r, row + c.first);
    } else if constexpr (MODE == kPair) {
        const uint32_t *at = (const uint32_t *)(row + c.first);
        if (c.whole(dim)) {
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 2; ++i) r.w[i] = at[i * c.stride];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 2; ++i) r.w[i] = c.at(2 * i) < dim ? at[i * c.stride] : 0u;
        }
    } else {
        T e[kChunk];
        const T *at = row + c.first;
        if (c.whole(dim)) {
#pragma unroll
            for (uint32_t i = 0; i < kChunk; ++i) e[i] = at[i * c.stride];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kChunk; ++i) e[i] = c.at(i) < dim ? at[i * c.stride] : from_f32<T>(0.f);
        }
        memcpy(&r, e, sizeof r);
    }
    return r;
}
// Pairs at a time: one instruction converts or packs two 16-bit values that share a register, and
// sm_100 multiplies and adds two f32 at once.
__device__ __forceinline__ float2 pair_f32(__half, uint32_t w) { return __half22float2(*(__half2 *)&w); }
__device__ __forceinline__ float2 pair_f32(__nv_bfloat16, uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ uint32_t pair_bits(__half, float2 v) { const __half2 h = __float22half2_rn(v); return *(const uint32_t *)&h; }
__device__ __forceinline__ uint32_t pair_bits(__nv_bfloat16, float2 v) { const __nv_bfloat162 h = __float22bfloat162_rn(v); return *(const uint32_t *)&h; }

constexpr int kPairs = kChunk / 2;
struct Chunk { float2 p[kPairs]; };
template <typename T> __device__ __forceinline__ Chunk unpack(const Raw<T> &r) {
    Chunk v;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        if constexpr (sizeof(T) == 4) v.p[i] = make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
        else v.p[i] = pair_f32(T(), r.w[i]);
    }
    return v;
}
template <typename T> __device__ __forceinline__ Raw<T> pack(const Chunk &v) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        if constexpr (sizeof(T) == 4) { r.w[2 * i] = __float_as_uint(v.p[i].x); r.w[2 * i + 1] = __float_as_uint(v.p[i].y); }
        else r.w[i] = pair_bits(T(), v.p[i]);
    }
    return r;
}
__device__ __forceinline__ float &at(Chunk &v, uint32_t i) { return i & 1 ? v.p[i / 2].y : v.p[i / 2].x; }
__device__ __forceinline__ float at(const Chunk &v, uint32_t i) { return i & 1 ? v.p[i / 2].y : v.p[i / 2].x; }
__device__ __forceinline__ Chunk filled(float f) {
    Chunk v;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) v.p[i] = make_float2(f, f);
    return v;
}
__device__ __forceinline__ float2 both(float f) { return make_float2(f, f); }
template <typename T, int MODE, bool RAGGED = false> __device__ __forceinline__ void store_chunk(T *row, const Columns<MODE> &c, uint32_t dim, const Chunk &v) {
    if (MODE == kWhole && (!RAGGED || c.first + kChunk <= dim)) {
        store_words(pack<T>(v), row + c.first);
    } else if constexpr (MODE == kPair) {
        uint32_t *to = (uint32_t *)(row + c.first);
        const Raw<T> r = pack<T>(v);
        if (c.whole(dim)) {
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 2; ++i) to[i * c.stride] = r.w[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 2; ++i)
                if (c.at(2 * i) < dim) to[i * c.stride] = r.w[i];
        }
    } else {
        T *to = row + c.first;
        const Raw<T> r = pack<T>(v);
        T e[kChunk];
        memcpy(e, &r, sizeof r);
        if (c.whole(dim)) {
#pragma unroll
            for (uint32_t i = 0; i < kChunk; ++i) to[i * c.stride] = e[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kChunk; ++i)
                if (c.at(i) < dim) to[i * c.stride] = e[i];
        }
    }
}
// The norm's weights, of the rows' type or f32: the same few for every row (L1).
template <typename T, int MODE> __device__ __forceinline__ Chunk load_weight(const void *w, int w_f32, const Columns<MODE> &c, uint32_t dim) {
    if (!w) return filled(1.f);
    Chunk v;
    if (MODE == kWhole) {
        if (sizeof(T) == 4 || w_f32) {
            const float4 lo = __ldg((const float4 *)((const float *)w + c.first)), hi = __ldg((const float4 *)((const float *)w + c.first) + 1);
            v.p[0] = make_float2(lo.x, lo.y); v.p[1] = make_float2(lo.z, lo.w);
            v.p[2] = make_float2(hi.x, hi.y); v.p[3] = make_float2(hi.z, hi.w);
        } else if constexpr (sizeof(T) == 2) {
            const uint4 q = __ldg((const uint4 *)((const T *)w + c.first));
            Raw<T> r;
            r.w[0] = q.x; r.w[1] = q.y; r.w[2] = q.z; r.w[3] = q.w;
            v = unpack(r);
        }
    } else if constexpr (MODE == kPair) {
#pragma unroll
        for (uint32_t i = 0; i < kChunk / 2; ++i) {
            if (c.at(2 * i) >= dim) v.p[i] = both(0.f);
            else if (w_f32) v.p[i] = __ldg((const float2 *)((const float *)w + c.first) + i * c.stride);
            else v.p[i] = pair_f32(T(), __ldg((const uint32_t *)((const T *)w + c.first) + i * c.stride));
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kChunk; ++i)
            at(v, i) = c.at(i) >= dim ? 0.f : sizeof(T) == 4 || w_f32 ? __ldg((const float *)w + c.first + i * c.stride) : to_f32(((const T *)w + c.first)[i * c.stride]);
    }
    return v;
}

// ---------------------------------------------------------------- dropout --
struct Drop {
    uint32_t on;   // 0: no dropout
    uint32_t bar;  // an element stays iff its 16 random bits, moved to the upper half of a word, are above (T << 16) - 1
    float scale;
    uint64_t seed, offset;
};

__device__ __forceinline__ uint4 lots_of(const Drop &d, uint64_t row, uint32_t chunk) {
    return philox4x32_10(d.seed, (uint32_t)d.offset, row << 32 | chunk, (uint32_t)(d.offset >> 32));
}
// Bits of element i of a chunk; i is a constant where this is used.  The lower bits of an odd element's
// word stay: they cannot lift it over the bar, which ends in ones.
__device__ __forceinline__ uint32_t lot(const uint4 &r, uint32_t i) {
    const uint32_t w = i < 2 ? r.x : i < 4 ? r.y : i < 6 ? r.z : r.w;
    return i & 1 ? w : w << 16;
}
// Selects: a dropped infinity or NaN is gone.
__device__ __forceinline__ float kept(const Drop &d, uint32_t bits, float v) { return bits > d.bar ? v : 0.f; }
__device__ __forceinline__ void drop_chunk(const Drop &d, const uint4 &lots, Chunk &v) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        const float2 f = __fmul2_rn(v.p[i], both(d.scale));
        v.p[i] = make_float2(kept(d, lot(lots, 2 * i), f.x), kept(d, lot(lots, 2 * i + 1), f.y));
    }
}

// Dropout of a thread's eight columns.  Unless they are a chunk, the group's lanes make the lots of one
// chunk each and pass them around in shared memory (16 bytes a lane); the whole warp calls this.
template <int MODE>
__device__ __forceinline__ void drop_columns(const Drop &d, uint32_t row, uint32_t lane, uint32_t lanes, uint32_t step_chunk, uint4 *warp_lots, Chunk &v) {
    const uint4 r = lots_of(d, row, step_chunk + lane);
    if (MODE == kWhole) {
        drop_chunk(d, r, v);
    } else {
        __syncwarp();
        warp_lots[threadIdx.x & 31] = r;
        __syncwarp();
        const uint16_t *group = (const uint16_t *)(warp_lots + ((threadIdx.x & 31) - lane));
        if constexpr (MODE == kPair) {
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 2; ++i) {  // the lots of two neighbours are a word, as in a chunk
                const uint32_t u = ((const uint32_t *)group)[lane + i * lanes];
                const float2 f = __fmul2_rn(v.p[i], both(d.scale));
                v.p[i] = make_float2(kept(d, u << 16, f.x), kept(d, u, f.y));
            }
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kChunk; ++i) at(v, i) = kept(d, (uint32_t)group[lane + i * lanes] << 16, at(v, i) * d.scale);
    }
}

// Bit e: element e of a chunk stays.  bits > bar is the carry of bits + ~bar; the next addition takes it in.
__device__ __forceinline__ uint32_t stay_bits(const uint4 &r, uint32_t not_bar) {
    uint32_t m;
    asm("{\n .reg .u32 t;\n"
        " add.cc.u32 t, %4, %9;\n addc.u32 %0, 0, 0;\n"
        " add.cc.u32 t, %8, %9;\n addc.u32 %0, %0, %0;\n"
        " add.cc.u32 t, %3, %9;\n addc.u32 %0, %0, %0;\n"
        " add.cc.u32 t, %7, %9;\n addc.u32 %0, %0, %0;\n"
        " add.cc.u32 t, %2, %9;\n addc.u32 %0, %0, %0;\n"
        " add.cc.u32 t, %6, %9;\n addc.u32 %0, %0, %0;\n"
        " add.cc.u32 t, %1, %9;\n addc.u32 %0, %0, %0;\n"
        " add.cc.u32 t, %5, %9;\n addc.u32 %0, %0, %0;\n}"
        : "=&r"(m) : "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(r.x << 16), "r"(r.y << 16), "r"(r.z << 16), "r"(r.w << 16), "r"(not_bar));
    return m;
}

// Which of a thread's eight columns stay, a bit each, where one mask is used twice: the lots are as in drop_columns.
template <int MODE>
__device__ __forceinline__ uint32_t stay_columns(const Drop &d, uint32_t row, uint32_t lane, uint32_t lanes, uint32_t step_chunk, uint4 *warp_lots) {
    const uint4 r = lots_of(d, row, step_chunk + lane);
    if (MODE == kWhole) return stay_bits(r, ~d.bar);
    __syncwarp();
    warp_lots[threadIdx.x & 31] = r;
    __syncwarp();
    const uint16_t *group = (const uint16_t *)(warp_lots + ((threadIdx.x & 31) - lane));
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < kChunk / 2; ++i) {
        const uint32_t lo = MODE == kPair ? ((const uint32_t *)group)[lane + i * lanes] << 16 : (uint32_t)group[lane + 2 * i * lanes] << 16,
                       hi = MODE == kPair ? ((const uint32_t *)group)[lane + i * lanes] : (uint32_t)group[lane + (2 * i + 1) * lanes] << 16;
        m |= (lo > d.bar ? 1u << 2 * i : 0u) | (hi > d.bar ? 2u << 2 * i : 0u);
    }
    return m;
}
__device__ __forceinline__ void drop_by_bits(const Drop &d, uint32_t stay, Chunk &v) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        const float2 f = __fmul2_rn(v.p[i], both(d.scale));
        v.p[i] = make_float2(stay >> 2 * i & 1 ? f.x : 0.f, stay >> (2 * i + 1) & 1 ? f.y : 0.f);
    }
}

constexpr int kThreads = 256;

// Two chunks a thread, a block's width apart; both loads are in flight before either is used.  38 411 x 256
// bf16: 10.6 us (0.57 of the copy rate), bound by instructions: of 156 a chunk the generator's ten rounds are
// less than half, the rest is addresses, conversion, selects and packing.
template <typename T, int MODE, bool RAGGED>
__global__ void __launch_bounds__(kThreads)
k_dropout(const T *x, T *y, uint64_t total, uint32_t dim, Divide chunks, uint64_t x_stride, uint64_t y_stride, Drop d) {
    Raw<T> r[2];
    uint64_t row[2];
    uint32_t chunk[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint64_t i = ((uint64_t)blockIdx.x * 2 + u) * kThreads + threadIdx.x;
        row[u] = chunks(i, chunk[u]);
        if (i < total) r[u] = load_chunk<T, MODE, RAGGED>(x + row[u] * x_stride, Columns<MODE>(0, 1, chunk[u]), dim);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (((uint64_t)blockIdx.x * 2 + u) * kThreads + threadIdx.x >= total) break;
        Chunk v = unpack(r[u]);
        if (d.on) drop_chunk(d, lots_of(d, row[u], chunk[u]), v);
        store_chunk<T, MODE, RAGGED>(y + row[u] * y_stride, Columns<MODE>(0, 1, chunk[u]), dim, v);
    }
}

// Contiguous rows whose length is no multiple of eight: the lots belong to chunks, the memory is walked
// in aligned vectors of eight elements, whatever row they are in.  A block takes 1024 vectors, four a
// thread, and makes the lots of every chunk that reaches into them (those at its ends are made by two
// blocks): a bit per element in shared memory says whether it stays.  250 007 x 301 f16: 67 us (0.68 of the copy
// rate; bound by instructions: generator, bits, two atomics a chunk), a chunk a thread with loads of single
// elements 174.  Fewer vectors a block or more resident blocks are slower (two vectors 78 us, five blocks 72).
constexpr uint32_t kFlatVectors = 4, kFlatElements = kThreads * kFlatVectors * kChunk;
constexpr uint64_t kFlatMaxDim = 1u << 28;  // positions within a block's rows fit 32 bits

template <typename T>
__global__ void __launch_bounds__(kThreads)
k_dropout_flat(const T *x, T *y, uint64_t total, Divide dim, Divide chunks, Drop d) {
    __shared__ uint32_t stays[kFlatElements / 32];
    for (uint32_t i = threadIdx.x; i < kFlatElements / 32; i += kThreads) stays[i] = 0;
    const uint64_t origin = (uint64_t)blockIdx.x * kFlatElements, at = origin + threadIdx.x * kChunk;
    const int end = (int)min(total - origin, (uint64_t)kFlatElements);
    Raw<T> r[kFlatVectors];
#pragma unroll
    for (uint32_t j = 0; j < kFlatVectors; ++j)
        if (at + j * kThreads * kChunk + kChunk <= total) load_words(r[j], x + at + j * kThreads * kChunk);
    uint32_t c0;
    const uint64_t row0 = dim(origin, c0);
    __syncthreads();
    for (uint32_t k = c0 / kChunk + threadIdx.x;; k += kThreads) {
        const uint32_t over = chunks(k), chunk = k - over * chunks.by;
        int pos = (int)(over * dim.by + chunk * kChunk - c0);  // of the chunk's first element, from the origin
        if (pos >= end) break;
        const uint4 lots = lots_of(d, row0 + over, chunk);
        uint32_t m = stay_bits(lots, ~d.bar);
        const uint32_t len = dim.by - chunk * kChunk;
        if (len < kChunk) m &= (1u << len) - 1;
        if (pos < 0) { m >>= -pos; pos = 0; }
        const uint32_t word = (uint32_t)pos / 32, shift = pos % 32;
        atomicOr(&stays[word], m << shift);
        if (shift > 32 - kChunk && word + 1 < kFlatElements / 32) atomicOr(&stays[word + 1], m >> (32 - shift));
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kFlatVectors; ++j) {
        const uint64_t f = at + j * kThreads * kChunk;
        if (f >= total) break;
        const uint32_t m = ((const uint8_t *)stays)[threadIdx.x + j * kThreads];
        if (f + kChunk <= total) {
            Chunk v = unpack(r[j]);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                const float2 s = __fmul2_rn(v.p[i], both(d.scale));
                v.p[i] = make_float2(m >> 2 * i & 1 ? s.x : 0.f, m >> (2 * i + 1) & 1 ? s.y : 0.f);
            }
            store_words(pack<T>(v), y + f);
        } else {
            for (uint32_t e = 0; f + e < total; ++e) y[f + e] = from_f32<T>(m >> e & 1 ? to_f32(x[f + e]) * d.scale : 0.f);
        }
    }
}

// ------------------------------------------------------------------- norm --
struct NormArgs {
    const void *x, *res, *weight;
    void *y, *h;
    float *rstd;
    uint8_t *codes;  // 8-bit output instead of y
    float *scales;
    uint32_t rows, x_stride, res_stride, y_stride, h_stride, code_stride;  // pitches in elements
    uint32_t dim;
    int w_f32, plain;  // plain: no norm, the rows themselves are encoded
    float eps, inv_dim;
    Drop drop;
};

// Sum over the `lanes` (power of two, at most 32) of a row's group, or over the whole block: through
// `shared`, a word a warp, which the block's next call but one may use again (one barrier a call).
template <bool BLOCK> __device__ __forceinline__ float row_sum(float v, uint32_t lanes, float *shared) {
#pragma unroll
    for (uint32_t o = 16; o > 0; o /= 2)
        if (BLOCK || o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (BLOCK) {
        if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
        for (uint32_t i = 0; i < blockDim.x / 32; ++i) v += shared[i];
    }
    return v;
}

// Scale of a block of 128 columns whose largest magnitude has the bits `top` (as bits NaN lies above
// infinity above every number), and its reciprocal.  The scale puts that magnitude on 448; a block with an infinity or
// NaN gets a NaN scale, so that every value read from it is NaN.  At least the least normal
// f32, so that the reciprocal is finite.  Its approximation is good to one step and products are
// rounded once: a code is off by half a step and 2^-22 of the value.
__device__ __forceinline__ float scale_of(uint32_t top, float &inv) {
    const bool bad = top >= 0x7F800000u;
    const float scale = bad ? __uint_as_float(0x7FC00000u) : fmaxf(__uint_as_float(top) * (1.f / kE4M3Max), 1.17549435e-38f);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
    if (bad) inv = 0.f;
    return scale;
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// A reciprocal of 0 (a block that is not finite) gives codes of 0 or NaN: its scale is NaN anyway.
__device__ __forceinline__ uint32_t code2(float2 v, float inv) {
    return __nv_cvt_float2_to_fp8x2(__fmul2_rn(v, both(inv)), __NV_SATFINITE, __NV_E4M3);
}

// e4m3 codes and scales of a group's step; the whole warp calls this.
template <int MODE>
__device__ __forceinline__ void encode_columns(const Chunk &v, const Columns<MODE> &c, uint32_t lane, uint32_t lanes, uint32_t dim, uint8_t *codes, float *scales) {
    if (MODE == kWhole) {  // the 16 lanes of a block reduce; a chunk lies in one block
        uint32_t top = 0;
#pragma unroll
        for (uint32_t i = 0; i < kChunk; ++i) top = max(top, magnitude(at(v, i)));
        #pragma unroll
        for (uint32_t o = 8; o > 0; o /= 2)
            if (o < lanes) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (c.first >= dim) return;
        float inv;
        const float scale = scale_of(top, inv);
        if (c.first % kF8Block == 0) scales[c.first / kF8Block] = scale;
        *(uint2 *)(codes + c.first) = make_uint2(code2(v.p[0], inv) | code2(v.p[1], inv) << 16, code2(v.p[2], inv) | code2(v.p[3], inv) << 16);
    } else {  // 32 lanes: columns 0 - 3 of each thread are one block, 4 - 7 the next; fewer lanes have at most one block
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (uint32_t i = 0; i < kChunk / 2; ++i) { lo = max(lo, magnitude(at(v, i))); hi = max(hi, magnitude(at(v, i + kChunk / 2))); }
        if (lanes < 32) lo = hi = max(lo, hi);
#pragma unroll
        for (uint32_t o = 16; o > 0; o /= 2) {
            if (o >= lanes) continue;
            lo = max(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        float inv_lo, inv_hi;
        const float scale_lo = scale_of(lo, inv_lo), scale_hi = scale_of(hi, inv_hi);
        if (lane == 0) {
            if (c.first < dim) scales[c.first / kF8Block] = scale_lo;
            if (lanes == 32 && c.first + kF8Block < dim) scales[c.first / kF8Block + 1] = scale_hi;
        }
        if constexpr (MODE == kPair) {
#pragma unroll
            for (uint32_t i = 0; i < kChunk / 2; ++i)
                if (c.at(2 * i) < dim) *(uint16_t *)(codes + c.at(2 * i)) = (uint16_t)code2(v.p[i], i < kChunk / 4 ? inv_lo : inv_hi);
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kChunk; ++i)
            if (c.at(i) < dim) codes[c.at(i)] = (uint8_t)code2(make_float2(at(v, i), 0.f), i < kChunk / 2 ? inv_lo : inv_hi);
    }
}

// h = res + dropout(x); y = h rsqrt(mean(h^2) + eps) w.  `lanes` lanes a row (BLOCK: the whole
// block), C chunks each; the row stays in registers between the sum and the output, so memory is gone
// through once.  524 288 x 512 bf16 with residual to 8 bits: 288 us, the measured copy rate; 16 384 x 4096
// f16: 50 us (0.83); 38 411 x 256 bf16 with residual and dropout: 17 us (0.70, instructions); 20 011 x 602 f32,
// not aligned, the same: 32 us (0.93).  16-bit rows that are not aligned are bound by instructions: 300 000 x 100
// bf16 with residual to 8 bits 60 us in pairs (0.54), 77 in single elements.
// L: the lanes of a row where they are known (rows that are not aligned: their strides are then constants), else 0.
template <typename T, int MODE, int C, bool BLOCK, bool F8, int L>
__global__ void __launch_bounds__(BLOCK ? 512 : kThreads, BLOCK ? (sizeof(T) * C <= 8 ? 2 : 1) : C == 1 ? 5 : 4)
k_norm(const NormArgs a, uint32_t log2_lanes) {
    const uint32_t lanes = C > 1 || BLOCK ? 32 : L ? L : 1u << log2_lanes;  // more chunks than one: all lanes
    __shared__ float shared[32];
    __shared__ uint4 lots[MODE == kWhole ? 1 : BLOCK ? 512 : kThreads];
    uint4 *warp_lots = MODE == kWhole ? lots : lots + (threadIdx.x & ~31u);
    const uint32_t lane = threadIdx.x & (lanes - 1), group_chunk = BLOCK ? threadIdx.x & ~31u : 0, width = BLOCK ? blockDim.x : lanes;
    const uint32_t row = BLOCK ? blockIdx.x : blockIdx.x * (kThreads >> log2_lanes) + (threadIdx.x >> log2_lanes);
    const uint32_t dim = row < a.rows ? a.dim : 0;  // lanes without a row still take part in the exchanges
    Chunk v[C], w[C];
    {
        const T *x = (const T *)a.x + (uint64_t)row * a.x_stride, *res = (const T *)a.res + (uint64_t)row * a.res_stride;
        Raw<T> rx[C], rr[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const Columns<MODE> c(lane, lanes, j * width + group_chunk);
            if (c.first >= dim) continue;
            rx[j] = load_chunk<T, MODE>(x, c, dim);
            if (a.res) rr[j] = load_chunk<T, MODE>(res, c, dim);
            if (C == 1) w[j] = load_weight<T, MODE>(a.weight, a.w_f32, c, dim);  // early, where it costs few registers
        }
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const uint32_t step = j * width + group_chunk;
            const Columns<MODE> c(lane, lanes, step);
            v[j] = c.first < dim ? unpack(rx[j]) : filled(0.f);
            if (a.drop.on) drop_columns<MODE>(a.drop, row, lane, lanes, step, warp_lots, v[j]);
            if (a.res && c.first < dim) {
                const Chunk r = unpack(rr[j]);
#pragma unroll
                for (int i = 0; i < kPairs; ++i) v[j].p[i] = __fadd2_rn(v[j].p[i], r.p[i]);
            }
        }
    }
    if (a.h) {
        T *h = (T *)a.h + (uint64_t)row * a.h_stride;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const Columns<MODE> c(lane, lanes, j * width + group_chunk);
            if (c.first < dim) store_chunk<T, MODE>(h, c, dim, v[j]);
        }
    }
    if (!a.plain) {
        float2 sum = both(0.f);
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
            for (int i = 0; i < kPairs; ++i) sum = __ffma2_rn(v[j].p[i], v[j].p[i], sum);
        const float rstd = rsqrtf(row_sum<BLOCK>(sum.x + sum.y, lanes, shared) * a.inv_dim + a.eps);
        if (a.rstd && dim && (BLOCK ? threadIdx.x : lane) == 0) a.rstd[row] = rstd;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const Columns<MODE> c(lane, lanes, j * width + group_chunk);
            if (c.first >= dim) continue;
            if (C > 1) w[j] = load_weight<T, MODE>(a.weight, a.w_f32, c, dim);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[j].p[i] = __fmul2_rn(v[j].p[i], __fmul2_rn(w[j].p[i], both(rstd)));
        }
    }
    T *y = (T *)a.y + (uint64_t)row * a.y_stride;
    uint8_t *codes = a.codes + (uint64_t)row * a.code_stride;
    float *scales = a.scales + (uint64_t)row * ((a.dim + kF8Block - 1) / kF8Block);
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const Columns<MODE> c(lane, lanes, j * width + group_chunk);
        if (F8) encode_columns<MODE>(v[j], c, lane, lanes, dim, codes, scales);
        else if (c.first < dim) store_chunk<T, MODE>(y, c, dim, v[j]);
    }
}

struct NormBackArgs {
    const void *dy, *dh, *h, *weight;
    const void *x, *res;  // h null: what h is made of (16-bit rows)
    const float *rstd;
    void *dx, *dres;
    float *partial;  // [blocks, dim] sums of dy h rstd over a block's rows, or null
    uint32_t rows, dy_stride, dh_stride, h_stride, x_stride, res_stride;
    uint32_t dim;
    int w_f32;
    float inv_dim;
    Drop drop;
};

// g = dy w; t = dh + rstd g - h rstd^3 / dim sum(g h): the gradient of h and of the residual; dx = dropout(t).
// dw = sum over rows of dy h rstd: a thread's columns are the same in every row, so it keeps their
// sums; a block adds its lane groups in order into its row of `partial`, and k_norm_dw adds those.
// No atomics: the same bits every time on the same GPU.  Everything is computed from the h of 32 bits that the forward
// pass normalised: f32 rows (and x alone) hold it, for 16-bit rows it is made again from x and residual, which is
// one tensor more to read than the rounded h where there is a residual.
//
// 16 384 x 4096 f16: 101 us (0.81 of the copy rate), 38 411 x 256 bf16 with residual and dropout 25 us (0.73), 20 011 x 602 f32
// 42 us (0.88).  What is made again costs its bytes: 38 411 x 256 bf16 took 21 us from the rounded h, 16 384 x 4096 bf16 with
// residual, forward and backward, 187 where it takes 207.
// Bound by instructions with 16 to 32 warps an SM: bringing the next row into shared memory meanwhile (cp.async) made
// it slower (139 us where this took 122), leaving the ragged path out of the aligned kernel faster (122 to 102).
// AGAIN: h may have to be made again.  The mask is then needed twice and kept as bits; else it is made where dx is.
template <typename T, int MODE, int C, bool BLOCK, int L, bool AGAIN>
__global__ void __launch_bounds__(BLOCK ? 512 : kThreads, BLOCK ? (C == 1 ? 2 : 1) : C == 1 ? 4 : 2)
k_norm_back(const NormBackArgs a, uint32_t log2_lanes) {
    const uint32_t lanes = C > 1 || BLOCK ? 32 : L ? L : 1u << log2_lanes;
    __shared__ float shared[32];
    __shared__ uint4 lots[MODE == kWhole ? 1 : BLOCK ? 512 : kThreads];
    extern __shared__ float sums[];  // [groups of the block][dim], not BLOCK
    uint4 *warp_lots = MODE == kWhole ? lots : lots + (threadIdx.x & ~31u);
    const uint32_t lane = threadIdx.x & (lanes - 1), group_chunk = BLOCK ? threadIdx.x & ~31u : 0, width = BLOCK ? blockDim.x : lanes;
    const uint32_t per_block = BLOCK ? 1 : kThreads >> log2_lanes;
    Chunk dw[C];
#pragma unroll
    for (int j = 0; j < C; ++j) dw[j] = filled(0.f);
    uint32_t turn = 0;
    for (uint32_t base = blockIdx.x * per_block; base < a.rows; base += gridDim.x * per_block, turn ^= 16) {  // rows + a grid's worth fit 32 bits
        const uint32_t row = base + (BLOCK ? 0 : threadIdx.x >> log2_lanes);
        const uint32_t dim = row < a.rows ? a.dim : 0;
        const bool again = AGAIN && !a.h;
        const T *h_row = again ? (const T *)a.x + (uint64_t)row * a.x_stride : (const T *)a.h + (uint64_t)row * a.h_stride,
                *res_row = (const T *)a.res + (uint64_t)row * a.res_stride, *dy_row = (const T *)a.dy + (uint64_t)row * a.dy_stride,
                *dh_row = (const T *)a.dh + (uint64_t)row * a.dh_stride;
        Raw<T> ry[C], rh[C], rd[C], rr[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const Columns<MODE> c(lane, lanes, j * width + group_chunk);
            ry[j] = rh[j] = rd[j] = rr[j] = Raw<T>{};
            if (c.first >= dim) continue;
            rh[j] = load_chunk<T, MODE>(h_row, c, dim);
            if (again && a.res) rr[j] = load_chunk<T, MODE>(res_row, c, dim);
            if (a.dy) ry[j] = load_chunk<T, MODE>(dy_row, c, dim);
            if (a.dh) rd[j] = load_chunk<T, MODE>(dh_row, c, dim);
        }
        const float rstd = dim ? a.rstd[row] : 0.f;
        Chunk gw[C], h[C];  // dy w and h
        uint32_t stay[C];
        float2 sum = both(0.f);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const uint32_t step = j * width + group_chunk;
            const Columns<MODE> c(lane, lanes, step);
            if (AGAIN && a.drop.on) stay[j] = stay_columns<MODE>(a.drop, row, lane, lanes, step, warp_lots);
            const Chunk g = unpack(ry[j]), w = c.first < dim ? load_weight<T, MODE>(a.weight, a.w_f32, c, dim) : filled(0.f);
            h[j] = unpack(rh[j]);
            if (again) {
                if (a.drop.on) drop_by_bits(a.drop, stay[j], h[j]);
                const Chunk r = unpack(rr[j]);
#pragma unroll
                for (int i = 0; i < kPairs; ++i) if (a.res) h[j].p[i] = __fadd2_rn(h[j].p[i], r.p[i]);
            }
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                dw[j].p[i] = __ffma2_rn(__fmul2_rn(g.p[i], h[j].p[i]), both(rstd), dw[j].p[i]);
                gw[j].p[i] = __fmul2_rn(g.p[i], w.p[i]);
                sum = __ffma2_rn(gw[j].p[i], h[j].p[i], sum);
            }
        }
        const float coef = -row_sum<BLOCK>(sum.x + sum.y, lanes, shared + turn) * rstd * rstd * rstd * a.inv_dim;
        T *dres = (T *)a.dres + (uint64_t)row * a.dim, *dx = (T *)a.dx + (uint64_t)row * a.dim;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const uint32_t step = j * width + group_chunk;
            const Columns<MODE> c(lane, lanes, step);
            Chunk t = unpack(rd[j]);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) t.p[i] = __fadd2_rn(t.p[i], __ffma2_rn(gw[j].p[i], both(rstd), __fmul2_rn(h[j].p[i], both(coef))));
            if (a.dres && c.first < dim) store_chunk<T, MODE>(dres, c, dim, t);
            if (a.dx) {
                if (AGAIN && a.drop.on) drop_by_bits(a.drop, stay[j], t);
                else if (a.drop.on) drop_columns<MODE>(a.drop, row, lane, lanes, step, warp_lots, t);
                if (c.first < dim) store_chunk<T, MODE>(dx, c, dim, t);
            }
        }
    }
    if (!a.partial) return;
    float *mine = a.partial + (uint64_t)blockIdx.x * a.dim;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const Columns<MODE> c(lane, lanes, j * width + group_chunk);
        float *to = BLOCK ? mine : sums + (threadIdx.x >> log2_lanes) * a.dim;
#pragma unroll
        for (uint32_t i = 0; i < kChunk; ++i)
            if (c.at(i) < a.dim) to[c.at(i)] = at(dw[j], i);
    }
    if (BLOCK) return;
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
        float s = 0.f;
        for (uint32_t q = 0; q < per_block; ++q) s += sums[q * a.dim + c];
        mine[c] = s;
    }
}

// dw[c] = sum of the blocks' partial sums: COLS columns a block, 1024 / COLS slices of the rows.  Eight columns
// (a sector of every partial row) as long as that is no more than one block per SM, 32 beyond: 602
// columns (19 blocks of 32) 9.5 and 5.8 us, 4096 columns (512 blocks of 8) 5.6 and 9.8.
template <typename T, uint32_t kDwCols>
__global__ void __launch_bounds__(1024)
k_norm_dw(const float *partial, uint32_t blocks, uint32_t dim, T *dw) {
    chain_sync();  // launched as a programmatic dependent of k_norm_back
    constexpr uint32_t kDwSlices = 1024 / kDwCols;
    __shared__ float sums[kDwSlices][kDwCols + 1];
    const uint32_t c = blockIdx.x * kDwCols + threadIdx.x;
    float s = 0.f;
    if (c < dim) {
#pragma unroll 8
        for (uint32_t b = threadIdx.y; b < blocks; b += kDwSlices) s += partial[(uint64_t)b * dim + c];
    }
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    const uint32_t thread = threadIdx.y * kDwCols + threadIdx.x, column = thread / 32, lane = thread % 32, out = blockIdx.x * kDwCols + column;
    if (column >= kDwCols) return;
    s = 0.f;
#pragma unroll
    for (uint32_t q = 0; q < kDwSlices / 32; ++q) s += sums[q * 32 + lane][column];
#pragma unroll
    for (uint32_t o = 16; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0 && out < dim) dw[out] = from_f32<T>(s);
}

// ---------------------------------------------------- weights in 8 bits --
// A block of 128 x 128 weights per thread block: its largest magnitude, then the codes.
template <typename T>
__global__ void __launch_bounds__(kThreads)
k_encode_weight(const T *w, uint64_t out, uint32_t dim, uint64_t stride, uint8_t *codes, uint64_t code_stride, float *scales) {
    __shared__ uint32_t peak;
    if (threadIdx.x == 0) peak = 0;
    __syncthreads();
    const uint32_t blocks_per_row = (dim + kF8Block - 1) / kF8Block;
    const uint32_t bk = blockIdx.x % blocks_per_row;
    const uint64_t bn = blockIdx.x / blocks_per_row;
    uint32_t top = 0;
    for (uint32_t i = threadIdx.x; i < kF8Block * kF8Block; i += kThreads) {
        const uint64_t n = bn * kF8Block + i / kF8Block;
        const uint32_t c = bk * kF8Block + i % kF8Block;
        if (n < out && c < dim) top = max(top, magnitude(to_f32(w[n * stride + c])));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) atomicMax(&peak, top);
    __syncthreads();
    float inv;
    const float scale = scale_of(peak, inv);
    if (threadIdx.x == 0) scales[blockIdx.x] = scale;
    for (uint32_t i = threadIdx.x; i < kF8Block * kF8Block; i += kThreads) {
        const uint64_t n = bn * kF8Block + i / kF8Block;
        const uint32_t c = bk * kF8Block + i % kF8Block;
        if (n < out && c < dim)
            codes[n * code_stride + c] = (uint8_t)code2(make_float2(to_f32(w[n * stride + c]), 0.f), inv);
    }
}

// --------------------------------------------------------------- launches --
// Whether every row of a tensor starts on a multiple of eight elements' bytes.
bool vec_rows(const void *p, uint64_t stride, uint32_t elem) {
    return !p || ((uintptr_t)p % (kChunk * elem) == 0 && stride % kChunk == 0);
}

// Whether pairs of its 16-bit elements are words, and pairs of f32 weights eight bytes.
bool pair_rows(const void *p, uint64_t stride, uint32_t elem) { return !p || ((uintptr_t)p % (2 * elem) == 0 && stride % 2 == 0); }
// f(std::integral_constant<int, MODE>) of the ways that rows of type T are walked.
template <typename T, typename F> auto with_mode(bool vec, bool pairs, F f) {
    if (vec) return f(std::integral_constant<int, kWhole>{});
    if constexpr (sizeof(T) == 2)
        if (pairs) return f(std::integral_constant<int, kPair>{});
    return f(std::integral_constant<int, kSingle>{});
}

template <typename F> void with_type(int dtype, F f) {
    if (dtype == AG_F32) f((float *)nullptr);
    else if (dtype == AG_F16) f((__half *)nullptr);
    else f((__nv_bfloat16 *)nullptr);
}

int32_t make_drop(double p, uint64_t seed, uint64_t offset, Drop *d) {
    if (!(p >= 0.0 && p <= 1.0)) return fail(AG_ERR_VALUE, "dropout probability must be in [0, 1], got %g", p);
    const uint32_t t = (uint32_t)std::floor(p * 65536.0 + 0.5);
    d->on = t != 0;
    d->bar = (uint32_t)(((uint64_t)t << 16) - 1);  // t = 65536: nothing is above
    d->scale = t < 65536 ? 65536.0f / (65536 - t) : 0.0f;
    d->seed = seed; d->offset = offset;
    return AG_OK;
}

int32_t check_rows(const char *who, uint64_t rows, uint64_t dim, int32_t dtype) {
    if (dtype < AG_F32 || dtype > AG_BF16) return fail(AG_ERR_VALUE, "%s: rows are f32, f16 or bf16, got dtype tag %d", who, dtype);
    if (rows > 0xF0000000ull) return fail(AG_ERR_VALUE, "%s: at most 0xF0000000 rows, got %llu", who, (unsigned long long)rows);
    if (dim == 0 || dim > 0xFFFFFFF0ull) return fail(AG_ERR_VALUE, "%s: rows of 1 to 2^32 - 16 columns, got %llu", who, (unsigned long long)dim);
    return AG_OK;
}

int32_t check_pitches(const char *who, std::initializer_list<uint64_t> pitches) {
    for (const uint64_t p : pitches)
        if (p > 0xFFFFFFFFull) return fail(AG_ERR_VALUE, "%s: rows at most 2^32 - 1 elements apart, got %llu", who, (unsigned long long)p);
    return AG_OK;
}

// How a row of `dim` columns is shared out: `lanes` of a warp (0: a whole block of `threads`) with up to
// `chunks` chunks each.  Whole blocks: as few threads as hold the row in
// `most` chunks each (64 bytes of f16 / bf16 or f32: a thread's loads are all in flight together, and the sum
// waits for fewer warps), unless that leaves many of them idle; a chunk each where there are no more rows than
// SMs, and the time is one row's latency, and in the backward pass over rows that are not aligned (registers); two where the backward
// pass makes h again through a mask, as long as the row fits (registers).  16 384 rows of 4096 bf16 with residual, forward and
// backward: two chunks 250 us, four 256; without dropout 219 and 207.  16 384 rows of 4096 f16, forward: four chunks 52 us, two 64, one 66.
struct Split {
    uint32_t lanes, threads;
    int chunks;
    uint32_t log2_lanes() const { uint32_t l = 0; while ((1u << l) < lanes) ++l; return lanes ? l : 5; }
};
Split split_row(uint64_t rows, uint32_t dim, int dtype, bool vec, bool backward, bool mask_again = false) {
    const uint32_t n = (dim + kChunk - 1) / kChunk;
    Split s{1, kThreads, 1};
    if (!vec) s.lanes = 4;
    if (n <= (!vec && backward ? 32u : 64u)) {
        while (s.lanes < 32 && s.lanes < n) s.lanes *= 2;
        while ((uint32_t)s.chunks * s.lanes < n) s.chunks *= 2;
        return s;
    }
    s.lanes = 0;
    const int most = rows <= (uint64_t)kSMs || (!vec && backward) ? 1 : dtype == AG_F32 || mask_again ? 2 : 4;
    uint32_t slots = 0xFFFFFFFFu;
    for (int c = most; c; c /= 2) {
        const uint32_t threads = (n + 32 * c - 1) / (32 * c) * 32;
        if (threads > 512 || threads * c + threads * c / 8 >= slots) continue;
        slots = threads * c; s.threads = threads; s.chunks = c;
    }
    if (slots == 0xFFFFFFFFu) {  // longer than that many chunks a thread
        s.chunks = n <= 1024 ? 2 : 4;
        s.threads = (n + 32 * s.chunks - 1) / (32 * s.chunks) * 32;
    }
    return s;
}

// f(std::integral_constant<int, L>) for the lanes of a row that is not aligned; 0 for others.
template <int MODE, typename F> auto with_lanes(uint32_t lanes, F f) {
    if constexpr (MODE == kWhole) return f(std::integral_constant<int, 0>{});
    else return lanes == 4 ? f(std::integral_constant<int, 4>{}) : lanes == 8 ? f(std::integral_constant<int, 8>{}) :
                lanes == 16 ? f(std::integral_constant<int, 16>{}) : f(std::integral_constant<int, 32>{});
}

template <typename T, int MODE, bool F8>
cudaError_t launch_norm(const NormArgs &a, int dtype, cudaStream_t st) {
    const Split s = split_row(a.rows, a.dim, dtype, MODE == kWhole, false);
    const uint64_t per = s.lanes ? s.threads / s.lanes : 1;
    const uint32_t grid = (uint32_t)((a.rows + per - 1) / per), lanes = s.log2_lanes();  // rows of a whole block are 1 KB and more
    if (s.lanes) {
        if (s.chunks == 1)
            with_lanes<MODE>(s.lanes, [&](auto l) { k_norm<T, MODE, 1, false, F8, decltype(l)::value><<<grid, s.threads, 0, st>>>(a, lanes); });
        else k_norm<T, MODE, 2, false, F8, 0><<<grid, s.threads, 0, st>>>(a, lanes);
    } else {
        if (s.chunks == 1) k_norm<T, MODE, 1, true, F8, 0><<<grid, s.threads, 0, st>>>(a, lanes);
        else if (s.chunks == 2) k_norm<T, MODE, 2, true, F8, 0><<<grid, s.threads, 0, st>>>(a, lanes);
        else k_norm<T, MODE, 4, true, F8, 0><<<grid, s.threads, 0, st>>>(a, lanes);
    }
    return cudaGetLastError();
}

// Blocks of the backward pass: those that are resident together, `per_sm` of them on each SM, and no more
// than there are rows for.
uint32_t back_blocks(uint64_t rows, const Split &s, uint32_t per_sm) {
    const uint64_t per = s.lanes ? s.threads / s.lanes : 1;
    return (uint32_t)std::min<uint64_t>((rows + per - 1) / per, (uint64_t)kSMs * per_sm);
}
uint32_t back_blocks_bound(uint64_t rows, uint32_t dim, int dtype) {
    uint32_t most = 0;
    for (const int form : {0, 1, 3}) {
        const Split s = split_row(rows, dim, dtype, form & 1, true, form & 2);
        most = std::max(most, back_blocks(rows, s, std::min(2048 / s.threads, 32u)));
    }
    return most;
}

template <typename T, int MODE, int C, bool BLOCK, int L = 0, bool AGAIN = sizeof(T) == 2>
cudaError_t launch_back(const NormBackArgs &a, const Split &s, uint32_t &grid, cudaStream_t st) {
    const size_t shared = BLOCK || !a.partial ? 0 : (size_t)(s.threads / s.lanes) * a.dim * 4;
    static std::atomic<int> known[17];  // blocks of 32 i threads that an SM holds; registers decide, not the sums' shared memory
    int per_sm = known[s.threads / 32].load(std::memory_order_relaxed);
    if (per_sm == 0) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k_norm_back<T, MODE, C, BLOCK, L, AGAIN>, (int)s.threads, shared);
        if (e != cudaSuccess) return e;
        per_sm = std::max(1, per_sm);
        known[s.threads / 32].store(per_sm, std::memory_order_relaxed);
    }
    grid = back_blocks(a.rows, s, per_sm);
    k_norm_back<T, MODE, C, BLOCK, L, AGAIN><<<grid, s.threads, shared, st>>>(a, s.log2_lanes());
    return cudaGetLastError();
}

template <typename T, int MODE>
cudaError_t launch_back(const NormBackArgs &a, int dtype, uint32_t &grid, cudaStream_t st) {
    const Split s = split_row(a.rows, a.dim, dtype, MODE == kWhole, true, !a.h && a.drop.on);
    if (s.lanes) {
        if (s.chunks == 1) return with_lanes<MODE>(s.lanes, [&](auto l) { return launch_back<T, MODE, 1, false, decltype(l)::value>(a, s, grid, st); });
        return launch_back<T, MODE, 2, false>(a, s, grid, st);
    }
    if (s.chunks == 1) return launch_back<T, MODE, 1, true>(a, s, grid, st);
    if (s.chunks == 2) return launch_back<T, MODE, 2, true>(a, s, grid, st);
    if constexpr (sizeof(T) == 2)
        if (!a.h) return launch_back<T, MODE, 4, true, 0, true>(a, s, grid, st);
    return launch_back<T, MODE, 4, true, 0, false>(a, s, grid, st);  // without the registers that the other needs
}

}  // namespace

}  // namespace ag

namespace ag {

namespace {
__global__ void k_scales_bad(const float *scales, uint64_t n, uint32_t *bad) {
    for (uint64_t i = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x)
        if (isnan(scales[i])) *bad = 1;
}

// A row a block, for rows of any length; encode_columns does the work.
__global__ void __launch_bounds__(kThreads)
k_encode_rows(const float *src, uint64_t rows, uint32_t dim, uint64_t pitch, uint8_t *codes, float *scales) {
    const uint64_t per_row = (dim + kF8Block - 1) / kF8Block;
    for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x)
        for (uint32_t c0 = 0; c0 < dim; c0 += kThreads * kChunk) {
            const uint32_t lane = threadIdx.x & 31;
            const Columns<kSingle> c(lane, 32, c0 / kChunk + (threadIdx.x & ~31u));
            const Chunk v = unpack(load_chunk<float, kSingle>(src + row * dim, c, dim));
            encode_columns<kSingle>(v, c, lane, 32, dim, codes + row * pitch, scales + row * per_row);
        }
}
}  // namespace

cudaError_t launch_encode_f8(const float *src, uint64_t rows, uint64_t dim, uint64_t pitch, uint8_t *codes, float *scales,
                             uint32_t *bad_dev, cudaStream_t st) {
    k_encode_rows<<<(uint32_t)std::min<uint64_t>(rows, 1u << 20), kThreads, 0, st>>>(src, rows, (uint32_t)dim, pitch, codes, scales);
    k_scales_bad<<<(uint32_t)kSMs * 4, kThreads, 0, st>>>(scales, rows * ((dim + kF8Block - 1) / kF8Block), bad_dev);
    return cudaGetLastError();
}

}  // namespace ag

using namespace ag;

extern "C" int32_t ag_rows_dropout(const void *x, void *y, uint64_t rows, uint64_t dim, uint64_t x_stride, uint64_t y_stride,
                                   int32_t dtype, double p, uint64_t seed, uint64_t offset, int32_t device, void *stream) {
    AG_TRY(check_rows("ag_rows_dropout", rows, dim, dtype));
    Drop d;
    AG_TRY(make_drop(p, seed, offset, &d));
    if (rows == 0) return AG_OK;
    if (!x || !y) return fail(AG_ERR_VALUE, "ag_rows_dropout: null argument");
    if (y_stride < dim) return fail(AG_ERR_VALUE, "ag_rows_dropout: rows of the output overlap");
    if (x == y && x_stride != y_stride && rows > 1)  // a row would be written over another that is still to be read
        return fail(AG_ERR_VALUE, "ag_rows_dropout: in place, both pitches are the same: got %llu and %llu", (unsigned long long)x_stride, (unsigned long long)y_stride);
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    const Divide by((uint32_t)((dim + kChunk - 1) / kChunk));
    const uint64_t chunks = rows * by.by;
    if (chunks >= (1ull << 38)) return fail(AG_ERR_VALUE, "ag_rows_dropout: too many rows of this length");  // beyond any memory
    if (!d.on && x == y) return AG_OK;
    const uint32_t grid = (uint32_t)((chunks + 2 * kThreads - 1) / (2 * kThreads));
    const bool vec = vec_rows(x, x_stride, elem_size(dtype)) && vec_rows(y, y_stride, elem_size(dtype));
    const bool flat = d.on && dim % kChunk && dim < kFlatMaxDim && (x_stride == dim || rows == 1) && (y_stride == dim || rows == 1) && vec_rows(x, 0, elem_size(dtype)) &&
                      vec_rows(y, 0, elem_size(dtype));
    with_type(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (flat) k_dropout_flat<T><<<(uint32_t)((rows * dim + kFlatElements - 1) / kFlatElements), kThreads, 0, (cudaStream_t)stream>>>(
            (const T *)x, (T *)y, rows * dim, Divide((uint32_t)dim), by, d);
        else if (vec && dim % kChunk == 0) k_dropout<T, kWhole, false><<<grid, kThreads, 0, (cudaStream_t)stream>>>((const T *)x, (T *)y, chunks, (uint32_t)dim, by, x_stride, y_stride, d);
        else if (vec) k_dropout<T, kWhole, true><<<grid, kThreads, 0, (cudaStream_t)stream>>>((const T *)x, (T *)y, chunks, (uint32_t)dim, by, x_stride, y_stride, d);
        else k_dropout<T, kSingle, true><<<grid, kThreads, 0, (cudaStream_t)stream>>>((const T *)x, (T *)y, chunks, (uint32_t)dim, by, x_stride, y_stride, d);
    });
    AG_CUDA(cudaGetLastError());
    return AG_OK;
}

extern "C" int32_t ag_rows_norm(const ag_norm *n, int32_t device, void *stream) {
    if (!n) return fail(AG_ERR_VALUE, "ag_rows_norm: null argument");
    AG_TRY(check_rows("ag_rows_norm", n->rows, n->dim, n->dtype));
    if (n->dim > kMaxNormDim) return fail(AG_ERR_VALUE, "ag_rows_norm: at most %u columns, got %llu", kMaxNormDim, (unsigned long long)n->dim);
    if (n->weight && n->weight_dtype != n->dtype && n->weight_dtype != AG_F32)
        return fail(AG_ERR_VALUE, "ag_rows_norm: the weights are f32 or of the rows' type");
    NormArgs a{};
    AG_TRY(make_drop(n->p, n->seed, n->offset, &a.drop));
    if (n->rows == 0) return AG_OK;
    if (!n->x || (!n->y && !n->codes) || (n->codes && !n->scales)) return fail(AG_ERR_VALUE, "ag_rows_norm: null argument");
    if (n->y && n->codes) return fail(AG_ERR_VALUE, "ag_rows_norm: either rows of their own type or 8-bit rows come out");
    if (!n->encode_only && !(n->eps >= 0.f)) return fail(AG_ERR_VALUE, "ag_rows_norm: eps must not be negative, got %g", n->eps);
    if (n->encode_only && (!n->codes || n->residual || n->weight || n->h || a.drop.on))
        return fail(AG_ERR_VALUE, "ag_rows_norm: encoding alone takes rows and gives 8-bit rows");
    if (n->codes && (n->code_stride % 16 != 0 || n->code_stride < n->dim || (uintptr_t)n->codes % 16 != 0))
        return fail(AG_ERR_VALUE, "ag_rows_norm: 8-bit rows start on multiples of 16 bytes and do not overlap");
    AG_TRY(check_pitches("ag_rows_norm", {n->x_stride, n->residual_stride, n->y_stride, n->h_stride, n->code_stride}));
    if ((n->y && n->y_stride < n->dim) || (n->h && n->h_stride < n->dim)) return fail(AG_ERR_VALUE, "ag_rows_norm: rows of the output overlap");
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    a.x = n->x; a.res = n->residual; a.weight = n->weight; a.y = n->y; a.h = n->h; a.rstd = n->rstd;
    a.codes = (uint8_t *)n->codes; a.scales = n->scales; a.rows = (uint32_t)n->rows; a.x_stride = (uint32_t)n->x_stride; a.res_stride = (uint32_t)n->residual_stride;
    a.y_stride = (uint32_t)n->y_stride; a.h_stride = (uint32_t)n->h_stride; a.code_stride = (uint32_t)n->code_stride; a.dim = (uint32_t)n->dim;
    a.w_f32 = n->weight_dtype == AG_F32; a.plain = n->encode_only; a.eps = n->eps; a.inv_dim = 1.0f / (float)n->dim;
    const uint32_t e = elem_size(n->dtype);
    const bool vec = a.dim % kChunk == 0 && vec_rows(a.weight, 0, elem_size(n->weight_dtype)) && vec_rows(a.x, a.x_stride, e) && vec_rows(a.res, a.res_stride, e) && vec_rows(a.y, a.y_stride, e) && vec_rows(a.h, a.h_stride, e);
    const bool pairs = a.dim % 2 == 0 && pair_rows(a.weight, 0, elem_size(n->weight_dtype)) && pair_rows(a.x, a.x_stride, e) && pair_rows(a.res, a.res_stride, e) &&
                       pair_rows(a.y, a.y_stride, e) && pair_rows(a.h, a.h_stride, e);
    cudaError_t err = cudaSuccess;
    with_type(n->dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        cudaStream_t st = (cudaStream_t)stream;
        err = with_mode<T>(vec, pairs, [&](auto mode) {
            return a.codes ? launch_norm<T, decltype(mode)::value, true>(a, n->dtype, st) : launch_norm<T, decltype(mode)::value, false>(a, n->dtype, st);
        });
    });
    AG_CUDA(err);
    return AG_OK;
}

extern "C" int32_t ag_rows_norm_backward_scratch(uint64_t rows, uint64_t dim, int32_t dtype, int32_t device, uint64_t *bytes) {
    if (!bytes) return fail(AG_ERR_VALUE, "ag_rows_norm_backward_scratch: null argument");
    *bytes = 0;
    if (rows == 0 || dim == 0 || dim > kMaxNormDim) return AG_OK;
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    *bytes = (uint64_t)back_blocks_bound(rows, (uint32_t)dim, dtype) * dim * 4;
    return AG_OK;
}

extern "C" int32_t ag_rows_norm_backward(const ag_norm_grad *n, int32_t device, void *stream) {
    if (!n) return fail(AG_ERR_VALUE, "ag_rows_norm_backward: null argument");
    AG_TRY(check_rows("ag_rows_norm_backward", n->rows, n->dim, n->dtype));
    if (n->dim > kMaxNormDim) return fail(AG_ERR_VALUE, "ag_rows_norm_backward: at most %u columns, got %llu", kMaxNormDim, (unsigned long long)n->dim);
    if ((n->weight || n->dw) && n->weight_dtype != n->dtype && n->weight_dtype != AG_F32)
        return fail(AG_ERR_VALUE, "ag_rows_norm_backward: the weights are f32 or of the rows' type");
    AG_TRY(check_pitches("ag_rows_norm_backward", {n->dy_stride, n->dh_stride, n->h_stride, n->x_stride, n->residual_stride}));
    NormBackArgs a{};
    AG_TRY(make_drop(n->p, n->seed, n->offset, &a.drop));
    if (n->rows && ((!n->h && !n->x) || !n->rstd || (n->dw && !n->scratch))) return fail(AG_ERR_VALUE, "ag_rows_norm_backward: null argument");
    if (n->h && (n->x || n->residual)) return fail(AG_ERR_VALUE, "ag_rows_norm_backward: either h or what it is made of");
    if (n->x && n->dtype == AG_F32) return fail(AG_ERR_VALUE, "ag_rows_norm_backward: rows of f32 come with their h");
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    if (n->rows == 0) {
        if (n->dw) AG_CUDA(cudaMemsetAsync(n->dw, 0, n->dim * elem_size(n->weight_dtype), (cudaStream_t)stream));
        return AG_OK;
    }
    uint32_t grid = back_blocks_bound(n->rows, (uint32_t)n->dim, n->dtype);
    if (n->dw && n->scratch_bytes < (uint64_t)grid * n->dim * 4)
        return fail(AG_ERR_VALUE, "ag_rows_norm_backward: %llu bytes of scratch, %llu are needed", (unsigned long long)n->scratch_bytes,
                    (unsigned long long)grid * n->dim * 4);
    a.dy = n->dy; a.dh = n->dh; a.h = n->h; a.weight = n->weight; a.rstd = n->rstd; a.dx = n->dx; a.dres = n->dresidual;
    a.x = n->x; a.res = n->residual; a.x_stride = (uint32_t)n->x_stride; a.res_stride = (uint32_t)n->residual_stride;
    a.partial = n->dw ? (float *)n->scratch : nullptr;
    a.rows = (uint32_t)n->rows; a.dim = (uint32_t)n->dim; a.dy_stride = (uint32_t)n->dy_stride; a.dh_stride = (uint32_t)n->dh_stride; a.h_stride = (uint32_t)n->h_stride;
    a.w_f32 = n->weight_dtype == AG_F32; a.inv_dim = 1.0f / (float)n->dim;
    const uint32_t e = elem_size(n->dtype);
    const bool vec = a.dim % kChunk == 0 && vec_rows(a.weight, 0, elem_size(n->weight_dtype)) && vec_rows(a.dy, a.dy_stride, e) && vec_rows(a.dh, a.dh_stride, e) && vec_rows(a.h, a.h_stride, e) &&
                     vec_rows(a.x, a.x_stride, e) && vec_rows(a.res, a.res_stride, e) && vec_rows(a.dx, a.dim, e) && vec_rows(a.dres, a.dim, e);
    const bool pairs = a.dim % 2 == 0 && pair_rows(a.weight, 0, elem_size(n->weight_dtype)) && pair_rows(a.dy, a.dy_stride, e) && pair_rows(a.dh, a.dh_stride, e) &&
                       pair_rows(a.h, a.h_stride, e) && pair_rows(a.x, a.x_stride, e) && pair_rows(a.res, a.res_stride, e) && pair_rows(a.dx, a.dim, e) && pair_rows(a.dres, a.dim, e);
    cudaError_t err = cudaSuccess;
    with_type(n->dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        err = with_mode<T>(vec, pairs, [&](auto mode) { return launch_back<T, decltype(mode)::value>(a, n->dtype, grid, (cudaStream_t)stream); });
    });
    AG_CUDA(err);
    if (n->dw)
        with_type(n->weight_dtype, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            const float *partial = (const float *)n->scratch;
            const uint32_t dim = (uint32_t)n->dim;
            if (dim <= (uint32_t)kSMs * 8) launch_chained(k_norm_dw<T, 8>, dim3((dim + 7) / 8), dim3(8, 128), (cudaStream_t)stream, partial, grid, dim, (T *)n->dw);
            else launch_chained(k_norm_dw<T, 32>, dim3((dim + 31) / 32), dim3(32, 32), (cudaStream_t)stream, partial, grid, dim, (T *)n->dw);
        });
    AG_CUDA(cudaGetLastError());
    return AG_OK;
}

extern "C" int32_t ag_rows_encode_weight(const void *w, uint64_t out, uint64_t dim, uint64_t stride, int32_t dtype, void *codes,
                                         uint64_t code_stride, float *scales, int32_t device, void *stream) {
    AG_TRY(check_rows("ag_rows_encode_weight", out, dim, dtype));
    if (out == 0) return AG_OK;
    if (!w || !codes || !scales) return fail(AG_ERR_VALUE, "ag_rows_encode_weight: null argument");
    if (code_stride % 16 != 0 || code_stride < dim || (uintptr_t)codes % 16 != 0)
        return fail(AG_ERR_VALUE, "ag_rows_encode_weight: 8-bit rows start on multiples of 16 bytes and do not overlap");
    const uint64_t blocks = (out + kF8Block - 1) / kF8Block * ((dim + kF8Block - 1) / kF8Block);
    if (blocks > 0x7FFFFFFFull) return fail(AG_ERR_VALUE, "ag_rows_encode_weight: too many weights");
    DeviceGuard guard(device);
    if (!guard.ok) return AG_ERR_CUDA;
    with_type(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        k_encode_weight<T><<<(uint32_t)blocks, kThreads, 0, (cudaStream_t)stream>>>((const T *)w, out, (uint32_t)dim, stride, (uint8_t *)codes,
                                                                                      code_stride, scales);
    });
    AG_CUDA(cudaGetLastError());
    return AG_OK;
}
