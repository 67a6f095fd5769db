// 4-bit microscaled matrices: quantisation, the values a quantised matrix
// holds, and the product of two of them on the block-scaled tensor cores.
//
// A block of 32 elements along a row shares the scale X = 2^(floor(log2
// max|v|) - 2), exponent at least -127 (2 is the exponent of the largest
// E2M1 magnitude, 6), and each element is v / X rounded to nearest even onto
// {0, .5, 1, 1.5, 2, 3, 4, 6}, at most 6 in magnitude. X is a power of two,
// so v / X is exact wherever its rounding could matter, and the one rounding
// is the conversion's. A block that holds an infinity or a NaN has the scale
// code 255 and reads as NaN throughout.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "ops.hpp"
#include "sm100.cuh"

namespace azb {

namespace {

__device__ int g_mx4_error;   // KernelError of a product whose bounded wait ran out

// ---------------------------------------------------------- conversions

// Eight magnitudes' worth of E2M1 codes, element 0 in the low four bits.
__device__ __forceinline__ uint32_t pack_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

__device__ __forceinline__ void unpack_e2m1(uint32_t codes, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// Elements [c, c + 8) of a row as floats; zeros past cols. kVec: the row is
// 16-byte aligned and c + 8 <= cols.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* row, long long c, long long cols, float (&v)[8]) {
    if constexpr (kVec && sizeof(T) == 2) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(row + c));
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(h[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else if constexpr (kVec) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(row + c));
        const float4 b = __ldg(reinterpret_cast<const float4*>(row + c) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? float(row[c + i]) : 0.0f;
    }
}

template <typename T, bool kVec>
__device__ __forceinline__ void store8(T* row, long long c, long long cols, const float (&v)[8]) {
    if constexpr (kVec && sizeof(T) == 2) {
        uint4 q;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(row + c) = q;
    } else if constexpr (kVec) {
        float4* p = reinterpret_cast<float4*>(row + c);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < cols) row[c + i] = T(v[i]);
    }
}

__device__ __forceinline__ size_t scale_offset(const MxShape& s, long long row, long long block) {
    return size_t((row >> 7) * s.scale_tiles() + (block >> 2)) * 512 + size_t(row & 31) * 16 +
           size_t((row >> 5) & 3) * 4 + size_t(block & 3);
}

// ---------------------------------------------------------- quantisation

// One thread takes 8 elements, four neighbours one block: a warp's load is
// 256 consecutive elements. The block's maximum is an integer maximum of
// magnitudes (an infinity or NaN has the largest), over the four threads.
// A warp item is kCastSpan elements of one row, all loads in flight before
// the first is used. Rows up to the next multiple of 128 and blocks up to
// the next multiple of 4 are visited too: their scales are set to zero.
constexpr int kCastThreads = 256, kCastUnroll = 4, kCastSpan = 256 * kCastUnroll;

template <typename T, bool kAligned>
__global__ void __launch_bounds__(kCastThreads) mx4_quantise_kernel(const MxCastArgs a) {
    const MxShape s = a.shape;
    const int lane = threadIdx.x & 31;
    const long long spans = (s.scale_tiles() * 128 + kCastSpan - 1) / kCastSpan;
    const long long items = s.row_tiles() * 128 * spans;
    const long long warps = (long long)gridDim.x * (kCastThreads / 32);
    for (long long it = (long long)blockIdx.x * (kCastThreads / 32) + (threadIdx.x >> 5); it < items; it += warps) {
        const long long row = it / spans, c0 = (it - row * spans) * kCastSpan + lane * 8;
        const T* src = static_cast<const T*>(a.plain) + size_t(row) * size_t(a.ld);
        float v[kCastUnroll][8];
#pragma unroll
        for (int u = 0; u < kCastUnroll; ++u) {
            const long long c = c0 + u * 256;
            if (kAligned && row < s.rows && c + 8 <= s.cols) load8<T, true>(src, c, s.cols, v[u]);
            else load8<T, false>(src, c, row < s.rows ? s.cols : 0, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kCastUnroll; ++u) {
            const long long c = c0 + u * 256, block = c >> 5;
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[u][i]) & 0x7FFFFFFFu);
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const uint32_t field = top >> 23;
            const bool bad = field == 255;
            const uint32_t code = bad ? 255u : (field > 2 ? field - 2 : 0u);
            const float inv = __uint_as_float((bad ? 127u : 254u - code) << 23);   // 1 / X
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = bad ? 0.0f : v[u][i] * inv;
            const uint32_t codes = pack_e2m1(y);
            if (row < s.rows && block < s.blocks())
                reinterpret_cast<uint32_t*>(a.codes + size_t(row) * size_t(s.pitch()))[c >> 3] = codes;
            // Four blocks' scales are one 4-byte word.
            uint32_t word = code;
            word |= __shfl_down_sync(0xFFFFFFFFu, code, 4) << 8;
            word |= __shfl_down_sync(0xFFFFFFFFu, code, 8) << 16;
            word |= __shfl_down_sync(0xFFFFFFFFu, code, 12) << 24;
            if ((lane & 15) == 0 && (block >> 2) < s.scale_tiles())
                *reinterpret_cast<uint32_t*>(a.scales + scale_offset(s, row, block)) = word;
        }
    }
    grid_launch_dependents();
}

template <typename T, bool kAligned>
__global__ void __launch_bounds__(kCastThreads) mx4_values_kernel(const MxCastArgs a) {
    const MxShape s = a.shape;
    const int lane = threadIdx.x & 31;
    const long long spans = (s.cols + kCastSpan - 1) / kCastSpan;
    const long long items = s.rows * spans;
    const long long warps = (long long)gridDim.x * (kCastThreads / 32);
    for (long long it = (long long)blockIdx.x * (kCastThreads / 32) + (threadIdx.x >> 5); it < items; it += warps) {
        const long long row = it / spans, c0 = (it - row * spans) * kCastSpan + lane * 8;
        uint32_t codes[kCastUnroll], scale[kCastUnroll];
#pragma unroll
        for (int u = 0; u < kCastUnroll; ++u) {
            const long long c = c0 + u * 256;
            const bool in = c < s.cols;
            codes[u] = in ? __ldg(reinterpret_cast<const uint32_t*>(a.codes + size_t(row) * size_t(s.pitch())) + (c >> 3)) : 0u;
            scale[u] = in ? __ldg(a.scales + scale_offset(s, row, c >> 5)) : 0u;
        }
        T* dst = static_cast<T*>(a.plain) + size_t(row) * size_t(a.ld);
#pragma unroll
        for (int u = 0; u < kCastUnroll; ++u) {
            const long long c = c0 + u * 256;
            if (c >= s.cols) continue;
            float v[8];
            unpack_e2m1(codes[u], v);
            // 2^(code - 127): code 0 is the subnormal 2^-127, code 255 NaN.
            const float x = scale[u] == 255 ? __uint_as_float(0x7FC00000u)
                                            : __uint_as_float(scale[u] ? scale[u] << 23 : 0x00400000u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= x;
            if (kAligned && c + 8 <= s.cols) store8<T, true>(dst, c, s.cols, v);
            else store8<T, false>(dst, c, s.cols, v);
        }
    }
}

int cast_grid(long long items, int sms) {
    const long long ctas = (items + kCastThreads / 32 - 1) / (kCastThreads / 32);
    return int(std::min<long long>(ctas, (long long)sms * 8));
}

bool rows_aligned(const MxCastArgs& a) {
    return reinterpret_cast<uintptr_t>(a.plain) % 16 == 0 && (a.shape.rows == 1 || size_t(a.ld) * elem_size(a.type) % 16 == 0);
}

// --------------------------------------------------------------- product

// D[128 rows of w][tn rows of x] per CTA: w's rows are the tensor core's
// lanes and x's its columns, so one kernel serves a single row of x (a
// 16-column tile) and thousands (256 columns). Operands and scales are
// staged by TMA in chunks of 256 elements of K (128-byte swizzled rows; a
// scale tile is 128 rows x 4 blocks in exactly the order tcgen05.cp's
// 32x128b.warpx4 form writes TMEM's scale columns).
struct ProductTile {
    int m, n;              // rows of x, rows of w
    int chunks, steps;     // K in chunks of 256 and in MMA steps of 64
    int scale_tiles;       // per 128 rows
    int tn;                // columns per tile: a multiple of 16; 64 or a multiple of 128 if there are several tiles
    int stages;
    int splits;            // CTAs (one cluster) that share a tile's K
    uint32_t tmem_cols;
    const uint8_t* x_scales;
    const uint8_t* w_scales;
    const float* bias;
    int relu;
    void* out;
    long long ld;
    int early_w;           // w and its scales may be read before the previous launch ends
};

constexpr int kPTile = 128, kPChunkBytes = 128, kPThreads = 192, kPMaxStages = 8;
constexpr uint32_t kPWBytes = kPTile * kPChunkBytes;

__host__ __device__ constexpr int scale_groups(int tn) { return (tn + 127) / 128; }
__host__ __device__ constexpr uint32_t stage_bytes(int tn) {
    return kPWBytes + uint32_t(tn) * kPChunkBytes + 1024u + 1024u * uint32_t(scale_groups(tn));
}
__host__ __device__ constexpr uint32_t stage_scale_cols(int tn) { return 8u + 8u * uint32_t(scale_groups(tn)); }

// 128 scale words (512 bytes at saddr) into 4 TMEM columns, in all four lane
// quarters.
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint32_t saddr) {
    uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(128 >> 4) << 32;   // stride between groups of 8 rows of 16 bytes
    d |= 1ull << 46;                              // fixed 0b001; no swizzle
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// kind::mxf4: E2M1 operands, one E8M0 scale per 32 elements of K (two per
// MMA step of 64), fp32 accumulation.
__device__ __forceinline__ void umma_mx4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                         uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// M = 128, N columns, E2M1 x E2M1, E8M0 scales taken from bytes sf_id, sf_id
// + 1 of each scale word.
__device__ __forceinline__ uint32_t mx4_idesc(int n, uint32_t sf_id) {
    return (sf_id << 4)                            // B's scales
           | (1u << 7) | (1u << 10)                // E2M1
           | (static_cast<uint32_t>(n >> 3) << 17)
           | (1u << 23)                            // E8M0 scales
           | (static_cast<uint32_t>(kPTile >> 4) << 24)
           | (sf_id << 29);                        // A's scales
}

template <typename T>
__device__ __forceinline__ void store_out(const ProductTile& p, int row, int col, float v, float bias) {
    v += bias;
    if (p.relu) v = v < 0.0f ? 0.0f : v;   // keeps a NaN
    static_cast<T*>(p.out)[size_t(row) * size_t(p.ld) + size_t(col)] = T(v);
}

template <typename T>
__global__ void __launch_bounds__(kPThreads, 1)
    mx4_product_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx, const ProductTile p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[kPMaxStages], empty[kPMaxStages], done;
    __shared__ uint32_t tmem_slot;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = int(blockIdx.x) % p.splits;
    const int n0 = int(blockIdx.x) / p.splits * kPTile, x0 = int(blockIdx.y) * p.tn;
    // This CTA's chunks of K: an even share, in order.
    const int c_begin = int((long long)p.chunks * split / p.splits);
    const int c_end = int((long long)p.chunks * (split + 1) / p.splits);
    const int groups = scale_groups(p.tn);
    const uint32_t stage = stage_bytes(p.tn), x_bytes = uint32_t(p.tn) * kPChunkBytes;
    const int x_tile = x0 >> 7, x_tiles = (p.m + 127) >> 7;
    const uint32_t scale_col0 = uint32_t(max(p.tn, 32));

    if (warp == 0 && lane == 0) {
        tma_prefetch_map(&mw);
        tma_prefetch_map(&mx);
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(&done, 1);
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(&tmem_slot, p.tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0 && lane == 0) {
        auto scale_bytes = [&](int c) { return min(2, p.scale_tiles - 2 * c) * 512; };
        auto x_groups = [&] { return min(groups, x_tiles - x_tile); };
        auto load_w = [&](int c, int s) {   // arms the barrier for the whole stage
            uint8_t* b = base + size_t(s) * stage;
            const uint32_t sb = uint32_t(scale_bytes(c));
            mbar_arrive_expect_tx(&full[s], kPWBytes + x_bytes + sb * (1u + uint32_t(x_groups())));
            tma_load_2d(&mw, b, &full[s], c * kPChunkBytes, n0);
            bulk_load(b + kPWBytes + x_bytes, p.w_scales + (size_t(n0 >> 7) * p.scale_tiles + 2 * c) * 512, sb, &full[s]);
        };
        auto load_x = [&](int c, int s) {
            uint8_t* b = base + size_t(s) * stage;
            tma_load_2d(&mx, b + kPWBytes, &full[s], c * kPChunkBytes, x0);
            for (int g = 0; g < x_groups(); ++g)
                bulk_load(b + kPWBytes + x_bytes + 1024 + 1024 * g,
                          p.x_scales + (size_t(x_tile + g) * p.scale_tiles + 2 * c) * 512, uint32_t(scale_bytes(c)), &full[s]);
        };
        const int ahead = min(p.stages, c_end - c_begin);
        if (!p.early_w) grid_dependency_wait();
        for (int i = 0; i < ahead; ++i) load_w(c_begin + i, i);
        if (p.early_w) grid_dependency_wait();
        for (int i = 0; i < ahead; ++i) load_x(c_begin + i, i);
        Ring r;
        int loaded = ahead;
        for (int c = c_begin + ahead; c < c_end; ++c) {
            if (!mbar_wait(&empty[r.idx], r.phase, &g_mx4_error, kErrWaitProducer)) break;
            load_w(c, int(r.idx));
            load_x(c, int(r.idx));
            r.next(uint32_t(p.stages));
            ++loaded;
        }
        // Every copy has landed before this CTA's shared memory goes away
        // (the MMA warp has waited for them unless a wait ran out).
        for (int i = max(0, loaded - p.stages); i < loaded; ++i)
            mbar_wait(&full[i % p.stages], uint32_t(i / p.stages) & 1u, &g_mx4_error, kErrWaitDrain);
    } else if (warp == 1 && lane == 0) {
        Ring r;
        bool first = true;
        for (int c = c_begin; c < c_end; ++c) {
            if (!mbar_wait(&full[r.idx], r.phase, &g_mx4_error, kErrWaitMma)) break;
            tc_fence_after();
            const uint32_t b = smem_u32(base) + r.idx * stage;
            const uint32_t sw = b + kPWBytes + x_bytes, sx = sw + 1024;
            const uint32_t tw = tmem + scale_col0 + r.idx * stage_scale_cols(p.tn), tx = tw + 8;
            const int tiles = min(2, p.scale_tiles - 2 * c);
            // Each stage has its own scale columns: they are overwritten only
            // once the MMAs that read them have freed the stage.
            for (int t = 0; t < tiles; ++t) {
                tmem_copy_scales(tw + uint32_t(t) * 4, sw + uint32_t(t) * 512);
                for (int g = 0; g < groups; ++g)
                    tmem_copy_scales(tx + uint32_t(t * groups + g) * 4, sx + uint32_t(g) * 1024 + uint32_t(t) * 512);
            }
            const uint64_t da = sw128_desc(b), db = sw128_desc(b + kPWBytes);
            const int steps = min(4, p.steps - 4 * c);
            for (int k = 0; k < steps; ++k) {
                const uint32_t t = uint32_t(k) >> 1;
                umma_mx4(tmem, da + uint64_t(2 * k), db + uint64_t(2 * k), mx4_idesc(p.tn, (uint32_t(k) & 1u) * 2u),
                         tw + t * 4, tx + t * uint32_t(groups) * 4 + (uint32_t(x0 & 127) >> 5), first ? 0u : 1u);
                first = false;
            }
            umma_commit(&empty[r.idx]);
            r.next(uint32_t(p.stages));
        }
        umma_commit(&done);
    }
    __syncwarp();

    const int quarter = warp & 3;                 // the TMEM lanes this warp may read
    const int j = n0 + quarter * 32 + lane;       // this thread's row of w: an output column
    const float bias = p.bias && j < p.n ? p.bias[j] : 0.0f;
    const int live = min(p.tn, p.m - x0);         // the tile's rows of x
    float* part = reinterpret_cast<float*>(base);
    if (warp >= 2) {
        mbar_wait(&done, 0, &g_mx4_error, kErrWaitEpilogue);
        tc_fence_after();
        if (p.early_w) grid_dependency_wait();    // the output may be what earlier launches read
        for (int c0 = 0; c0 < live; c0 += 32) {
            uint32_t v[32];
            if (live - c0 > 16) {
                tmem_ld32(tmem + (uint32_t(quarter) << 21) + uint32_t(c0), v);
            } else {
                uint32_t h[16];
                tmem_ld16(tmem + (uint32_t(quarter) << 21) + uint32_t(c0), h);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = h[i], v[i + 16] = 0;
            }
            tmem_wait_ld();
            tmem_hold(v);
            if (p.splits > 1) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c0 + i < live) part[(c0 + i) * kPTile + quarter * 32 + lane] = __uint_as_float(v[i]);
            } else if (j < p.n) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c0 + i < live) store_out<T>(p, x0 + c0 + i, j, __uint_as_float(v[i]), bias);
            }
        }
    }
    // TMEM goes back before any wait for another CTA: a CTA that waits for a
    // peer while it holds TMEM could wait for one that cannot allocate its own.
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, p.tmem_cols);
    if (p.splits > 1) {
        // The parts' sum, in order of K (the same bits on every run): CTA
        // `split` finishes rows split, split + splits, ... of the tile.
        cluster_sync();
        if (warp >= 2) {
            for (int i = split; i < live; i += p.splits) {
                float sum = 0.0f;
                for (int r = 0; r < p.splits; ++r) {
                    const uint32_t a = mapa(smem_u32(part + i * kPTile + quarter * 32 + lane), uint32_t(r));
                    float v;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
                    sum += v;
                }
                if (j < p.n) store_out<T>(p, x0 + i, j, sum, bias);
            }
        }
        cluster_sync();
    }
}

template <typename T>
cudaError_t launch_product_t(const CUtensorMap& mw, const CUtensorMap& mx, const ProductTile& p, dim3 grid, bool pdl,
                             cudaStream_t s) {
    const size_t smem = 1024 + size_t(p.stages) * stage_bytes(p.tn);
    if (const cudaError_t e = open_smem<mx4_product_kernel<T>>(smem); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kPThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (p.splits > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim = {unsigned(p.splits), 1, 1};
        ++na;
    }
    if (pdl) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = unsigned(na);
    return cudaLaunchKernelEx(&cfg, mx4_product_kernel<T>, mw, mx, p);
}

}  // namespace

cudaError_t launch_mx4_quantise(const MxCastArgs& a, int sms, cudaStream_t s) {
    const MxShape& sh = a.shape;
    const int grid = cast_grid(sh.row_tiles() * 128 * ((sh.scale_tiles() * 128 + kCastSpan - 1) / kCastSpan), sms);
    const bool v = rows_aligned(a);
    if (a.type == kElemBF16) {
        if (v) mx4_quantise_kernel<__nv_bfloat16, true><<<grid, kCastThreads, 0, s>>>(a);
        else mx4_quantise_kernel<__nv_bfloat16, false><<<grid, kCastThreads, 0, s>>>(a);
    } else {
        if (v) mx4_quantise_kernel<float, true><<<grid, kCastThreads, 0, s>>>(a);
        else mx4_quantise_kernel<float, false><<<grid, kCastThreads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

cudaError_t launch_mx4_values(const MxCastArgs& a, int sms, cudaStream_t s) {
    const MxShape& sh = a.shape;
    const int grid = cast_grid(sh.rows * ((sh.cols + kCastSpan - 1) / kCastSpan), sms);
    const bool v = rows_aligned(a);
    if (a.type == kElemBF16) {
        if (v) mx4_values_kernel<__nv_bfloat16, true><<<grid, kCastThreads, 0, s>>>(a);
        else mx4_values_kernel<__nv_bfloat16, false><<<grid, kCastThreads, 0, s>>>(a);
    } else {
        if (v) mx4_values_kernel<float, true><<<grid, kCastThreads, 0, s>>>(a);
        else mx4_values_kernel<float, false><<<grid, kCastThreads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

cudaError_t launch_mx4_product(const MxProductArgs& a, int sms, cudaStream_t s) {
    const MxShape xs{a.m, a.k}, ws{a.n, a.k};
    ProductTile p{};
    p.m = int(a.m);
    p.n = int(a.n);
    p.chunks = int((a.k + 255) / 256);
    p.steps = int((a.k + 63) / 64);
    p.scale_tiles = int(xs.scale_tiles());
    // Columns per tile: as few as hold all of x up to 128; more rows of x in
    // tiles of 256 where those alone fill the SMs, else 128, else 64.
    const int n_tiles = int((a.n + kPTile - 1) / kPTile);
    if (a.m <= 128) p.tn = int((a.m + 15) / 16 * 16);
    else p.tn = 64;
    for (const int tn : {128, 256})
        if (a.m > 128 && (a.m + tn - 1) / tn * n_tiles >= sms) p.tn = tn;
    const int x_tiles = int((a.m + p.tn - 1) / p.tn);
    // K is shared by a cluster of CTAs while the tiles leave SMs idle and
    // every CTA keeps a chunk or more (the parts fit a stage's memory up to
    // 64 columns).
    p.splits = 1;
    while (p.tn <= 64 && p.splits < 8 && (long long)n_tiles * x_tiles * p.splits * 2 <= sms && p.splits * 2 <= p.chunks)
        p.splits *= 2;
    const int per_cta = (p.chunks + p.splits - 1) / p.splits;
    p.stages = int(std::min<size_t>(kPMaxStages, (size_t(220) << 10) / stage_bytes(p.tn)));
    p.stages = std::max(1, std::min(p.stages, per_cta));
    // The parts of a shared K reuse the stages' memory: 512 bytes a column.
    while (p.splits > 1 && size_t(p.stages) * stage_bytes(p.tn) < size_t(p.tn) * kPTile * 4) ++p.stages;
    const uint32_t cols = uint32_t(std::max(p.tn, 32)) + uint32_t(p.stages) * stage_scale_cols(p.tn);
    p.tmem_cols = 32;
    while (p.tmem_cols < cols) p.tmem_cols *= 2;
    p.x_scales = a.x_scales;
    p.w_scales = a.w_scales;
    p.bias = a.bias;
    p.relu = a.relu;
    p.out = a.out;
    p.ld = a.ld;
    p.early_w = a.after_quantise ? 1 : 0;
    const CUtensorMap mw = make_byte_map(a.w_codes, uint64_t(ws.pitch()), uint64_t(a.n), kPTile);
    const CUtensorMap mx = make_byte_map(a.x_codes, uint64_t(xs.pitch()), uint64_t(a.m), uint32_t(p.tn));
    const dim3 grid(unsigned(n_tiles * p.splits), unsigned(x_tiles));
    return a.type == kElemBF16 ? launch_product_t<__nv_bfloat16>(mw, mx, p, grid, a.after_quantise, s)
                               : launch_product_t<float>(mw, mx, p, grid, a.after_quantise, s);
}

cudaError_t mx4_take_error(int* code) {
    *code = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(code, g_mx4_error, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(g_mx4_error, &zero, sizeof(int));
    return e;
}

}  // namespace azb
