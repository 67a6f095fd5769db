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
#include <type_traits>

#include "ops.hpp"
#include "sm100.cuh"

namespace azb {

namespace {

__device__ int g_mx4_error;   // KernelError of the first product whose bounded wait ran out; never cleared

// ---------------------------------------------------------- conversions

// Eight values' E2M1 codes (round to nearest even, at most 6), value 0's in
// the low four bits.
__device__ __forceinline__ uint32_t pack_e2m1(const float* v) {
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

__device__ __forceinline__ void unpack_e2m1(uint32_t codes, float* v) {
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

template <int kBytes>
__device__ __forceinline__ void load_piece(uint32_t* dst, const uint32_t* src) {
    if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(dst) = __ldcs(reinterpret_cast<const uint4*>(src));
    else *reinterpret_cast<uint2*>(dst) = __ldcs(reinterpret_cast<const uint2*>(src));
}

// kN neighbouring elements of a row as they lie in memory (kN T in words).
template <typename T, int kN>
struct Run {
    static constexpr int kWords = kN * int(sizeof(T)) / 4;
    uint32_t u[kWords];

    // Elements [c, c + kN), zeros past `cols`; c a multiple of kN. kBytes: 16
    // or 8, of which the row starts at a multiple, or 0 (any row).
    template <int kBytes>
    __device__ __forceinline__ void load(const T* row, long long c, long long cols) {
        if constexpr (kBytes > 0) {
            if (c + kN <= cols) {
#pragma unroll
                for (int i = 0; i < kWords; i += kBytes / 4)
                    load_piece<kBytes>(u + i, reinterpret_cast<const uint32_t*>(row + c) + i);
                return;
            }
        } else {
            // The run lies `off` bytes into its first 16: those and the ones
            // after are read whole, where they are the row's, and shifted.
            const uint32_t off = uint32_t(reinterpret_cast<uintptr_t>(row + c) & 15);
            const long long first = c - off / int(sizeof(T)), end = first + kN + (off ? 16 / int(sizeof(T)) : 0);
            if (first >= 0 && end <= cols) {
                uint32_t w[kWords + 4];
                const uint32_t* from = reinterpret_cast<const uint32_t*>(row + first);
#pragma unroll
                for (int i = 0; i < kWords; i += 4) load_piece<16>(w + i, from + i);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[kWords + i] = 0;
                if (off) load_piece<16>(w + kWords, from + kWords);
                if (off & 8) {
#pragma unroll
                    for (int i = 0; i < kWords + 2; ++i) w[i] = w[i + 2];
                }
                if (off & 4) {
#pragma unroll
                    for (int i = 0; i < kWords + 1; ++i) w[i] = w[i + 1];
                }
#pragma unroll
                for (int i = 0; i < kWords; ++i) u[i] = sizeof(T) == 2 && (off & 2) ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) {
                u[i] = c + i < cols ? __ldg(reinterpret_cast<const uint32_t*>(row + c) + i) : 0u;
            } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(row + c) + 2 * i;
                u[i] = c + 2 * i < cols ? __ldg(h) : 0u;
                if (c + 2 * i + 1 < cols) u[i] |= uint32_t(__ldg(h + 1)) << 16;
            }
        }
    }
    // The largest magnitude's exponent field (255: an infinity or a NaN).
    // Magnitudes compare as their bits do.
    __device__ __forceinline__ uint32_t top_field() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kWords; ++i) top = max(top, u[i] & 0x7FFFFFFFu);
            return top >> 23;
        } else {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kWords; ++i) top = __vmaxu2(top, u[i] & 0x7FFF7FFFu);
            return max(top >> 16, top & 0xFFFFu) >> 7;
        }
    }
    // Codes of elements [8 i, 8 i + 8) over the scale 2^(code - 127). The
    // product with the scale's reciprocal is exact (in bfloat16 too) unless it
    // is far below the smallest magnitude's half.
    __device__ __forceinline__ uint32_t codes(int i, uint32_t code) const {
        if (code == 255) return 0u;
        float y[8];
        if constexpr (sizeof(T) == 4) {
            const float inv = __uint_as_float((254u - code) << 23);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(u[8 * i + e]) * inv;
        } else {
            const uint32_t h = (254u - code) << 7, hh = h | h << 16;
            const __nv_bfloat162 inv = *reinterpret_cast<const __nv_bfloat162*>(&hh);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 t = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&u[4 * i + e]), inv);
                const uint32_t w = *reinterpret_cast<const uint32_t*>(&t);
                y[2 * e] = __uint_as_float(w << 16);
                y[2 * e + 1] = __uint_as_float(w & 0xFFFF0000u);
            }
        }
        return pack_e2m1(y);
    }
};

// The scale code (exponent + 127) of a block whose largest magnitude has this
// exponent field.
__device__ __forceinline__ uint32_t scale_code(uint32_t field) { return field == 255 ? 255u : field > 2 ? field - 2 : 0u; }

__device__ __forceinline__ size_t scale_offset(const MxShape& s, long long row, long long block) {
    return size_t((row >> 7) * s.scale_tiles() + (block >> 2)) * 512 + size_t(row & 31) * 16 +
           size_t((row >> 5) & 3) * 4 + size_t(block & 3);
}

// ---------------------------------------------------------- quantisation

// A thread takes 16 elements, two neighbours one block; a warp 512 neighbours
// of a row at a time, kCastUnroll of those with all loads in flight before
// the first is used. blockIdx.x: the span of columns (there may be more than
// 65535); rows are shared out over blockIdx.y and the block's warps. Rows up
// to the next multiple of 128 and blocks up to the next multiple of 4 are
// visited too: their scales are set to zero. Loads are of 16 bytes, shifted
// into place where the rows do not start at multiples of 16 (16384 x 8191 of
// fp32 108 us so and 277 us by elements, of bfloat16 67 and 150), but for
// bfloat16 rows at multiples of 8, which take loads of 8 (59 us and 66).
//
// Bound by DRAM where the matrix is large: 16384 x 8192 of bfloat16 in 50 us
// with nothing in L2 (5.8 TB/s of 268 MB read and the codes written). Five
// blocks an SM (at most 51 registers) and two steps in flight: there and back
// 113 us, with four blocks 3 us more. Few rows are bound by the launch: 3 us.
constexpr int kCastThreads = 256, kCastWarps = kCastThreads / 32, kCastStep = 512;
template <typename T>
constexpr int kCastUnroll = sizeof(T) == 2 ? 2 : 1;   // as many as five blocks' registers hold
template <typename T>
constexpr int kCastSpan = kCastStep * kCastUnroll<T>;

template <typename T, int kBytes>
__global__ void __launch_bounds__(kCastThreads, 5) mx4_quantise_kernel(const MxCastArgs a) {
    // Past the wait every earlier launch has completed, so that the next may
    // start (it waits itself, or reads only what earlier ones wrote).
    grid_dependency_wait();
    grid_launch_dependents();
    const MxShape s = a.shape;
    const int lane = threadIdx.x & 31;
    const long long c0 = (long long)blockIdx.x * kCastSpan<T> + lane * 16;
    const long long rows = s.row_tiles() * 128, blocks = s.blocks(), tiles = s.scale_tiles();
    for (long long row = (long long)blockIdx.y * kCastWarps + (threadIdx.x >> 5); row < rows; row += (long long)gridDim.y * kCastWarps) {
        const T* src = static_cast<const T*>(a.plain) + size_t(row) * size_t(a.ld);
        const long long cols = row < s.rows ? s.cols : 0;
        Run<T, 16> v[kCastUnroll<T>];
#pragma unroll
        for (int u = 0; u < kCastUnroll<T>; ++u) v[u].template load<kBytes>(src, c0 + u * kCastStep, cols);
        uint8_t* codes = a.codes + size_t(row) * size_t(s.pitch());
        uint8_t* scales = a.scales + scale_offset(s, row, 0);
#pragma unroll
        for (int u = 0; u < kCastUnroll<T>; ++u) {
            const long long c = c0 + u * kCastStep, block = c >> 5;
            uint32_t field = v[u].top_field();
            field = max(field, __shfl_xor_sync(0xFFFFFFFFu, field, 1));
            const uint32_t code = scale_code(field);
            if (row < s.rows && block < blocks)
                *reinterpret_cast<uint2*>(codes + (c >> 1)) = make_uint2(v[u].codes(0, code), v[u].codes(1, code));
            // Four blocks' scales are one 4-byte word.
            uint32_t word = code | __shfl_down_sync(0xFFFFFFFFu, code, 2) << 8;
            word |= __shfl_down_sync(0xFFFFFFFFu, word, 4) << 16;
            if ((lane & 7) == 0 && (block >> 2) < tiles) *reinterpret_cast<uint32_t*>(scales + (block >> 2) * 512) = word;
        }
    }
}

// The inverse; a thread takes 8 elements, so that a warp's 16-byte stores of
// bfloat16 are neighbours (kBytes: what the rows are multiples of). Values of
// fp32, and of bfloat16 in rows of odd places (kBytes 0), are exchanged so
// that neighbouring lanes store neighbouring elements (16384 x 8192 of fp32 99
// us, two stores of 16 bytes a lane 142; 16384 x 8191 108 us, by single
// elements of a lane 518, of bfloat16 83 and 369). A value is a code's
// magnitude times a power of two: exact in either type (the smallest, 2^-128,
// is a subnormal that both hold). Bound by DRAM too: 16384 x 8192 into
// bfloat16 in 56 us (6.1 TB/s of 71 MB read and 268 MB written).
constexpr int kValuesUnroll = 4, kValuesStep = 256, kValuesSpan = kValuesStep * kValuesUnroll;

// The magnitude's three bits on top of a float's significand and exponent are
// that magnitude times 2^-126 (for 0.5 a subnormal).
__device__ __forceinline__ float value_of(uint32_t code) {
    return __uint_as_float((code & 8u) << 28 | (code & 7u) << 22) * 8.50705917e37f;
}

template <typename T, int kBytes>
__global__ void __launch_bounds__(kCastThreads, 6) mx4_values_kernel(const MxCastArgs a) {
    grid_dependency_wait();
    grid_launch_dependents();
    const MxShape s = a.shape;
    const int lane = threadIdx.x & 31;
    const long long c0 = (long long)blockIdx.x * kValuesSpan + lane * 8;
    for (long long row = (long long)blockIdx.y * kCastWarps + (threadIdx.x >> 5); row < s.rows; row += (long long)gridDim.y * kCastWarps) {
        const uint8_t* codes = a.codes + size_t(row) * size_t(s.pitch());
        const uint8_t* scales = a.scales + scale_offset(s, row, 0);
        uint32_t q[kValuesUnroll], scale[kValuesUnroll];
#pragma unroll
        for (int u = 0; u < kValuesUnroll; ++u) {
            const long long c = c0 + u * kValuesStep, block = c >> 5;
            const bool in = c < s.cols;
            q[u] = in ? __ldg(reinterpret_cast<const uint32_t*>(codes + (c >> 1))) : 0u;
            scale[u] = in ? __ldg(scales + (block >> 2) * 512 + (block & 3)) : 0u;
        }
        T* dst = static_cast<T*>(a.plain) + size_t(row) * size_t(a.ld);
#pragma unroll
        for (int u = 0; u < kValuesUnroll; ++u) {
            const long long c = c0 + u * kValuesStep;
            // 2^(code - 127): code 0 is the subnormal 2^-127, code 255 NaN.
            const float x = __uint_as_float(scale[u] == 255 ? 0x7FC00000u : scale[u] ? scale[u] << 23 : 0x00400000u);
            if constexpr (kBytes > 0) {
                float v[8];
                unpack_e2m1(q[u], v);
                if (c + 8 <= s.cols) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i] * x, v[2 * i + 1] * x);
                        w[i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    uint32_t* const to = reinterpret_cast<uint32_t*>(dst + c);
                    if constexpr (kBytes == 16) {
                        __stcs(reinterpret_cast<uint4*>(to), make_uint4(w[0], w[1], w[2], w[3]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i += kBytes / 4) {
                            if constexpr (kBytes == 8) __stcs(reinterpret_cast<uint2*>(to + i), make_uint2(w[i], w[i + 1]));
                            else __stcs(to + i, w[i]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (c + i < s.cols) dst[c + i] = T(v[i] * x);
                }
            } else {
                const long long step = c - lane * 8;
                const int left = int(min((long long)kValuesStep, s.cols - step)) - lane;
                T* const to = dst + step + lane;
#pragma unroll
                for (int j = 0; j < 8; ++j) {   // a block
                    const uint32_t code = __shfl_sync(0xFFFFFFFFu, q[u], 4 * j + (lane >> 3)) >> (4 * (lane & 7));
                    const float v = value_of(code) * __shfl_sync(0xFFFFFFFFu, x, 4 * j);
                    if (32 * j < left) {
                        if constexpr (sizeof(T) == 2)
                            __stcs(reinterpret_cast<unsigned short*>(to + 32 * j), __bfloat16_as_ushort(__float2bfloat16_rn(v)));
                        else __stcs(to + 32 * j, v);
                    }
                }
            }
        }
    }
}

// The largest of 16, 8, 4 and 2 bytes of which every row starts at a multiple.
int row_bytes(const void* p, long long rows, long long ld, int type) {
    const uintptr_t low = reinterpret_cast<uintptr_t>(p) | (rows > 1 ? uintptr_t(ld) * elem_size(type) : 0);
    return low % 16 == 0 ? 16 : low % 8 == 0 ? 8 : low % 4 == 0 ? 4 : 2;
}

dim3 cast_grid(long long rows, long long cols, int span, int sms) {
    const long long spans = (cols + span - 1) / span;
    const long long most = std::max<long long>(1, (long long)sms * 16 / spans);   // sixteen blocks an SM in all
    return dim3(unsigned(spans), unsigned(std::min((rows + kCastWarps - 1) / kCastWarps, most)));
}

// --------------------------------------------------------------- product

// D[128 rows of w][tn rows of x] per CTA: w's rows are the tensor core's
// lanes and x's its columns, so one kernel serves a single row of x (a
// 16-column tile) and thousands (256 columns). Operands and scales are
// staged by TMA in chunks of 256 elements of K (128-byte swizzled rows; a
// scale tile is 128 rows x 4 blocks in exactly the order tcgen05.cp's
// 32x128b.warpx4 form writes TMEM's scale columns).
//
// Few rows of x are bound by w's bytes and, at these sizes, by what comes
// before and after them: 32 x 16384 x 4096 in 9.3 us with x's quantisation
// (37 MB; 5.6 us at the rate of a copy), 1 x 4096 x 4096 in 4.9 us. Products
// in between (333 x 1111 x 2501 in 10.5 us with x's quantisation) have too few
// tiles to fill the SMs and run at the latency of a tile's K.
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
    int out_fours;         // four neighbouring outputs may be stored at once
    const void* x;         // plain x, where the kernel quantises it itself, and its rows
    long long x_ld;
    int k, x_aligned;      // x_aligned: every row starts at a multiple of 16 bytes
};

constexpr int kPTile = 128, kPChunkBytes = 128, kPThreads = 192, kPMaxStages = 8, kPMaxSplits = 8;
constexpr uint32_t kPWBytes = kPTile * kPChunkBytes;

__host__ __device__ constexpr int scale_groups(int tn) { return (tn + 127) / 128; }
__host__ __device__ constexpr uint32_t stage_bytes(int tn) {
    return kPWBytes + uint32_t(tn) * kPChunkBytes + 1024u + 1024u * uint32_t(scale_groups(tn));
}
__host__ __device__ constexpr uint32_t stage_scale_cols(int tn) { return 8u + 8u * uint32_t(scale_groups(tn)); }

// The descriptor of 128 scale words (512 bytes at saddr) for tmem_copy_scales.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
    uint64_t d = static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(128 >> 4) << 32;   // stride between groups of 8 rows of 16 bytes
    d |= 1ull << 46;                              // fixed 0b001; no swizzle
    return d;
}

// 128 scale words into 4 TMEM columns, in all four lane quarters.
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
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

// One thread of the (whole, converged) warp. A branch on this tells the
// compiler that a single thread issues: the tensor core's and TMA's operands
// are uniform registers, which under `lane == 0` it filled through a loop
// over the lanes (8192^3: 561 us under `lane == 0`, 389 us so).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ float activated(const ProductTile& p, float v) { return p.relu && v < 0.0f ? 0.0f : v; }   // keeps a NaN

// A lane's four of a tile's 128 outputs of a row: neighbours where they can
// be stored at once or come from other CTAs' parts, else every 32nd, so that
// a warp's stores are neighbours.
__device__ __forceinline__ int out_place(const ProductTile& p, int lane, int e) {
    return p.out_fours || p.splits > 1 ? lane * 4 + e : lane + 32 * e;
}

template <typename T>
__device__ __forceinline__ void store_four(const ProductTile& p, int row, int n0, int lane, const float (&sum)[4], const float (&bias)[4]) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = activated(p, sum[e] + bias[e]);
    T* to = static_cast<T*>(p.out) + size_t(row) * size_t(p.ld) + n0;
    if (p.out_fours && n0 + lane * 4 + 4 <= p.n) {
        if constexpr (sizeof(T) == 2) {
            uint2 w;
            reinterpret_cast<__nv_bfloat162*>(&w)[0] = __floats2bfloat162_rn(y[0], y[1]);
            reinterpret_cast<__nv_bfloat162*>(&w)[1] = __floats2bfloat162_rn(y[2], y[3]);
            *reinterpret_cast<uint2*>(to + lane * 4) = w;
        } else {
            *reinterpret_cast<float4*>(to + lane * 4) = make_float4(y[0], y[1], y[2], y[3]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n0 + out_place(p, lane, e) < p.n) to[out_place(p, lane, e)] = T(y[e]);
    }
}

// The four of `row` of a part in this CTA's shared memory.
__device__ __forceinline__ void load_four(const ProductTile& p, const float* row, int lane, float (&v)[4]) {
    if (p.out_fours) {
        const float4 f = *reinterpret_cast<const float4*>(row + lane * 4);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = row[lane + 32 * e];
    }
}

// The same of a part in another CTA's, at a shared::cluster address.
__device__ __forceinline__ void load_four_of(uint32_t row, int lane, float (&v)[4]) {
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(row + uint32_t(lane) * 16) : "memory");
}

// A block of 32 elements of plain x.
template <typename X>
struct PlainBlock {
    Run<X, 16> a, b;
    __device__ __forceinline__ void load(const X* row, long long c, long long cols, bool aligned) {
        if (aligned) {
            a.template load<16>(row, c, cols);
            b.template load<16>(row, c + 16, cols);
        } else {
            a.template load<0>(row, c, cols);
            b.template load<0>(row, c + 16, cols);
        }
    }
    __device__ __forceinline__ uint4 codes(uint32_t* code) const {
        *code = scale_code(max(a.top_field(), b.top_field()));
        return make_uint4(a.codes(0, *code), a.codes(1, *code), b.codes(0, *code), b.codes(1, *code));
    }
};

constexpr int kPEpiThreads = kPThreads - 64;
// Up to so many rows, and chunks of K a CTA, a plain x is quantised by the
// product's CTAs: 1 x 4096 x 4096 4.8 us so and 6.3 us with a launch before it
// (16 rows: 6.6 and 6.5), and the launch's host time is saved. With 32 rows
// 8.9 and 7.0.
constexpr int kPPlainRows = 16, kPPlainChunks = 8;

// kGroups: scale tiles of 128 rows of x (tn <= 128: 1, else 2). X: void, or
// the type of plain x, which the epilogue's warps then quantise into the
// stages themselves while w is on its way (every CTA its part of K; for few
// rows that costs less than a launch of its own).
template <typename T, int kGroups, typename X>
__global__ void __launch_bounds__(kPThreads)
    mx4_product_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx, const ProductTile p) {
    constexpr bool kPlain = !std::is_void_v<X>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[kPMaxStages], empty[kPMaxStages], done;
    __shared__ uint32_t tmem_slot;

    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const int split = int(blockIdx.x) % p.splits;
    const int n0 = int(blockIdx.x) / p.splits * kPTile, x0 = int(blockIdx.y) * p.tn;
    // This CTA's chunks of K: an even share, in order.
    const int c_begin = p.chunks * split / p.splits, c_end = p.chunks * (split + 1) / p.splits;
    const int ahead = min(p.stages, c_end - c_begin);
    const uint32_t stage = stage_bytes(p.tn), x_bytes = uint32_t(p.tn) * kPChunkBytes;
    const int x_tile = x0 >> 7, x_tiles = (p.m + 127) >> 7;
    const uint32_t scale_col0 = uint32_t(max(p.tn, 32));

    const auto scale_bytes = [&](int c) { return uint32_t(min(2, p.scale_tiles - 2 * c)) * 512u; };
    const auto x_groups = [&] { return min(kGroups, x_tiles - x_tile); };
    const auto load_w = [&](int c, int s) {   // arms the barrier for all of the stage's copies
        uint8_t* b = base + size_t(s) * stage;
        const uint32_t sb = scale_bytes(c);
        mbar_arrive_expect_tx(&full[s], kPWBytes + sb + (kPlain ? 0u : x_bytes + sb * uint32_t(x_groups())));
        tma_load_2d(&mw, b, &full[s], c * kPChunkBytes, n0);
        bulk_load(b + kPWBytes + x_bytes, p.w_scales + (size_t(n0 >> 7) * p.scale_tiles + 2 * c) * 512, sb, &full[s]);
    };
    const auto load_x = [&](int c, int s) {
        if constexpr (!kPlain) {
            uint8_t* b = base + size_t(s) * stage;
            tma_load_2d(&mx, b + kPWBytes, &full[s], c * kPChunkBytes, x0);
            for (int g = 0; g < x_groups(); ++g)
                bulk_load(b + kPWBytes + x_bytes + 1024 + 1024 * g,
                          p.x_scales + (size_t(x_tile + g) * p.scale_tiles + 2 * c) * 512, scale_bytes(c), &full[s]);
        }
    };

    // The first stages' copies are under way before the block meets.
    if (warp == 0 && elect_one()) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(&full[i], kPlain ? 1 + kPEpiThreads : 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(&done, 1);
        fence_barrier_init();
        if (!p.early_w) grid_dependency_wait();
        for (int i = 0; i < ahead; ++i) load_w(c_begin + i, i);
        if (p.early_w) grid_dependency_wait();
        for (int i = 0; i < ahead; ++i) load_x(c_begin + i, i);
    }
    if (warp == 1) tmem_alloc(&tmem_slot, p.tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // A call of one launch lets the next one's CTAs in at once (1 x 4096 x 4096
    // 5.0 us so, 5.7 without); behind a product with a quantisation before it
    // the next quantisation's blocks only take up SMs (333 x 1111 x 2501 11.0
    // us so, 10.2 without). Not before this CTA has its TMEM: a CTA let in
    // sooner could take it first, and keep it until this one is done.
    if constexpr (kPlain) grid_launch_dependents();

    if (warp == 0 && elect_one()) {
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
    } else if (warp == 1 && elect_one()) {
        Ring r;
        uint32_t more = 0;   // the tile's first MMA overwrites
        const uint32_t idesc[2] = {mx4_idesc(p.tn, 0), mx4_idesc(p.tn, 2)};
        const uint32_t x_off = uint32_t(x0 & 127) >> 5;
        // One scale tile (128 elements of K): its scales to TMEM, then its two
        // MMAs (the tile's second half may be past K: then one).
        auto tile = [&](uint32_t b, uint32_t tw, int t, bool both) {
            const uint32_t tx = tw + 8;
            const uint64_t sw = scale_desc(b + kPWBytes + x_bytes) + uint64_t(t * 32), sx = sw + 64;
            tmem_copy_scales(tw + uint32_t(t) * 4, sw);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) tmem_copy_scales(tx + uint32_t(t * kGroups + g) * 4, sx + uint64_t(g * 64));
            const uint64_t da = sw128_desc(b) + uint64_t(4 * t), db = sw128_desc(b + kPWBytes) + uint64_t(4 * t);
            const uint32_t fx = tx + uint32_t(t * kGroups) * 4 + x_off;
            umma_mx4(tmem, da, db, idesc[0], tw + uint32_t(t) * 4, fx, more);
            more = 1;
            if (both) umma_mx4(tmem, da + 2, db + 2, idesc[1], tw + uint32_t(t) * 4, fx, 1);
        };
        for (int c = c_begin; c < c_end; ++c) {
            if (!mbar_wait(&full[r.idx], r.phase, &g_mx4_error, kErrWaitMma)) break;
            tc_fence_after();
            const uint32_t b = smem_u32(base) + r.idx * stage;
            // Each stage has its own scale columns: they are overwritten only
            // once the MMAs that read them have freed the stage.
            const uint32_t tw = tmem + scale_col0 + r.idx * stage_scale_cols(p.tn);
            const int steps = p.steps - 4 * c;
            if (steps >= 4) {
                tile(b, tw, 0, true);
                tile(b, tw, 1, true);
            } else {
                tile(b, tw, 0, steps > 1);
                if (steps > 2) tile(b, tw, 1, false);
            }
            umma_commit(&empty[r.idx]);
            r.next(uint32_t(p.stages));
        }
        umma_commit(&done);
    }
    __syncwarp();

    const int quarter = warp & 3;                 // the TMEM lanes this warp may read
    const int live = min(p.tn, p.m - x0);         // the tile's rows of x
    float* part = reinterpret_cast<float*>(base);
    if constexpr (kPlain) {
        if (warp >= 2) {
            const int t = int(threadIdx.x) - 64;
            grid_dependency_wait();
            // Block b of row r of chunk c into stage s, as TMA and the scales'
            // copies lay them out. (x is one tile of at most 16 rows; rows past
            // m stay as they are: they reach no column that is stored.)
            const auto put = [&](int c, int s, int r, int b) {
                PlainBlock<X> v;
                v.load(static_cast<const X*>(p.x) + size_t(r) * size_t(p.x_ld), (long long)c * 256 + b * 32, p.k, p.x_aligned != 0);
                uint32_t code;
                const uint4 q = v.codes(&code);
                uint8_t* to = base + size_t(s) * stage + kPWBytes;
                *reinterpret_cast<uint4*>(to + r * kPChunkBytes + ((b ^ (r & 7)) << 4)) = q;
                to[x_bytes + 1024 + (b >> 2) * 512 + r * 16 + (b & 3)] = uint8_t(code);
            };
            const int each = live * 8;
            for (int i = t; i < ahead * each; i += kPEpiThreads) put(c_begin + i / each, i / each, (i % each) >> 3, i & 7);
            fence_proxy_async_smem();
            for (int i = 0; i < ahead; ++i) mbar_arrive(&full[i]);
            Ring r;
            for (int c = c_begin + ahead; c < c_end; ++c) {
                if (!mbar_wait(&empty[r.idx], r.phase, &g_mx4_error, kErrWaitProducer)) break;
                for (int i = t; i < each; i += kPEpiThreads) put(c, int(r.idx), i >> 3, i & 7);
                fence_proxy_async_smem();
                mbar_arrive(&full[r.idx]);
                r.next(uint32_t(p.stages));
            }
            __syncwarp();
        }
    }
    if (warp >= 2) {
        mbar_wait(&done, 0, &g_mx4_error, kErrWaitEpilogue);
        __syncwarp();   // the lanes poll each for itself; the loads from TMEM are the warp's
        tc_fence_after();
        // The accumulator into shared memory (the stages are done with), a
        // row of x after the other: from there a warp stores a row's 128
        // outputs at a time, neighbours together.
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
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (c0 + i < live) part[(c0 + i) * kPTile + quarter * 32 + lane] = __uint_as_float(v[i]);
        }
    }
    // TMEM goes back before any wait for another CTA: a CTA that waits for a
    // peer while it holds TMEM could wait for one that cannot allocate its own.
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, p.tmem_cols);
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = n0 + out_place(p, lane, e);
        bias[e] = p.bias && n < p.n ? p.bias[n] : 0.0f;
    }
    if (p.splits == 1) {
        constexpr int kAhead = 4, kStep = kPThreads / 32;
        for (int i0 = warp; i0 < live; i0 += kStep * kAhead) {
            float v[kAhead][4];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (i0 + u * kStep < live) load_four(p, part + (i0 + u * kStep) * kPTile, lane, v[u]);
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (i0 + u * kStep < live) store_four<T>(p, x0 + i0 + u * kStep, n0, lane, v[u], bias);
        }
        return;
    }
    // The parts' sum, in order of K (the same bits on every run): CTA `split`
    // finishes rows split, split + splits, ... of the tile.
    __syncwarp();
    cluster_sync();
    constexpr int kAhead = 4;   // rows whose parts are all asked for before the first sum
    const int step = p.splits * (kPThreads / 32);
    for (int i0 = split + p.splits * warp; i0 < live; i0 += step * kAhead) {
        float v[kAhead][kPMaxSplits][4];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i0 + u * step >= live) break;
            const uint32_t at = smem_u32(part + (i0 + u * step) * kPTile);
#pragma unroll
            for (int r = 0; r < kPMaxSplits; ++r)
                if (r < p.splits) load_four_of(mapa(at, uint32_t(r)), lane, v[u][r]);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * step;
            if (i >= live) break;
            float sum[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[e] = v[u][0][e];
#pragma unroll
                for (int r = 1; r < kPMaxSplits; ++r)
                    if (r < p.splits) sum[e] += v[u][r][e];
            }
            store_four<T>(p, x0 + i, n0, lane, sum, bias);
        }
    }
    __syncwarp();
    cluster_sync();   // no CTA leaves while another reads its part
}

// ------------------------------------------------- product by CTA pairs

// Large products: the two CTAs of a cluster compute 256 x 256 tiles together
// (cta_group::2, M = 256). Each stages 128 rows of either operand, so that a
// tile's operands cross from L2 to 2/3 of the bytes that 128 x 256 tiles take
// (those were bound by L2: 8192^3 at 12 TB/s of it). Persistent: a pair takes
// every (number of pairs)-th tile, and its copies run ahead into the next
// tile while the epilogue drains. The epilogue's eight warps read their whole
// share of the accumulator into registers and free it before converting and
// storing. 8192^3 in 178 to 185 us: 5.9 to 6.2 PFLOP/s, at which the GPU is at
// its power limit (1.5 GHz); 4096^3, 3.5 tiles a pair, in 31 us.
//
// kRowsOnLanes: TMEM's lanes are rows of x, so a thread holds neighbouring
// outputs of one row; its warp lays them out in shared memory, 32 rows of 128
// bytes at a time, and TMA stores them (where `out` is aligned for it; 16-byte
// stores of 32 lanes into 32 rows took 6600 cycles a tile). Otherwise the
// lanes are rows of w and a warp stores 32 neighbouring outputs at a time,
// whatever the alignment (6000 x 2049 x 64 into bfloat16 in 19 us, 6000 x 2048
// x 64 by boxes in 13; 4096 x 4097 x 4096 37 us, x 4096 30).
struct PairTile {
    int lanes, cols;                 // rows of the operand on the lanes and of the other
    int lane_tiles, tiles;           // tiles along the lanes, and in all
    int chunks, steps, scale_tiles;  // as in ProductTile
    const float* bias;
    int relu;
    void* out;
    long long ld;
};

// From so many tiles, and more than 128 rows on either side: 64 tiles of
// 1024 x 4096 x 2048 11.6 us by pairs and 16.9 us without, 32 of 512 x 4096 x
// 4096 12.9 and 11.7 (with x's quantisation).
constexpr int kPairFromTiles = 48;
constexpr int kPairThreads = 320, kPairEpiWarps = 8, kPairStages = 5;
constexpr uint32_t kPairBox = 32 * 128;   // an epilogue warp's rows on their way out
constexpr uint32_t kPairScaleCols = 24, kPairTmemCols = 512;   // per stage: 2 x 4 of the lanes' scales, 2 x 8 of the columns'
constexpr uint32_t kPairStageBytes = 2 * kPWBytes + 1024 + 2048;

__device__ __forceinline__ void tmem_copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void umma_mx4_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                              uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

template <typename T, bool kRowsOnLanes>
__global__ void __launch_bounds__(kPairThreads, 1)
    mx4_pair_kernel(const __grid_constant__ CUtensorMap ml, const __grid_constant__ CUtensorMap mc,
                    const __grid_constant__ CUtensorMap sl, const __grid_constant__ CUtensorMap sc,
                    const __grid_constant__ CUtensorMap mo, const PairTile p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[kPairStages], empty[kPairStages], acc_full, acc_empty, done;
    __shared__ uint32_t tmem_slot;
    const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pairs = int(gridDim.x) >> 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPairStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(&acc_full, 1);
        mbar_init(&acc_empty, 2 * kPairEpiWarps);   // every epilogue warp of both CTAs
        mbar_init(&done, 1);
        fence_barrier_init();
        tma_prefetch_map(&ml);
        tma_prefetch_map(&mc);
        tma_prefetch_map(&sl);
        tma_prefetch_map(&sc);
    }
    if (warp == 1) tmem_alloc_pair(&tmem_slot, kPairTmemCols);
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // both CTAs' barriers exist before either addresses the other's
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    grid_dependency_wait();
    grid_launch_dependents();

    if (warp == 0) {
        if (elect_one()) {
            Ring r;
            uint32_t issued = 0;
            const uint32_t full0 = mapa(smem_u32(full), 0);   // both CTAs' copies complete on the leader's barriers
            bool ok = true;
            for (int tile = int(blockIdx.x) >> 1; tile < p.tiles && ok; tile += pairs) {
                const int tl = tile % p.lane_tiles, tc = tile / p.lane_tiles;
                const int yl = tl * 256 + int(rank) * 128, yc = tc * 256 + int(rank) * 128;
                const int zl = (yl >> 7) * p.scale_tiles, zc = 2 * tc * p.scale_tiles;
                for (int c = 0; c < p.chunks; ++c) {
                    if (!(ok = mbar_wait(&empty[r.idx], r.phase ^ 1u, &g_mx4_error, kErrWaitProducer))) break;
                    if (rank == 0) mbar_arrive_expect_tx(&full[r.idx], 2 * kPairStageBytes);
                    uint8_t* b = base + r.idx * kPairStageBytes;
                    const uint32_t bar = full0 + r.idx * 8u;
                    tma_load_2d_pair(&ml, b, bar, c * kPChunkBytes, yl);
                    tma_load_2d_pair(&mc, b + kPWBytes, bar, c * kPChunkBytes, yc);
                    // Two scale tiles of 512 bytes at a time. Past an odd last one
                    // this reads another row tile's (or zeros), which no MMA uses.
                    tma_load_2d_pair(&sl, b + 2 * kPWBytes, bar, 0, zl + 2 * c);
                    tma_load_2d_pair(&sc, b + 2 * kPWBytes + 1024, bar, 0, zc + 2 * c);
                    tma_load_2d_pair(&sc, b + 2 * kPWBytes + 2048, bar, 0, zc + p.scale_tiles + 2 * c);
                    r.next(kPairStages);
                    ++issued;
                }
            }
            // The leader's full barriers count both CTAs' copies: once each
            // stage's last phase has completed, every copy of the pair has landed.
            if (rank == 0)
                for (uint32_t i = issued > kPairStages ? issued - kPairStages : 0; i < issued; ++i)
                    mbar_wait(&full[i % kPairStages], (i / kPairStages) & 1u, &g_mx4_error, kErrWaitDrain);
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            Ring r;
            uint32_t j = 0;
            bool ok = true;
            const uint32_t empty0 = mapa(smem_u32(empty), 0), empty1 = mapa(smem_u32(empty), 1);
            const uint32_t full_a = mapa(smem_u32(&acc_full), 0), full_b = mapa(smem_u32(&acc_full), 1);
            constexpr uint32_t kIdesc = (1u << 7) | (1u << 10) | (uint32_t(256 >> 3) << 17) | (1u << 23) | (uint32_t(256 >> 4) << 24);
            constexpr uint32_t kSecond = (2u << 4) | (2u << 29);   // the scale words' upper two bytes
            for (int tile = int(blockIdx.x) >> 1; tile < p.tiles && ok; tile += pairs, ++j) {
                if (!(ok = mbar_wait_cluster(&acc_empty, (j & 1u) ^ 1u, &g_mx4_error, kErrWaitMma))) break;
                tc_fence_after();
                uint32_t more = 0;
                for (int c = 0; c < p.chunks; ++c) {
                    if (!(ok = mbar_wait(&full[r.idx], r.phase, &g_mx4_error, kErrWaitMma))) break;
                    tc_fence_after();
                    const uint32_t b = smem_u32(base) + r.idx * kPairStageBytes;
                    const uint32_t tw = tmem + 256u + r.idx * kPairScaleCols;
                    auto tile_of = [&](int t, bool both) {
                        const uint64_t z = scale_desc(b + 2 * kPWBytes) + uint64_t(t * 32);
                        const uint32_t fl = tw + uint32_t(t) * 4, fc = tw + 8 + uint32_t(t) * 8;
                        tmem_copy_scales_pair(fl, z);
                        tmem_copy_scales_pair(fc, z + 64);
                        tmem_copy_scales_pair(fc + 4, z + 128);
                        const uint64_t da = sw128_desc(b) + uint64_t(4 * t), db = sw128_desc(b + kPWBytes) + uint64_t(4 * t);
                        umma_mx4_pair(tmem, da, db, kIdesc, fl, fc, more);
                        more = 1;
                        if (both) umma_mx4_pair(tmem, da + 2, db + 2, kIdesc | kSecond, fl, fc, 1);
                    };
                    const int steps = p.steps - 4 * c;
                    if (steps >= 4) {
                        tile_of(0, true);
                        tile_of(1, true);
                    } else {
                        tile_of(0, steps > 1);
                        if (steps > 2) tile_of(1, false);
                    }
                    umma_commit_pair(empty0 + r.idx * 8u);
                    umma_commit_pair(empty1 + r.idx * 8u);
                    r.next(kPairStages);
                }
                if (!ok) break;
                umma_commit_pair(full_a);
                umma_commit_pair(full_b);
            }
            umma_commit_pair(mapa(smem_u32(&done), 0));
            mbar_wait(&done, 0, &g_mx4_error, kErrWaitDrain);
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t taddr = tmem + (uint32_t(quarter) << 21) + uint32_t(half) * 128;
        const uint32_t to_leader = mapa(smem_u32(&acc_empty), 0);
        T* const out = static_cast<T*>(p.out);
        const float floor = p.relu ? 0.0f : __uint_as_float(0xFF800000u);
        uint8_t* const boxes = base + size_t(kPairStages) * kPairStageBytes;   // 1024-byte aligned, as the swizzle needs
        uint8_t* const box = boxes + size_t(warp - 2) * kPairBox;
        float* const bias_of = reinterpret_cast<float*>(boxes + kPairEpiWarps * kPairBox) + (warp - 2) * 128;   // of its columns
        uint32_t j = 0;
        for (int tile = int(blockIdx.x) >> 1; tile < p.tiles; tile += pairs, ++j) {
            // The lanes poll each for itself; the loads from TMEM are the warp's.
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(&acc_full, j & 1u, &g_mx4_error, kErrWaitEpilogue))) break;
            tc_fence_after();
            uint32_t v[4][32];
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld32(taddr + uint32_t(q) * 32, v[q]);
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_hold(v[q]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(to_leader);
            const int l = (tile % p.lane_tiles) * 256 + int(rank) * 128 + quarter * 32 + lane;
            const int c0 = tile / p.lane_tiles * 256 + half * 128;
            const auto act = [&](uint32_t bits, float bias) {
                const float y = __uint_as_float(bits) + bias;
                return y < floor ? floor : y;   // keeps a NaN
            };
            if constexpr (kRowsOnLanes) {
                constexpr int kW = 16 / int(sizeof(T)), kCols = 8 * kW;   // columns in 16 and in 128 bytes
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = lane + 32 * e;
                    bias_of[i] = p.bias && c0 + i < p.cols ? __ldg(p.bias + c0 + i) : 0.0f;
                }
#pragma unroll
                for (int q = 0; q < 128 / kCols; ++q) {
                    if (lane == 0) bulk_wait_read<0>();   // the box's previous store has read it
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        float y[kW];
#pragma unroll
                        for (int e = 0; e < kW; ++e) {
                            const int i = q * kCols + u * kW + e;
                            y[e] = act(v[i >> 5][i & 31], bias_of[i]);
                        }
                        uint4 w;
                        if constexpr (sizeof(T) == 2) {
#pragma unroll
                            for (int e = 0; e < kW; e += 2)
                                reinterpret_cast<__nv_bfloat162*>(&w)[e >> 1] = __floats2bfloat162_rn(y[e], y[e + 1]);
                        } else {
#pragma unroll
                            for (int e = 0; e < kW; ++e) reinterpret_cast<float*>(&w)[e] = y[e];
                        }
                        *reinterpret_cast<uint4*>(box + lane * 128 + ((u ^ (lane & 7)) << 4)) = w;   // (128-byte swizzle)
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0 && l < p.lanes && c0 + q * kCols < p.cols) tma_store_2d(&mo, box, c0 + q * kCols, l);
                    if (lane == 0) bulk_commit();
                }
            } else {
                const bool in = l < p.lanes;
                const float bias = p.bias && in ? __ldg(p.bias + l) : 0.0f;
                T* dst = out + size_t(c0) * size_t(p.ld) + l;
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (in && c0 + q * 32 + i < p.cols) *dst = T(act(v[q][i], bias));
                        dst += p.ld;
                    }
            }
        }
        if (kRowsOnLanes && lane == 0) bulk_wait_all();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // no remote arrival or pair MMA is still in flight
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, kPairTmemCols);
    }
}

template <typename T, bool kRowsOnLanes>
cudaError_t launch_pair(const MxProductArgs& a, int sms, cudaStream_t s) {
    const MxShape xs{a.m, a.k}, ws{a.n, a.k};
    const MxShape& ls = kRowsOnLanes ? xs : ws;
    const MxShape& cs = kRowsOnLanes ? ws : xs;
    const uint8_t* lc = kRowsOnLanes ? a.x_codes : a.w_codes;
    const uint8_t* cc = kRowsOnLanes ? a.w_codes : a.x_codes;
    const uint8_t* lsc = kRowsOnLanes ? a.x_scales : a.w_scales;
    const uint8_t* csc = kRowsOnLanes ? a.w_scales : a.x_scales;
    PairTile p{};
    p.lanes = int(ls.rows);
    p.cols = int(cs.rows);
    p.lane_tiles = int((ls.rows + 255) / 256);
    p.tiles = p.lane_tiles * int((cs.rows + 255) / 256);
    p.chunks = int((a.k + 255) / 256);
    p.steps = int((a.k + 63) / 64);
    p.scale_tiles = int(ls.scale_tiles());
    p.bias = a.bias;
    p.relu = a.relu;
    p.out = a.out;
    p.ld = a.ld;
    const CUtensorMap ml = make_byte_map(lc, uint64_t(ls.pitch()), uint64_t(ls.rows), 128);
    const CUtensorMap mc = make_byte_map(cc, uint64_t(cs.pitch()), uint64_t(cs.rows), 128);
    const CUtensorMap sl = make_scale_map(lsc, uint64_t(ls.row_tiles()) * uint64_t(ls.scale_tiles()));
    const CUtensorMap sc = make_scale_map(csc, uint64_t(cs.row_tiles()) * uint64_t(cs.scale_tiles()));
    const CUtensorMap mo = kRowsOnLanes ? make_out_map(a.out, a.type, uint64_t(a.n), uint64_t(a.m), uint64_t(a.ld)) : ml;
    const size_t smem = 1024 + size_t(kPairStages) * kPairStageBytes + (kRowsOnLanes ? kPairEpiWarps * (kPairBox + 512) : 0);
    if (const cudaError_t e = open_smem<mx4_pair_kernel<T, kRowsOnLanes>>(smem); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(2 * std::min(p.tiles, sms / 2)));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {2, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, mx4_pair_kernel<T, kRowsOnLanes>, ml, mc, sl, sc, mo, p);
}

// Whether TMA can store rows of `out`: they start at multiples of 16 bytes and
// end at such. (Of a row that ends elsewhere it writes the last 16 bytes whole,
// into what lies between the caller's rows.)
bool out_aligned(const MxProductArgs& a) {
    const size_t es = elem_size(a.type);
    return reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && size_t(a.ld) * es % 16 == 0 && size_t(a.n) * es % 16 == 0;
}

template <typename T, int kGroups, typename X>
cudaError_t launch_product_t(const CUtensorMap& mw, const CUtensorMap& mx, const ProductTile& p, dim3 grid,
                             cudaStream_t s) {
    const size_t smem = 1024 + size_t(p.stages) * stage_bytes(p.tn);
    if (const cudaError_t e = open_smem<mx4_product_kernel<T, kGroups, X>>(smem); e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kPThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int na = 0;
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
    if (p.splits > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na++].val.clusterDim = {unsigned(p.splits), 1, 1};
    }
    cfg.attrs = attr;
    cfg.numAttrs = unsigned(na);
    return cudaLaunchKernelEx(&cfg, mx4_product_kernel<T, kGroups, X>, mw, mx, p);
}

}  // namespace

cudaError_t launch_mx4_quantise(const MxCastArgs& a, int sms, cudaStream_t s) {
    const int span = a.type == kElemBF16 ? kCastSpan<__nv_bfloat16> : kCastSpan<float>;
    const dim3 grid = cast_grid(a.shape.row_tiles() * 128, a.shape.scale_tiles() * 128, span, sms);
    const int bytes = row_bytes(a.plain, a.shape.rows, a.ld, a.type);
    if (a.type == kElemBF16)
        return bytes == 16  ? launch_pdl(mx4_quantise_kernel<__nv_bfloat16, 16>, grid, dim3(kCastThreads), 0, s, a)
               : bytes == 8 ? launch_pdl(mx4_quantise_kernel<__nv_bfloat16, 8>, grid, dim3(kCastThreads), 0, s, a)
                            : launch_pdl(mx4_quantise_kernel<__nv_bfloat16, 0>, grid, dim3(kCastThreads), 0, s, a);
    return bytes == 16 ? launch_pdl(mx4_quantise_kernel<float, 16>, grid, dim3(kCastThreads), 0, s, a)
                       : launch_pdl(mx4_quantise_kernel<float, 0>, grid, dim3(kCastThreads), 0, s, a);
}

cudaError_t launch_mx4_values(const MxCastArgs& a, int sms, cudaStream_t s) {
    const dim3 grid = cast_grid(a.shape.rows, a.shape.cols, kValuesSpan, sms);
    const int bytes = row_bytes(a.plain, a.shape.rows, a.ld, a.type);
    if (a.type == kElemF32) return launch_pdl(mx4_values_kernel<float, 0>, grid, dim3(kCastThreads), 0, s, a);
    return bytes == 16  ? launch_pdl(mx4_values_kernel<__nv_bfloat16, 16>, grid, dim3(kCastThreads), 0, s, a)
           : bytes == 8 ? launch_pdl(mx4_values_kernel<__nv_bfloat16, 8>, grid, dim3(kCastThreads), 0, s, a)
           : bytes == 4 ? launch_pdl(mx4_values_kernel<__nv_bfloat16, 4>, grid, dim3(kCastThreads), 0, s, a)
                        : launch_pdl(mx4_values_kernel<__nv_bfloat16, 0>, grid, dim3(kCastThreads), 0, s, a);
}

namespace {

// How a product is cut up.
struct ProductPlan {
    bool pairs;            // 256 x 256 tiles by CTA pairs
    int tn, n_tiles, x_tiles, splits, per_cta, stages;
    bool quantises;        // a plain x is quantised by the product's own CTAs
};

ProductPlan plan_of(long long m, long long n, long long k) {
    constexpr int kSms = 148;
    ProductPlan p{};
    if (m > 128 && n > 128 && (m + 255) / 256 * ((n + 255) / 256) >= kPairFromTiles) {
        p.pairs = true;
        return p;
    }
    const int chunks = int((k + 255) / 256);
    // Columns per tile: as few as hold all of x up to 128; more rows of x in
    // tiles of 256 where those alone fill the SMs, else 128, else 64.
    p.n_tiles = int((n + kPTile - 1) / kPTile);
    if (m <= 128) p.tn = int((m + 15) / 16 * 16);
    else p.tn = 64;
    for (const int tn : {128, 256})
        if (m > 128 && (m + tn - 1) / tn * p.n_tiles >= kSms) p.tn = tn;
    p.x_tiles = int((m + p.tn - 1) / p.tn);
    // Up to 64 columns a CTA takes half an SM's memory. K is shared by a
    // cluster of CTAs while there are SMs for them (over a long K two CTAs an
    // SM, so that one's waits fill the other's: 1 x 8192 x 8192 6.9 us so, 10.3
    // us with one; 64 x 4096 x 4096 9.2 and 7.9), every CTA keeps a chunk or
    // more and there are enough of them to pay for the exchange (1024 x 362 x
    // 722, three chunks: 6.8 us in one piece, 9.1 us in two).
    const int slots = p.tn <= 64 && chunks >= 32 ? 2 * kSms : kSms;
    p.splits = 1;
    while (chunks >= 4 && p.splits < kPMaxSplits && (long long)p.n_tiles * p.x_tiles * p.splits * 2 <= slots &&
           p.splits * 2 <= chunks)
        p.splits *= 2;
    p.per_cta = (chunks + p.splits - 1) / p.splits;
    const size_t budget = p.tn <= 64 ? size_t(108) << 10 : size_t(220) << 10;
    p.stages = int(std::min<size_t>(kPMaxStages, budget / stage_bytes(p.tn)));
    p.stages = std::max(1, std::min(p.stages, p.per_cta));
    // The accumulator passes through the stages' memory: 512 bytes a column.
    while (size_t(p.stages) * stage_bytes(p.tn) < size_t(p.tn) * kPTile * 4) ++p.stages;
    p.quantises = m <= kPPlainRows && p.per_cta <= kPPlainChunks;
    return p;
}

}  // namespace

bool mx4_product_quantises(long long m, long long n, long long k) { return plan_of(m, n, k).quantises; }

cudaError_t launch_mx4_product(const MxProductArgs& a, int sms, cudaStream_t s) {
    const ProductPlan plan = plan_of(a.m, a.n, a.k);
    if (plan.pairs) {
        if (a.type == kElemBF16) return out_aligned(a) ? launch_pair<__nv_bfloat16, true>(a, sms, s) : launch_pair<__nv_bfloat16, false>(a, sms, s);
        return out_aligned(a) ? launch_pair<float, true>(a, sms, s) : launch_pair<float, false>(a, sms, s);
    }
    const MxShape xs{a.m, a.k}, ws{a.n, a.k};
    ProductTile p{};
    p.m = int(a.m);
    p.n = int(a.n);
    p.chunks = int((a.k + 255) / 256);
    p.steps = int((a.k + 63) / 64);
    p.scale_tiles = int(xs.scale_tiles());
    p.tn = plan.tn;
    p.stages = plan.stages;
    p.splits = plan.splits;
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
    p.out_fours = reinterpret_cast<uintptr_t>(a.out) % (4 * elem_size(a.type)) == 0 && a.ld % 4 == 0;
    p.x = a.x;
    p.x_ld = a.x_ld;
    p.k = int(a.k);
    p.x_aligned = a.x && row_bytes(a.x, a.m, a.x_ld, a.x_type) == 16;
    const CUtensorMap mw = make_byte_map(a.w_codes, uint64_t(ws.pitch()), uint64_t(a.n), kPTile);
    const CUtensorMap mx = a.x ? mw : make_byte_map(a.x_codes, uint64_t(xs.pitch()), uint64_t(a.m), uint32_t(p.tn));
    const dim3 grid(unsigned(plan.n_tiles * p.splits), unsigned(plan.x_tiles));
    const auto launch = [&](auto out) {
        using T = decltype(out);
        if (a.x) return a.x_type == kElemBF16 ? launch_product_t<T, 1, __nv_bfloat16>(mw, mx, p, grid, s)
                                              : launch_product_t<T, 1, float>(mw, mx, p, grid, s);
        return p.tn > 128 ? launch_product_t<T, 2, void>(mw, mx, p, grid, s)
                          : launch_product_t<T, 1, void>(mw, mx, p, grid, s);
    };
    return a.type == kElemBF16 ? launch(__nv_bfloat16()) : launch(0.0f);
}

cudaError_t mx4_error(int* code) {
    *code = 0;
    const cudaError_t e = cudaDeviceSynchronize();
    return e == cudaSuccess ? cudaMemcpyFromSymbol(code, g_mx4_error, sizeof(int)) : e;
}

cudaError_t mx4_error_probe(unsigned long long limit_ns) {
    void* word = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&word, g_mx4_error);
    return e == cudaSuccess ? launch_bounded_wait_probe(static_cast<int*>(word), limit_ns, nullptr) : e;
}

}  // namespace azb
