// The operators beside the network: 4-bit microscaled matrices (mx4.cu) and
// the move sampler (sample.cu), as the C ABI (ops_capi.cu) launches them.
// They work on device memory in the caller's stream: no launch here
// allocates, synchronises or keeps anything from one call to the next.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace azb {

enum ElemType : int { kElemF32 = 0, kElemBF16 = 1 };
inline size_t elem_size(int type) { return type == kElemBF16 ? 2 : 4; }

// ------------------------------------------------- 4-bit microscaled matrix
//
// rows x cols elements in blocks of 32 along a row. Codes: [rows][16 bytes
// per block], E2M1, element 2i in the low half of byte i, zeros past cols.
// Scales: one E8M0 byte per block, in tiles of 128 rows x 4 blocks (512
// bytes, the order in which the tensor core's scale columns are filled):
// row r, block b at ((r / 128) * ceil(blocks / 4) + b / 4) * 512
// + (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4; zeros outside the matrix.
constexpr int kMxBlock = 32;
struct MxShape {
    long long rows, cols;
    __host__ __device__ long long blocks() const { return (cols + kMxBlock - 1) / kMxBlock; }
    __host__ __device__ long long pitch() const { return blocks() * 16; }
    __host__ __device__ long long scale_tiles() const { return (blocks() + 3) / 4; }   // per 128 rows
    __host__ __device__ long long row_tiles() const { return (rows + 127) / 128; }
    size_t code_bytes() const { return size_t(rows) * size_t(pitch()); }
    size_t scale_bytes() const { return size_t(row_tiles()) * size_t(scale_tiles()) * 512; }
};

struct MxCastArgs {
    MxShape shape;
    void* plain;            // quantise: the source; values: the destination
    int type;               // ElemType of `plain`
    long long ld;           // elements from one row of `plain` to the next
    uint8_t* codes;
    uint8_t* scales;
};
cudaError_t launch_mx4_quantise(const MxCastArgs& a, int sms, cudaStream_t s);
cudaError_t launch_mx4_values(const MxCastArgs& a, int sms, cudaStream_t s);

// out[i][j] = act(sum_k x[i][k] w[j][k] + bias[j]), i < m, j < n; w and x in
// the 4-bit form. after_quantise: the launch before this one on the stream
// is the quantisation of x (and of nothing else), which this one overlaps.
struct MxProductArgs {
    const uint8_t* x_codes;
    const uint8_t* x_scales;
    const uint8_t* w_codes;
    const uint8_t* w_scales;
    long long m, n, k;
    const float* bias;   // [n] or null
    int relu;
    void* out;
    int type;            // ElemType of `out`
    long long ld;        // elements from one row of `out` to the next
    bool after_quantise;
    // Plain x in place of its codes and scales (then null), where
    // mx4_product_quantises(m, n, k).
    const void* x = nullptr;
    int x_type = 0;
    long long x_ld = 0;
};
// Whether the product quantises a plain x itself.
bool mx4_product_quantises(long long m, long long n, long long k);
cudaError_t launch_mx4_product(const MxProductArgs& a, int sms, cudaStream_t s);
// The product kernels' error word on the current device (KernelError; 0:
// none), read after waiting for the device.
cudaError_t mx4_error(int* code);
// A wait of limit_ns that runs out and is recorded there.
cudaError_t mx4_error_probe(unsigned long long limit_ns);

// ------------------------------------------------------------ move sampler

struct SampleArgs {
    const void* logits;
    int type;                // ElemType
    long long rows, ld;
    int cols;
    const float* noise;      // uniform numbers, [rows][cols], rows noise_ld apart
    long long noise_ld;
    const uint8_t* legal;    // or null: all legal
    long long legal_ld;
    float temperature, top_p, min_p;
    int top_k;
    const float* temperature_rows;   // per row, or null: the number above
    const float* top_p_rows;
    const float* min_p_rows;
    const int* top_k_rows;
    long long* moves;
    float* logprob;          // or null
};
cudaError_t launch_sample_moves(const SampleArgs& a, cudaStream_t s);

// A map of `rows` rows of `pitch` bytes (pitch a multiple of 16) in boxes of
// 128 bytes x box_rows rows, 128-byte swizzle.
CUtensorMap make_byte_map(const void* base, uint64_t pitch, uint64_t rows, uint32_t box_rows);
// A map of `tiles` scale tiles of 512 bytes, in boxes of two.
CUtensorMap make_scale_map(const void* base, uint64_t tiles);
// A map of rows x cols elements of an ElemType (rows `ld` elements apart, a
// multiple of 16 bytes) in boxes of 32 rows x 128 bytes, 128-byte swizzle.
CUtensorMap make_out_map(void* base, int type, uint64_t cols, uint64_t rows, uint64_t ld);

}  // namespace azb
