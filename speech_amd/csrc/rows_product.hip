// rows_product.hip -- Y = A B^T + bias for matrices in 8-bit form (e4m3 values, a power-of-two scale for each 128 columns), gfx950.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes one k-step of 128, which is one block of scales, and applies both operands' scale exponents
// inside the matrix unit: no vector instruction touches the sums before the epilogue.  Operands: lane l holds row l & 15 of a
// 16-row tile and 32 bytes of its k-step; which 32 is free as long as A and B agree, because a sum over k does not care about
// order and all 128 share their scale.  The unit adds the eight products of 8 bytes of a lane at a resolution of 2^-13 of the largest
// (measured: beside 448 x 448 a product of 2^3 counts, one of 2^2 is lost), the rest in 32-bit floats.  Result: lane l holds column l & 15 (B's row), rows 4 (l >> 4) ... + 3.
#include "rows_internal.hpp"

namespace speech {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v4f mfma_scaled(v8i a, v8i b, v4f c, int sa, int sb)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// the first `left` of 16 bytes, the others 0 (what stands behind a row may be anything, NaN included)
__device__ __forceinline__ uint4 keep_bytes(uint4 v, int left)
{
    unsigned *w = reinterpret_cast<unsigned *>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const int n = left - 4 * i;
        w[i] = n >= 4 ? w[i] : (n <= 0 ? 0u : w[i] & (0xFFFFFFFFu >> (8 * (4 - n))));
    }
    return v;
}

// 32 bytes of a row from k on: 16 bytes at k and 16 at k + 64, zeros from K on
__device__ __forceinline__ v8i load_frag(const uint8_t *row, size_t k, size_t K)
{
    uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
    if (k + 80 <= K)
    {
        x = *reinterpret_cast<const uint4 *>(row + k);
        y = *reinterpret_cast<const uint4 *>(row + k + 64);
    }
    else
    {
        if (k < K) { x = keep_bytes(*reinterpret_cast<const uint4 *>(row + k), (int)min(K - k, (size_t)16)); }
        if (k + 64 < K) { y = keep_bytes(*reinterpret_cast<const uint4 *>(row + k + 64), (int)min(K - k - 64, (size_t)16)); }
    }
    v8i r;
    r[0] = (int)x.x; r[1] = (int)x.y; r[2] = (int)x.z; r[3] = (int)x.w;
    r[4] = (int)y.x; r[5] = (int)y.y; r[6] = (int)y.z; r[7] = (int)y.w;
    return r;
}

// A workgroup computes 16 MT x 16 NN values; its WAVES waves split the k-steps and add their sums in wave order through LDS.
// Operands come straight from memory.
template <typename T, int MT, int NN, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void product_split_kernel(const ProductParams p, unsigned ntiles)
{
    __shared__ float part[WAVES][MT * NN][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
    const unsigned tm = blockIdx.x / ntiles, tn = blockIdx.x - tm * ntiles;
    const size_t m0 = (size_t)tm * 16 * MT, n0 = (size_t)tn * 16 * NN;
    const int nb = (int)((p.K + ROWS_BLOCK - 1) / ROWS_BLOCK);
    size_t ra[MT], rb[NN];
#pragma unroll
    for (int i = 0; i < MT; ++i) { const size_t r = m0 + 16 * i + l16; ra[i] = r < p.M ? r : p.M - 1; }
#pragma unroll
    for (int i = 0; i < NN; ++i) { const size_t r = n0 + 16 * i + l16; rb[i] = r < p.N ? r : p.N - 1; }
    v4f acc[MT][NN];
#pragma unroll
    for (int i = 0; i < MT; ++i)
    {
#pragma unroll
        for (int j = 0; j < NN; ++j) { acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f}; }
    }
    for (int b = wave; b < nb; b += WAVES)
    {
        const size_t k = (size_t)b * ROWS_BLOCK + g * 16;
        v8i fa[MT], fb[NN];
        int sa[MT], sb[NN];
#pragma unroll
        for (int i = 0; i < MT; ++i) { fa[i] = load_frag(p.A + ra[i] * p.lda, k, p.K); sa[i] = p.SA[ra[i] * p.ldsa + b]; }
#pragma unroll
        for (int i = 0; i < NN; ++i) { fb[i] = load_frag(p.B + rb[i] * p.ldb, k, p.K); sb[i] = p.SB[rb[i] * p.ldsb + b]; }
#pragma unroll
        for (int i = 0; i < MT; ++i)
        {
#pragma unroll
            for (int j = 0; j < NN; ++j) { acc[i][j] = mfma_scaled(fa[i], fb[j], acc[i][j], sa[i], sb[j]); }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
    {
#pragma unroll
        for (int j = 0; j < NN; ++j)
        {
#pragma unroll
            for (int q = 0; q < 4; ++q) { part[wave][i * NN + j][(4 * g + q) * 16 + l16] = acc[i][j][q]; }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < MT * NN * 256; e += 64 * WAVES)
    {
        const int tile = e >> 8, i = tile / NN, j = tile - i * NN, r = (e >> 4) & 15, c = e & 15;
        const size_t m = m0 + 16 * i + r, n = n0 + 16 * j + c;
        if (m >= p.M || n >= p.N) { continue; }
        float s = part[0][tile][e & 255];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) { s += part[w][tile][e & 255]; }
        if (p.bias) { s += p.bias[n]; }
        reinterpret_cast<T *>(p.Y)[m * p.ldy + n] = (T)s;
    }
}

template <typename T>
void product_go(const ProductParams &p, hipStream_t s)
{
    const size_t tm = (p.M + 31) / 32, tn = (p.N + 31) / 32;
    hipLaunchKernelGGL((product_split_kernel<T, 2, 2, 4>), dim3((unsigned)(tm * tn)), dim3(256), 0, s, p, (unsigned)tn);
}

}  // namespace

hipError_t launch_rows_product(int dtype, const ProductParams &p, hipStream_t s)
{
    switch (dtype)
    {
        case SPEECH_BF16: product_go<__bf16>(p, s); break;
        case SPEECH_F16: product_go<_Float16>(p, s); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace speech
