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

// ---- large products: tiles through LDS ----
// A workgroup computes TM x TN values with WM x WN waves, each (TM / WM) x (TN / WN) of them.  One k-step (128 bytes of TM + TN rows)
// is a stage in LDS; global_load_lds brings the next one while the matrix unit works on this one.
//
// In LDS a row is 8 chunks of 16 bytes, chunk c at place c ^ f(row), so that the lanes that read one chunk of neighbouring rows meet all
// banks; the loads write LDS in order and permute what they fetch instead.
//
// The unit gets B as its first operand, so that a lane's four results are four columns of one row of Y; which of a wave's rows of B sits at
// which place of which 16-row tile is chosen so that all of a lane's columns are next to each other: 4 NN values, one or more 16-byte
// stores.
__device__ __forceinline__ int swizzle_a(int row) { return row & 7; }
template <int NN> __device__ __forceinline__ int swizzle_b(int row) { return (row & 3) | (((row / (4 * NN)) & 1) << 2); }

// 16 bytes a lane from base + off into LDS at lds + 16 lane.  As an instruction of its own, because the compiler waits for every load
// into LDS that it knows of before it reads any LDS; the waits are the caller's (vmcnt(0) before the barrier that publishes a
// stage).  No register is written: nothing of the compiler's can be overtaken.
__device__ __forceinline__ void load_to_lds(const uint8_t *base, unsigned off, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
// a dword a lane from its own address into LDS at lds + 4 lane
__device__ __forceinline__ void load_dword_to_lds(const uint8_t *from, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds), "v"(from) : "memory", "m0");
}

template <typename T, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product_tile_kernel(const ProductParams p, unsigned tiles_m, unsigned tiles_n)
{
    constexpr int NTH = 64 * WM * WN, MT = TM / WM / 16, NN = TN / WN / 16, STAGE = (TM + TN) * 128;
    constexpr int LA = TM * 8 / NTH, LB = TN * 8 / NTH;                      // 16-byte loads a thread makes for a stage
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;

    // XCDs take workgroups in turn: each gets a run of consecutive tiles, which walk 8 tiles of rows at a time so that the 32 tiles an XCD
    // works on share their rows of A and B in its L2
    const unsigned total = tiles_m * tiles_n, per = (total + 7) / 8;
    const unsigned tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (tile >= total) { return; }
    const unsigned band = tile / (8 * tiles_n), in = tile - band * 8 * tiles_n, bh = min(8u, tiles_m - band * 8);
    const size_t m0 = (size_t)(band * 8 + in % bh) * TM, n0 = (size_t)(in / bh) * TN;

    const int nb = (int)((p.K + 127) / 128);
    const int am = (int)min(p.M - m0, (size_t)TM) - 1, bm = (int)min(p.N - n0, (size_t)TN) - 1;     // last row of the tile that exists
    const uint8_t *A = p.A + m0 * p.lda, *B = p.B + n0 * p.ldb;
    const unsigned lda = (unsigned)p.lda, ldb = (unsigned)p.ldb;
    unsigned oa[LA], ob[LB];
#pragma unroll
    for (int i = 0; i < LA; ++i)
    {
        const int row = i * (NTH / 8) + tid / 8;
        oa[i] = (unsigned)min(row, am) * lda + (unsigned)(((tid & 7) ^ swizzle_a(row)) * 16);
    }
#pragma unroll
    for (int i = 0; i < LB; ++i)
    {
        const int row = i * (NTH / 8) + tid / 8;
        ob[i] = (unsigned)min(row, bm) * ldb + (unsigned)(((tid & 7) ^ swizzle_b<NN>(row)) * 16);
    }
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds + (unsigned)wave * 1024u);
    const int last = (int)(p.K - (size_t)(nb - 1) * 128);                    // bytes of the last k-step: 1 ... 128

    // chunks that start at or behind K are fetched from the row's first bytes (they are cleared in LDS below)
    auto fetch = [&](int kb, int stage)
    {
        const bool cut = kb == nb - 1 && last < 128;
        const size_t k = (size_t)kb * 128;
        const unsigned dst = lds0 + (unsigned)(stage * STAGE);
#pragma unroll
        for (int i = 0; i < LA; ++i)
        {
            const int row = i * (NTH / 8) + tid / 8, c = (tid & 7) ^ swizzle_a(row);
            const unsigned o = cut && c * 16 >= last ? oa[i] - (unsigned)(c * 16) : oa[i];
            load_to_lds(A + k, o, dst + (unsigned)(i * (NTH * 16)));
        }
#pragma unroll
        for (int i = 0; i < LB; ++i)
        {
            const int row = i * (NTH / 8) + tid / 8, c = (tid & 7) ^ swizzle_b<NN>(row);
            const unsigned o = cut && c * 16 >= last ? ob[i] - (unsigned)(c * 16) : ob[i];
            load_to_lds(B + k, o, dst + (unsigned)(TM * 128 + i * (NTH * 16)));
        }
    };

    // scales: a dword holds a row's next four k-steps
    const uint8_t *SA[MT], *SB[NN];
    unsigned sa[MT], sb[NN], na[MT], nbx[NN];
#pragma unroll
    for (int i = 0; i < MT; ++i) { SA[i] = p.SA + (m0 + (size_t)min(wm * (TM / WM) + 16 * i + l16, am)) * p.ldsa; }
#pragma unroll
    for (int j = 0; j < NN; ++j) { SB[j] = p.SB + (n0 + (size_t)min(wn * (TN / WN) + 4 * NN * (l16 >> 2) + 4 * j + (l16 & 3), bm)) * p.ldsb; }
    auto fetch_scales = [&](int kb)
    {
#pragma unroll
        for (int i = 0; i < MT; ++i) { na[i] = *reinterpret_cast<const unsigned *>(SA[i] + kb); }
#pragma unroll
        for (int j = 0; j < NN; ++j) { nbx[j] = *reinterpret_cast<const unsigned *>(SB[j] + kb); }
    };

    v4f acc[MT][NN];
#pragma unroll
    for (int i = 0; i < MT; ++i)
    {
#pragma unroll
        for (int j = 0; j < NN; ++j) { acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f}; }
    }

    if (nb > 0) { fetch_scales(0); fetch(0, 0); }
    for (int kb = 0; kb < nb; ++kb)
    {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     // a barrier alone does not wait for this wave's loads into LDS
        __syncthreads();                                                     // this stage is in LDS, the other one is free
        if ((kb & 3) == 0)
        {
#pragma unroll
            for (int i = 0; i < MT; ++i) { sa[i] = na[i]; }
#pragma unroll
            for (int j = 0; j < NN; ++j) { sb[j] = nbx[j]; }
        }
        uint8_t *st = lds + (kb & 1) * STAGE;
        if (kb == nb - 1 && last < 128)
        {
            for (int r = tid; r < TM + TN; r += NTH)
            {
                const int f = r < TM ? swizzle_a(r) : swizzle_b<NN>(r - TM);
                for (int c = last / 16; c < 8; ++c)
                {
                    uint4 *q = reinterpret_cast<uint4 *>(st + r * 128 + ((c ^ f) * 16));
                    *q = keep_bytes(*q, last - c * 16);
                }
            }
            __syncthreads();
        }
        if (kb + 1 < nb)
        {
            if ((kb & 3) == 3) { fetch_scales(kb + 1); }
            fetch(kb + 1, (kb + 1) & 1);
        }
        v8i fb[NN];
#pragma unroll
        for (int j = 0; j < NN; ++j)
        {
            const int row = wn * (TN / WN) + 4 * NN * (l16 >> 2) + 4 * j + (l16 & 3);
            const uint8_t *q = st + TM * 128 + row * 128;
            const int c = g ^ swizzle_b<NN>(row);
            const int4 x = *reinterpret_cast<const int4 *>(q + c * 16), y = *reinterpret_cast<const int4 *>(q + (c ^ 4) * 16);
            fb[j] = v8i{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
        {
            const int row = wm * (TM / WM) + 16 * i + l16;
            const uint8_t *q = st + row * 128;
            const int c = g ^ swizzle_a(row);
            const int4 x = *reinterpret_cast<const int4 *>(q + c * 16), y = *reinterpret_cast<const int4 *>(q + (c ^ 4) * 16);
            const v8i fa = v8i{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < NN; ++j) { acc[i][j] = mfma_scaled(fb[j], fa, acc[i][j], (int)sb[j], (int)sa[i]); }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) { sa[i] >>= 8; }
#pragma unroll
        for (int j = 0; j < NN; ++j) { sb[j] >>= 8; }
    }

    const size_t n = n0 + (size_t)(wn * (TN / WN) + 4 * NN * g);
    const int left = n < p.N ? (int)min(p.N - n, (size_t)(4 * NN)) : 0;
    float bias[4 * NN];
#pragma unroll
    for (int q = 0; q < 4 * NN; ++q) { bias[q] = p.bias && q < left ? p.bias[n + q] : 0.0f; }
#pragma unroll
    for (int i = 0; i < MT; ++i)
    {
        const size_t m = m0 + (size_t)(wm * (TM / WM) + 16 * i + l16);
        if (m >= p.M) { continue; }
        T *y = reinterpret_cast<T *>(p.Y) + m * p.ldy + n;
#pragma unroll
        for (int h = 0; h < 4 * NN; h += 8)
        {
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) { v[q] = acc[i][(h + q) / 4][q % 4] + bias[h + q]; }
            store_vals(y + h, left - h, v);
        }
    }
}

// ---- the largest products: two groups of waves in turn ----
// 256 x 256 values, 8 waves of 128 x 64.  A SIMD holds one wave of each group; time runs in phases between barriers, and in each phase one
// group reads its operands of a k-step from LDS into registers while the other one's 32 matrix instructions run, so that neither the
// matrix unit nor LDS waits for the other:
//
//   phase 2 s      group 0 reads step s          group 1 computes step s - 1      all ask for stage s + 1
//   phase 2 s + 1  group 0 computes step s       group 1 reads step s             at its end stage s + 1 is there
//
// Stage s + 1 takes the buffer of stage s - 1, which group 1 read in phase 2 s - 1.  Scales go through LDS as well, four k-steps (a dword
// a row) at a time.
//
// 128 sums, 96 registers of operands and 12 of scales leave 20 for everything else: a wave's LDS addresses differ by constants only, and
// the last tiles of rows and columns are moved back to end with the matrix, so that no tile has an edge (what two tiles share they compute
// alike).  M and N are at least 256.
template <typename T>
__global__ __launch_bounds__(512) void product_turn_kernel(const ProductParams p, unsigned tiles_m, unsigned tiles_n)
{
    constexpr int TM = 256, TN = 256, MT = 8, NN = 4, STAGE = (TM + TN) * 128, SCALES = 2 * STAGE;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, l16 = tid & 15, g = (tid >> 4) & 3;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave >> 2, wn = wave & 3;

    const unsigned total = tiles_m * tiles_n, per = (total + 7) / 8;
    const unsigned tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (tile >= total) { return; }
    const unsigned band = tile / (8 * tiles_n), in = tile - band * 8 * tiles_n, bh = min(8u, tiles_m - band * 8);
    const size_t m0 = min((size_t)(band * 8 + in % bh) * TM, p.M - TM), n0 = min((size_t)(in / bh) * TN, p.N - TN);

    const int nb = (int)((p.K + 127) / 128), last = (int)(p.K - (size_t)(nb - 1) * 128);
    const uint8_t *A = p.A + m0 * p.lda, *B = p.B + n0 * p.ldb;
    // a load brings 64 rows, 8 a wave: thread t takes the chunk of row t / 8 that belongs at place t % 8
    const int lr = tid >> 3, ca = (tid & 7) ^ swizzle_a(lr), cb = (tid & 7) ^ swizzle_b<NN>(lr);
    const unsigned oa = (unsigned)lr * (unsigned)p.lda + (unsigned)(ca * 16), ob = (unsigned)lr * (unsigned)p.ldb + (unsigned)(cb * 16);
    const uint8_t *S = tid < TM ? p.SA + (m0 + tid) * p.ldsa : p.SB + (n0 + tid - TM) * p.ldsb;
    const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane(base) + (unsigned)wave * 1024u, sc0 = __builtin_amdgcn_readfirstlane(base) + SCALES + (unsigned)wave * 256u;

    // chunks that start at or behind K are fetched from the row's first bytes (clear() zeroes them)
    auto fetch = [&](int kb)
    {
        if (kb >= nb) { return; }
        unsigned fa = oa, fb = ob;
        if (kb == nb - 1 && last < 128)
        {
            if (ca * 16 >= last) { fa -= (unsigned)(ca * 16); }
            if (cb * 16 >= last) { fb -= (unsigned)(cb * 16); }
        }
        const uint8_t *a = A + (size_t)kb * 128, *b = B + (size_t)kb * 128;
        const unsigned dst = lds0 + (unsigned)((kb & 1) * STAGE);
#pragma unroll
        for (int i = 0; i < 4; ++i) { load_to_lds(a + (size_t)i * 64 * p.lda, fa, dst + (unsigned)(i * 8192)); }
#pragma unroll
        for (int i = 0; i < 4; ++i) { load_to_lds(b + (size_t)i * 64 * p.ldb, fb, dst + (unsigned)(TM * 128 + i * 8192)); }
        if ((kb & 3) == 0) { load_dword_to_lds(S + kb, sc0 + (unsigned)((kb >> 2 & 1) * 2048)); }
    };
    auto barrier = []()
    {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" : : : "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    // group 0, at the start of the phase in which it reads the last stage
    auto clear = [&]()
    {
        uint8_t *st = lds + ((nb - 1) & 1) * STAGE;
        for (int r = tid; r < TM + TN; r += 256)
        {
            const int f = r < TM ? swizzle_a(r) : swizzle_b<NN>(r - TM);
            for (int c = last / 16; c < 8; ++c)
            {
                uint4 *q = reinterpret_cast<uint4 *>(st + r * 128 + ((c ^ f) * 16));
                *q = keep_bytes(*q, last - c * 16);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    };

    v4f acc[MT][NN];
    v8i fa[MT], fb[NN];
    int sa[MT], sb[NN];
#pragma unroll
    for (int i = 0; i < MT; ++i)
    {
#pragma unroll
        for (int j = 0; j < NN; ++j) { acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f}; }
    }
    // row 16 i + l16 of A: chunk g ^ (row & 7); row 16 (l16 / 4) + 4 j + l16 % 4 of B: chunk g ^ (l16 % 4 + 4 (l16 / 4 % 2)) = g ^ (l16 & 7)
    const int place = (g ^ (l16 & 7)) * 16, brow = wn * 64 + 16 * (l16 >> 2) + (l16 & 3), arow = group * 128 + l16;
    const int qa = arow * 128 + place, qb = TM * 128 + brow * 128 + place, qsa = SCALES + arow * 4, qsb = SCALES + (TM + brow) * 4;
    auto read = [&](int kb)
    {
        const uint8_t *st = lds + (kb & 1) * STAGE, *sc = lds + ((kb >> 2 & 1) * 2048 + (kb & 3));
        const uint8_t *a0 = st + qa, *a1 = st + (qa ^ 64), *b0 = st + qb, *b1 = st + (qb ^ 64);
#pragma unroll
        for (int j = 0; j < NN; ++j)
        {
            const int4 x = *reinterpret_cast<const int4 *>(b0 + j * 512), y = *reinterpret_cast<const int4 *>(b1 + j * 512);
            fb[j] = v8i{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            sb[j] = sc[qsb + j * 16];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
        {
            const int4 x = *reinterpret_cast<const int4 *>(a0 + i * 2048), y = *reinterpret_cast<const int4 *>(a1 + i * 2048);
            fa[i] = v8i{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            sa[i] = sc[qsa + i * 64];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    };
    auto compute = [&]()
    {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MT; ++i)
        {
#pragma unroll
            for (int j = 0; j < NN; ++j) { acc[i][j] = mfma_scaled(fb[j], fa[i], acc[i][j], sb[j], sa[i]); }
        }
        __builtin_amdgcn_s_setprio(0);
    };

    fetch(0);
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    barrier();
    if (group == 0)
    {
        for (int kb = 0; kb < nb; ++kb)
        {
            if (kb == nb - 1 && last < 128) { clear(); barrier(); }
            fetch(kb + 1);
            read(kb);
            barrier();
            compute();
            asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
            barrier();
        }
    }
    else
    {
        for (int kb = -1; kb < nb; ++kb)
        {
            if (kb >= 0)
            {
                read(kb);
                asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
                barrier();
            }
            if (kb == nb - 2 && last < 128) { barrier(); }
            fetch(kb + 2);
            if (kb >= 0) { compute(); }
            if (kb < nb - 1) { barrier(); }
        }
    }

    const size_t n = n0 + (size_t)(wn * 64 + 16 * g);
    float bias[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) { bias[q] = p.bias ? p.bias[n + q] : 0.0f; }
    T *y = reinterpret_cast<T *>(p.Y) + (m0 + (size_t)arow) * p.ldy + n;
#pragma unroll
    for (int i = 0; i < MT; ++i)
    {
#pragma unroll
        for (int h = 0; h < 16; h += 8)
        {
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) { v[q] = acc[i][(h + q) / 4][q % 4] + bias[h + q]; }
            store_vals(y + (size_t)(16 * i) * p.ldy + h, 8, v);
        }
    }
}

template <typename T>
hipError_t turn_go(const ProductParams &p, hipStream_t s)
{
    constexpr int LDS = 2 * 512 * 128 + 2 * 2048;
    const hipError_t e = opt_in_lds_once(reinterpret_cast<const void *>(&product_turn_kernel<T>), LDS);
    if (e != hipSuccess) { return e; }
    const unsigned tm = (unsigned)((p.M + 255) / 256), tn = (unsigned)((p.N + 255) / 256);
    hipLaunchKernelGGL(product_turn_kernel<T>, dim3((tm * tn + 7) / 8 * 8), dim3(512), LDS, s, p, tm, tn);
    return hipSuccess;
}

template <typename T, int TM, int TN, int WM, int WN>
hipError_t tile_go(const ProductParams &p, hipStream_t s)
{
    constexpr int LDS = 2 * (TM + TN) * 128;
    const void *k = reinterpret_cast<const void *>(&product_tile_kernel<T, TM, TN, WM, WN>);
    const hipError_t e = opt_in_lds_once(k, LDS);
    if (e != hipSuccess) { return e; }
    const unsigned tm = (unsigned)((p.M + TM - 1) / TM), tn = (unsigned)((p.N + TN - 1) / TN);
    hipLaunchKernelGGL((product_tile_kernel<T, TM, TN, WM, WN>), dim3((tm * tn + 7) / 8 * 8), dim3(64 * WM * WN), LDS, s, p, tm, tn);
    return hipSuccess;
}

template <typename T>
hipError_t product_go(const ProductParams &p, hipStream_t s)
{
    // rows of a tile are addressed in 32 bits from its first
    const bool near = p.lda < ((size_t)1 << 23) && p.ldb < ((size_t)1 << 23);
    if (near && p.M >= 256 && p.N >= 256 && p.K > 0 && ((p.M + 255) / 256) * ((p.N + 255) / 256) >= 128) { return turn_go<T>(p, s); }
    if (near && ((p.M + 127) / 128) * ((p.N + 127) / 128) >= 64) { return tile_go<T, 128, 128, 2, 2>(p, s); }
    const size_t tm = (p.M + 31) / 32, tn = (p.N + 31) / 32;
    hipLaunchKernelGGL((product_split_kernel<T, 2, 2, 4>), dim3((unsigned)(tm * tn)), dim3(256), 0, s, p, (unsigned)tn);
    return hipSuccess;
}

}  // namespace

hipError_t launch_rows_product(int dtype, const ProductParams &p, hipStream_t s)
{
    hipError_t e = hipErrorInvalidValue;
    switch (dtype)
    {
        case SPEECH_BF16: e = product_go<__bf16>(p, s); break;
        case SPEECH_F16: e = product_go<_Float16>(p, s); break;
        default: break;
    }
    return e != hipSuccess ? e : hipGetLastError();
}

}  // namespace speech
