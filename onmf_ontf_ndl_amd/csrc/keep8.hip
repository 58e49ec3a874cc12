// Columns held in 8 bits and what the dictionary's update needs of them, on gfx950.
//
// Format: 128 consecutive columns of a row share a scale s = max |v| / 127 (float32); an entry stands for s q,
// q = rint(v / s) in -127..127.  codes is [row][padded columns] int8 (rows padded to whole groups with zeros),
// scales [row][group].  A minibatch X and its code H put away this way take a quarter of their room, and the
// sums H H^T and H X^T - the gradient to the dictionary is W (H H^T) - X H^T - run on the 8-bit matrix pipe:
// inside a group the products of whole numbers add up exactly in int32.
#include "common.h"

#include <algorithm>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

namespace {

constexpr int GROUP = 128;

__device__ __forceinline__ float bf16_to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float load_val(const float* p) { return *p; }
__device__ __forceinline__ float load_val(const uint16_t* p) { return bf16_to_f32(*p); }

// ------------------------------------------------------------------------------------------- put away
// Whole q nearest to v / s with ties to even, decided exactly: the remainder v - s q is a multiple of half an
// ulp of s and below 2^24 of them, so the fused multiply-add gives it without rounding and a quotient next to
// a half falls on its own side whatever the reciprocal's rounding.
__device__ __forceinline__ int nearest(float v, float s, float inv) {
    float q = rintf(v * inv);
    const float rest = 2.f * fmaf(-q, s, v);
    const bool odd = ((int)q & 1) != 0;
    if (rest > s || (rest == s && odd)) q += 1.f;
    else if (rest < -s || (rest == -s && odd)) q -= 1.f;
    return (int)q;
}

// 32 lanes per group, four columns a lane.
template <typename T>
__global__ __launch_bounds__(256) void keep8_kernel(int d, int n, int groups, const T* __restrict__ X, int ldx, int vec,
                                                     int8_t* __restrict__ codes, float* __restrict__ scales) {
    const size_t all = (size_t)d * groups;
    for (size_t at = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); at < all; at += (size_t)gridDim.x * 8) {
        const int row = (int)(at / groups), g = (int)(at % groups);
        const int c = g * GROUP + (threadIdx.x & 31) * 4;
        const T* src = X + (size_t)row * ldx + c;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (vec && c + 3 < n) {
            if constexpr (sizeof(T) == 4) {
                const float4 f = *reinterpret_cast<const float4*>(src);
                v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(src);
                v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
                v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < n) v[j] = load_val(src + j);
        }
        // the largest magnitude by its bits: a NaN's are above an infinity's, an infinity's above all others
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
        float s = __uint_as_float(most) / 127.f;
        int q[4] = {0, 0, 0, 0};
        if (most >= 0x7f800000u) {
            s = __uint_as_float(0x7fc00000u);            // a NaN or an infinity: the whole group reads NaN
        } else if (s < 1.17549435e-38f) {
            s = 0.f;                                       // nothing but (next to) zeros
        } else {
            const float inv = 1.f / s;
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = nearest(v[j], s, inv);
        }
        *reinterpret_cast<uint32_t*>(codes + (size_t)row * groups * GROUP + c) =
            (uint32_t)(q[0] & 0xff) | (uint32_t)(q[1] & 0xff) << 8 | (uint32_t)(q[2] & 0xff) << 16 | (uint32_t)(q[3] & 0xff) << 24;
        if ((threadIdx.x & 31) == 0) scales[at] = s;
    }
}

// ------------------------------------------------------------------------------------------- bring back
__global__ __launch_bounds__(256) void keep8_expand_kernel(int d, int n, int groups, const int8_t* __restrict__ codes,
                                                            const float* __restrict__ scales, float* __restrict__ X,
                                                            int ldx, int vec) {
    const size_t all = (size_t)d * groups;
    for (size_t at = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); at < all; at += (size_t)gridDim.x * 8) {
        const int row = (int)(at / groups), g = (int)(at % groups);
        const int c = g * GROUP + (threadIdx.x & 31) * 4;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + (size_t)row * groups * GROUP + c);
        const float s = scales[at];
        const float4 v = make_float4(s * (float)(int8_t)(w & 0xff), s * (float)(int8_t)((w >> 8) & 0xff),
                                     s * (float)(int8_t)((w >> 16) & 0xff), s * (float)(int8_t)(w >> 24));
        float* dst = X + (size_t)row * ldx + c;
        if (vec && c + 3 < n) {
            *reinterpret_cast<float4*>(dst) = v;
        } else {
            if (c + 0 < n) dst[0] = v.x;
            if (c + 1 < n) dst[1] = v.y;
            if (c + 2 < n) dst[2] = v.z;
            if (c + 3 < n) dst[3] = v.w;
        }
    }
}

// X[:, j] = column idx[j]; a negative index counts from the end, one out of range reads NaN.
__global__ __launch_bounds__(256) void keep8_gather_kernel(int d, int n, int groups, const int8_t* __restrict__ codes,
                                                            const float* __restrict__ scales,
                                                            const long long* __restrict__ idx, int b,
                                                            float* __restrict__ X, int ldx) {
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (j >= b) return;
    long long c = idx[j];
    if (c < 0) c += n;
    const bool fine = c >= 0 && c < n;
    for (int row = blockIdx.y; row < d; row += gridDim.y) {
        float v = __uint_as_float(0x7fc00000u);
        if (fine) v = scales[(size_t)row * groups + c / GROUP] * (float)codes[(size_t)row * groups * GROUP + c];
        X[(size_t)row * ldx + j] = v;
    }
}

// ------------------------------------------------------------------------------------------- sums
// 128 x 128 tiles of [H H^T | H X^T] (the columns of the second part start on a tile), one 128-column group
// of the contraction a step; a workgroup takes a run of groups and writes its sums to a slab.  int32 inside a
// group, float32 over a workgroup's run, double over the runs.
constexpr int BM = 128, BN = 128, LROW = GROUP + 16;       // LDS row stride in bytes: 16-byte reads of 16 rows meet every bank once

struct SumParams {
    const int8_t *hc, *xc;
    const float *hs, *xs;
    float* slab;              // [split][r][cols]
    int d, r, groups, per_split;
    int tiles_m, tiles_h;     // tiles along r (rows), tiles of the H H^T part along the columns
    int cols;                 // columns of a slab row: tiles_h * BN + d
};

__global__ __launch_bounds__(256) void keep8_sums_kernel(SumParams p) {
    __shared__ __align__(16) int8_t la[2][BM * LROW], lb[2][BN * LROW];
    __shared__ float sa[2][BM], sb[2][BN];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int tm = blockIdx.x % p.tiles_m, tn = blockIdx.x / p.tiles_m;
    const int m0 = tm * BM;
    const bool is_h = tn < p.tiles_h;
    const int n0 = is_h ? tn * BN : (tn - p.tiles_h) * BN;
    const int N = is_h ? p.r : p.d;
    const int8_t* bc = is_h ? p.hc : p.xc;
    const float* bs = is_h ? p.hs : p.xs;
    const size_t ld = (size_t)p.groups * GROUP;
    const int g0 = blockIdx.y * p.per_split, g1 = min(p.groups, g0 + p.per_split);
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;

    uint4 ra[4], rb[4];
    float fs = 0.f;
    auto fetch = [&](int g) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = (t >> 3) + 32 * j, col = (t & 7) * 16;
            ra[j] = rb[j] = make_uint4(0, 0, 0, 0);
            if (m0 + row < p.r) ra[j] = *reinterpret_cast<const uint4*>(p.hc + (size_t)(m0 + row) * ld + (size_t)g * GROUP + col);
            if (n0 + row < N) rb[j] = *reinterpret_cast<const uint4*>(bc + (size_t)(n0 + row) * ld + (size_t)g * GROUP + col);
        }
        const int row = t & 127;
        fs = 0.f;
        if (t < 128) { if (m0 + row < p.r) fs = p.hs[(size_t)(m0 + row) * p.groups + g]; }
        else if (n0 + row < N) fs = bs[(size_t)(n0 + row) * p.groups + g];
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = (t >> 3) + 32 * j, col = (t & 7) * 16;
            *reinterpret_cast<uint4*>(&la[buf][row * LROW + col]) = ra[j];
            *reinterpret_cast<uint4*>(&lb[buf][row * LROW + col]) = rb[j];
        }
        if (t < 128) sa[buf][t] = fs; else sb[buf][t - 128] = fs;
    };

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    fetch(g0);
    stage(0);
    for (int g = g0; g < g1; ++g) {
        const int buf = (g - g0) & 1;
        __syncthreads();
        if (g + 1 < g1) fetch(g + 1);
        i32x16 part[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) part[i][j][e] = 0;
        const int at = (lane & 31) * LROW + (lane >> 5) * 16;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            i32x4 fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = *reinterpret_cast<const i32x4*>(&la[buf][(wm + i * 32) * LROW + at + h * 32]);
                fb[i] = *reinterpret_cast<const i32x4*>(&lb[buf][(wn + i * 32) * LROW + at + h * 32]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    part[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], part[i][j], 0, 0, 0);
        }
        float cs[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) cs[j] = sb[buf][wn + j * 32 + (lane & 31)];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float rs = sa[buf][wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)];
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j][e] = fmaf(rs, cs[j] * (float)part[i][j][e], acc[i][j][e]);
            }
        if (g + 1 < g1) stage(buf ^ 1);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int n = n0 + wn + j * 32 + (lane & 31);
        if (n >= N) continue;
        const int col = is_h ? n : p.tiles_h * BN + n;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                if (m < p.r) p.slab[((size_t)blockIdx.y * p.r + m) * p.cols + col] = acc[i][j][e];
            }
    }
}

// A = keep A_in + w sum, B = keep B_in + w sum over the slabs, in order and in double.  With Ad, Bd (the gradient)
// the sums themselves are written there as doubles.
__global__ __launch_bounds__(256) void keep8_reduce_kernel(int d, int r, int colh, int cols, int splits,
                                                            const float* __restrict__ slab, double w, double keep,
                                                            const float* A_in, const float* B_in, float* A, float* B,
                                                            double* __restrict__ Ad, double* __restrict__ Bd) {
    const size_t one = (size_t)r * cols, all = (size_t)r * (r + d);
    for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (size_t)gridDim.x * 256) {
        const int k = (int)(e / (r + d)), j = (int)(e % (r + d));
        const float* src = slab + (size_t)k * cols + (j < r ? j : colh + (j - r));
        double s = 0.0;
        for (int z = 0; z < splits; ++z) s += (double)src[(size_t)z * one];
        if (Ad) {
            if (j < r) Ad[(size_t)k * r + j] = s;
            else Bd[(size_t)k * d + (j - r)] = s;
        } else if (j < r) {
            const size_t at = (size_t)k * r + j;
            A[at] = (float)(w * s + (A_in ? keep * (double)A_in[at] : 0.0));
        } else {
            const size_t at = (size_t)k * d + (j - r);
            B[at] = (float)(w * s + (B_in ? keep * (double)B_in[at] : 0.0));
        }
    }
}

// dW[i][k] = sum_j W[i][j] A[j][k] - B[k][i] in double, rounded once: near a stationary dictionary the two
// terms nearly cancel.
__global__ __launch_bounds__(256) void keep8_gradient_kernel(int d, int r, const float* __restrict__ W,
                                                              const double* __restrict__ A,
                                                              const double* __restrict__ B, float* __restrict__ dW) {
    __shared__ double tw[32][17], ta[16][33], tb[32][33];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int i0 = blockIdx.y * 32, k0 = blockIdx.x * 32;
    double acc[2][2] = {{0.0, 0.0}, {0.0, 0.0}};
    for (int j0 = 0; j0 < r; j0 += 16) {
        for (int e = threadIdx.x; e < 512; e += 256) {
            const int i = e >> 4, j = e & 15;
            tw[i][j] = (i0 + i < d && j0 + j < r) ? (double)W[(size_t)(i0 + i) * r + j0 + j] : 0.0;
            const int jj = e >> 5, k = e & 31;
            ta[jj][k] = (j0 + jj < r && k0 + k < r) ? A[(size_t)(j0 + jj) * r + k0 + k] : 0.0;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int c = 0; c < 2; ++c) acc[a][c] = fma(tw[ty + 16 * a][j], ta[j][tx + 16 * c], acc[a][c]);
        __syncthreads();
    }
    for (int e = threadIdx.x; e < 1024; e += 256) {
        const int k = e >> 5, i = e & 31;
        tb[i][k] = (k0 + k < r && i0 + i < d) ? B[(size_t)(k0 + k) * d + i0 + i] : 0.0;
    }
    __syncthreads();
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int i = i0 + ty + 16 * a, k = k0 + tx + 16 * c;
            if (i < d && k < r) dW[(size_t)i * r + k] = (float)(acc[a][c] - tb[ty + 16 * a][tx + 16 * c]);
        }
}

// ------------------------------------------------------------------------------------------- launches
struct SumPlan { int tiles_m, tiles_h, tiles_x, cols, splits, per; };
SumPlan sum_plan(int d, int r, int n) {
    SumPlan q;
    const int groups = (n + GROUP - 1) / GROUP;
    q.tiles_m = (r + BM - 1) / BM;
    q.tiles_h = (r + BN - 1) / BN;
    q.tiles_x = (d + BN - 1) / BN;
    q.cols = q.tiles_h * BN + d;
    const long long tiles = (long long)q.tiles_m * (q.tiles_h + q.tiles_x);
    long long splits = std::max<long long>(1, 512 / tiles);
    splits = std::min<long long>(splits, groups);
    q.per = (int)((groups + splits - 1) / splits);
    q.splits = (groups + q.per - 1) / q.per;
    return q;
}
size_t sums_bytes(const SumPlan& q, int r) { return ((size_t)q.splits * r * q.cols * sizeof(float) + 255) & ~(size_t)255; }

int check8(onmf_ctx* c, const char* what, int d, int n, const void* codes, const void* scales) {
    if (d <= 0 || n <= 0 || !codes || !scales || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3))
        return onmf_fail(c, ONMF_ERR_ARG, "%s: bad arguments (d=%d n=%d; codes must be aligned to 16 bytes)", what, d, n);
    if (n > 2147483647 - 2 * GROUP) return onmf_fail(c, ONMF_ERR_ARG, "%s: n=%d is too large", what, n);
    return ONMF_OK;
}

int run_sums(onmf_ctx* c, const SumPlan& q, int d, int r, int n, const int8_t* xc, const float* xs, const int8_t* hc,
             const float* hs, float* slab, hipStream_t s) {
    SumParams p;
    p.hc = hc; p.xc = xc; p.hs = hs; p.xs = xs; p.slab = slab;
    p.d = d; p.r = r; p.groups = (n + GROUP - 1) / GROUP; p.per_split = q.per;
    p.tiles_m = q.tiles_m; p.tiles_h = q.tiles_h; p.cols = q.cols;
    hipLaunchKernelGGL(keep8_sums_kernel, dim3(q.tiles_m * (q.tiles_h + q.tiles_x), q.splits), dim3(256), 0, s, p);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

unsigned reduce_blocks(int d, int r) { return (unsigned)std::min<size_t>(((size_t)r * (r + d) + 255) / 256, 8192); }
unsigned group_blocks(int d, int n) {
    return (unsigned)std::min<size_t>(((size_t)d * ((n + GROUP - 1) / GROUP) + 7) / 8, 8192);
}

}  // namespace

extern "C" {

int onmf_keep8(onmf_ctx* c, int d, int n, const void* X, int x_type, int ldx, int8_t* codes, float* scales, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check8(c, "keep8", d, n, codes, scales));
    if (!X || ldx < n || (x_type != ONMF_TYPE_F32 && x_type != ONMF_TYPE_BF16))
        return onmf_fail(c, ONMF_ERR_ARG, "keep8: bad arguments (ldx=%d type=%d)", ldx, x_type);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const int groups = (n + GROUP - 1) / GROUP;
    const size_t es = x_type == ONMF_TYPE_F32 ? 4 : 2;
    const int vec = ((uintptr_t)X & (4 * es - 1)) == 0 && (ldx & 3) == 0;
    if (x_type == ONMF_TYPE_F32)
        hipLaunchKernelGGL(keep8_kernel<float>, dim3(group_blocks(d, n)), dim3(256), 0, s, d, n, groups, (const float*)X, ldx,
                           vec, codes, scales);
    else
        hipLaunchKernelGGL(keep8_kernel<uint16_t>, dim3(group_blocks(d, n)), dim3(256), 0, s, d, n, groups,
                           (const uint16_t*)X, ldx, vec, codes, scales);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

int onmf_keep8_expand(onmf_ctx* c, int d, int n, const int8_t* codes, const float* scales, const int64_t* idx, int b,
                      float* X, int ldx, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check8(c, "keep8_expand", d, n, codes, scales));
    const int cols = idx ? b : n;
    if (!X || cols <= 0 || ldx < cols) return onmf_fail(c, ONMF_ERR_ARG, "keep8_expand: bad arguments (b=%d ldx=%d)", b, ldx);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const int groups = (n + GROUP - 1) / GROUP;
    if (idx)
        hipLaunchKernelGGL(keep8_gather_kernel, dim3((b + 255) / 256, std::min(d, 4096)), dim3(256), 0, s, d, n, groups, codes,
                           scales, (const long long*)idx, b, X, ldx);
    else
        hipLaunchKernelGGL(keep8_expand_kernel, dim3(group_blocks(d, n)), dim3(256), 0, s, d, n, groups, codes, scales, X, ldx,
                           (int)(((uintptr_t)X & 15) == 0 && (ldx & 3) == 0));
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

size_t onmf_keep8_workspace(int d, int r, int n, int gradient) {
    if (d <= 0 || r <= 0 || n <= 0 || n > 2147483647 - 2 * GROUP) return 0;
    return sums_bytes(sum_plan(d, r, n), r) + (gradient ? sizeof(double) * (size_t)r * ((size_t)r + d) : 0);
}

int onmf_keep8_aggregate(onmf_ctx* c, int d, int r, int n, const int8_t* x_codes, const float* x_scales,
                         const int8_t* h_codes, const float* h_scales, double w, const float* A_in, const float* B_in,
                         float* A_out, float* B_out, void* ws, size_t ws_bytes, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check8(c, "keep8_aggregate", d, n, x_codes, x_scales));
    ONMF_TRY(check8(c, "keep8_aggregate", r, n, h_codes, h_scales));
    if (!A_out || !B_out) return onmf_fail(c, ONMF_ERR_ARG, "keep8_aggregate: an output is null");
    const size_t need = onmf_keep8_workspace(d, r, n, 0);
    if (!ws || ws_bytes < need)
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_aggregate: workspace of %zu bytes, %zu needed", ws_bytes, need);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const SumPlan q = sum_plan(d, r, n);
    ONMF_TRY(run_sums(c, q, d, r, n, x_codes, x_scales, h_codes, h_scales, (float*)ws, s));
    hipLaunchKernelGGL(keep8_reduce_kernel, dim3(reduce_blocks(d, r)), dim3(256), 0, s, d, r, q.tiles_h * BN, q.cols, q.splits,
                       (const float*)ws, w, 1.0 - w, A_in, B_in, A_out, B_out, (double*)nullptr, (double*)nullptr);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

int onmf_keep8_gradient(onmf_ctx* c, int d, int r, int n, const float* W, const int8_t* x_codes, const float* x_scales,
                        const int8_t* h_codes, const float* h_scales, float* dW, void* ws, size_t ws_bytes,
                        void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check8(c, "keep8_gradient", d, n, x_codes, x_scales));
    ONMF_TRY(check8(c, "keep8_gradient", r, n, h_codes, h_scales));
    if (!W || !dW) return onmf_fail(c, ONMF_ERR_ARG, "keep8_gradient: W or dW is null");
    if (d > (1 << 18) || r > (1 << 18))
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_gradient: d=%d or r=%d is more than 2^18", d, r);
    const size_t need = onmf_keep8_workspace(d, r, n, 1);
    if (!ws || ws_bytes < need)
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_gradient: workspace of %zu bytes, %zu needed", ws_bytes, need);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const SumPlan q = sum_plan(d, r, n);
    double* Ad = (double*)((char*)ws + sums_bytes(q, r));
    double* Bd = Ad + (size_t)r * r;
    ONMF_TRY(run_sums(c, q, d, r, n, x_codes, x_scales, h_codes, h_scales, (float*)ws, s));
    hipLaunchKernelGGL(keep8_reduce_kernel, dim3(reduce_blocks(d, r)), dim3(256), 0, s, d, r, q.tiles_h * BN, q.cols, q.splits,
                       (const float*)ws, 1.0, 0.0, (const float*)nullptr, (const float*)nullptr, (float*)nullptr, (float*)nullptr,
                       Ad, Bd);
    HIP_TRY(c, hipGetLastError());
    hipLaunchKernelGGL(keep8_gradient_kernel, dim3((r + 31) / 32, (d + 31) / 32), dim3(256), 0, s, d, r, W, Ad, Bd, dW);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

}  // extern "C"
