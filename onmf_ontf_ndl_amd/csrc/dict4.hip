// A dictionary held in 4 bits and its two products on gfx950.
//
// Format: the entries of an atom (a column of W) are taken in groups of G = 32, 64 or 128 consecutive
// features that share a scale s (a bfloat16) and a whole number z; an entry stands for s (q + z), q in 0..15,
// |q + z| <= 255.  codes[k] holds atom k's features in words of eight: entry j of a word is nibble
// (j >> 1) + 4 (j & 1), so that (word >> 4 p) & 0x000f000f are entries 2p and 2p + 1.  Rows are padded to whole
// groups (zero nibbles).  scales[k][g] = bits of s (upper half of a float32) | (z & 0xffff).
// z keeps zeros exact (the usual case for a non-negative dictionary: z = 0) and lets a smooth atom, whose
// entries lie far from zero, spend its 16 levels on its own range.
#include "common.h"

#include <algorithm>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr int T_F32 = ONMF_TYPE_F32;

__device__ __forceinline__ float bf16_to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float load_val(const float* p) { return *p; }
__device__ __forceinline__ float load_val(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float word_scale(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float word_offset(uint32_t w) { return (float)(int16_t)(w & 0xffffu); }

// round to nearest even, two at a time: lower half = a
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ __forceinline__ float bf16_lo(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// the eight whole numbers q of a word
__device__ __forceinline__ void word_entries(uint32_t w, float (&q)[8]) {
    const uint32_t e = w & 0x0f0f0f0fu, o = (w >> 4) & 0x0f0f0f0fu;     // bytes of e: entries 0 4 1 5, of o: 2 6 3 7
    q[0] = (float)(e & 0xff);
    q[4] = (float)((e >> 8) & 0xff);
    q[1] = (float)((e >> 16) & 0xff);
    q[5] = (float)(e >> 24);
    q[2] = (float)(o & 0xff);
    q[6] = (float)((o >> 8) & 0xff);
    q[3] = (float)((o >> 16) & 0xff);
    q[7] = (float)(o >> 24);
}

// ------------------------------------------------------------------------------------------- packing
// smallest bfloat16 >= v (v >= 0, finite), as float
__device__ __forceinline__ float bf16_up(double v) {
    float f = (float)v;
    uint32_t u = __float_as_uint(f);
    if ((double)f < v) ++u;
    if (u & 0xffffu) u = (u & 0xffff0000u) + 0x10000u;
    return __uint_as_float(u);
}

// One thread per group: neighbouring threads take neighbouring atoms, so that reads of W (row-major) coalesce.
// The scale spans the group's range in 15 steps (14 where rounding both ends to the grid would need a 16th) and
// is rounded UP to bfloat16, so no entry is clipped and the error is at most s / 2.  Quotients in double: an
// entry next to a rounding border falls on its own side.
__global__ __launch_bounds__(256) void dict4_pack_kernel(int d, int r, int group, int groups,
                                                          const float* __restrict__ W, uint32_t* __restrict__ codes,
                                                          uint32_t* __restrict__ scales) {
    const int k = blockIdx.x * 256 + threadIdx.x, g = blockIdx.y;
    if (k >= r) return;
    const int i0 = g * group, n = min(group, d - i0);
    float lo = __int_as_float(0x7f800000), hi = -lo;
    bool fine = true;
    for (int i = 0; i < n; ++i) {
        const float v = W[(size_t)(i0 + i) * r + k];
        fine = fine && (fabsf(v) < __int_as_float(0x7f800000));
        lo = fminf(lo, v);
        hi = fmaxf(hi, v);
    }
    uint32_t* out = codes + ((size_t)k * groups + g) * (group / 8);
    if (!fine) {                       // a NaN or an infinity: the whole group reads NaN
        scales[(size_t)k * groups + g] = 0x7fc00000u;
        for (int w = 0; w < group / 8; ++w) out[w] = 0;
        return;
    }
    const double range = (double)hi - (double)lo;
    const double floor_ = fmax(fabs((double)lo), fabs((double)hi)) / 255.0;
    float s = bf16_up(fmax(range / 15.0, floor_));
    if (rint((double)hi / (double)s) - rint((double)lo / (double)s) > 15.0) s = bf16_up(fmax(range / 14.0, floor_));
    if (!(s >= 1.17549435e-38f)) {     // nothing but (next to) zeros
        scales[(size_t)k * groups + g] = 0;
        for (int w = 0; w < group / 8; ++w) out[w] = 0;
        return;
    }
    const double sd = (double)s, z = rint((double)lo / sd);
    scales[(size_t)k * groups + g] = __float_as_uint(s) | ((uint32_t)(int)z & 0xffffu);
    for (int w = 0; w < group / 8; ++w) {
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = w * 8 + j;
            if (i < n) {
                const double q = rint((double)W[(size_t)(i0 + i) * r + k] / sd) - z;
                word |= (uint32_t)(int)q << (4 * ((j >> 1) + 4 * (j & 1)));
            }
        }
        out[w] = word;
    }
}

// One thread per word of eight features; neighbouring threads take neighbouring atoms (W's fast index).
__global__ __launch_bounds__(256) void dict4_unpack_kernel(int d, int r, int group, int groups,
                                                            const uint32_t* __restrict__ codes,
                                                            const uint32_t* __restrict__ scales, float* __restrict__ W) {
    const int k = blockIdx.x * 256 + threadIdx.x, w = blockIdx.y;
    if (k >= r) return;
    const uint32_t sc = scales[(size_t)k * groups + (w * 8) / group];
    const float s = word_scale(sc), z = word_offset(sc);
    float q[8];
    word_entries(codes[(size_t)k * groups * (group / 8) + w], q);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (w * 8 + j < d) W[(size_t)(w * 8 + j) * r + k] = s * (q[j] + z);
}

// ------------------------------------------------------------------------------------------- few columns
// C = W^T X for up to NB columns: bound by reading the codes once.  A lane owns F = 8 CH consecutive features
// of a segment of 64 F; X is staged in LDS as float and a segment's F x NB values are held in registers while AT
// atoms stream past.  One code costs an extraction (0.4), a conversion and NB fused multiply-adds.
// LDS: quad q (of F / 4) of lane l of segment g and column n at [((g * F/4 + q) * 64 + l) * 4] of plane n.
template <int NB, int CH, int AT, typename T>
__global__ __launch_bounds__(256) void dict4_correlate_few_kernel(int d, int r, int b, int group, int groups,
                                                                   const uint32_t* __restrict__ codes,
                                                                   const uint32_t* __restrict__ scales,
                                                                   const T* __restrict__ X, int ldx,
                                                                   float* __restrict__ C, int segs_staged) {
    constexpr int F = 8 * CH, SEG = 64 * F;
    extern __shared__ __align__(16) float xs[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int segs = (d + SEG - 1) / SEG;
    const int words = groups * (group / 8);
    const int plane = segs_staged * SEG;
    const int chunks = (r + 4 * AT - 1) / (4 * AT);
    bool first = true;
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int k0 = chunk * 4 * AT + wave * AT;
        float acc[AT][NB];
#pragma unroll
        for (int a = 0; a < AT; ++a)
#pragma unroll
            for (int n = 0; n < NB; ++n) acc[a][n] = 0.f;
        for (int s0 = 0; s0 < segs; s0 += segs_staged) {
            if (first || segs_staged < segs) {          // the whole of X fits: staged once
                __syncthreads();
                const int i0 = s0 * SEG, in = min(plane, segs * SEG - i0);
                for (int e = threadIdx.x; e < in * NB; e += 256) {
                    const int n = NB == 1 ? 0 : e % NB, i = NB == 1 ? e : e / NB;
                    float v = 0.f;
                    if (i0 + i < d && n < b) v = load_val(X + (size_t)(i0 + i) * ldx + n);
                    const int g = i / SEG, l = (i % SEG) / F, f = i % F;
                    xs[n * plane + ((g * (F / 4) + (f >> 2)) * 64 + l) * 4 + (f & 3)] = v;
                }
                __syncthreads();
                first = false;
            }
            const int sn = min(segs_staged, segs - s0);
            for (int g = 0; g < sn; ++g) {
                const int w0 = (s0 + g) * (SEG / 8) + lane * CH;       // this lane's first word
                if (w0 >= words) continue;                               // padding of the last segment
                float x[F][NB], sum[NB];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    sum[n] = 0.f;
#pragma unroll
                    for (int q = 0; q < F / 4; ++q) {
                        const float4 v = *reinterpret_cast<const float4*>(&xs[n * plane + ((g * (F / 4) + q) * 64 + lane) * 4]);
                        x[4 * q + 0][n] = v.x; x[4 * q + 1][n] = v.y; x[4 * q + 2][n] = v.z; x[4 * q + 3][n] = v.w;
                        sum[n] += (v.x + v.y) + (v.z + v.w);
                    }
                }
                uint32_t cw[AT][CH], sc[AT];
#pragma unroll
                for (int a = 0; a < AT; ++a) {
                    const int k = min(k0 + a, r - 1);
                    const uint32_t* src = codes + (size_t)k * words + w0;
                    if constexpr (CH == 4) {
                        const uint4 v = *reinterpret_cast<const uint4*>(src);
                        cw[a][0] = v.x; cw[a][1] = v.y; cw[a][2] = v.z; cw[a][3] = v.w;
                    } else if constexpr (CH == 2) {
                        const uint2 v = *reinterpret_cast<const uint2*>(src);
                        cw[a][0] = v.x; cw[a][1] = v.y;
                    } else {
                        cw[a][0] = *src;
                    }
                    sc[a] = scales[(size_t)k * groups + (w0 * 8) / group];
                }
#pragma unroll
                for (int a = 0; a < AT; ++a) {
                    float t[NB];
#pragma unroll
                    for (int n = 0; n < NB; ++n) t[n] = word_offset(sc[a]) * sum[n];
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        float q[8];
                        word_entries(cw[a][c], q);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int n = 0; n < NB; ++n) t[n] = fmaf(q[j], x[8 * c + j][n], t[n]);
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n) acc[a][n] = fmaf(word_scale(sc[a]), t[n], acc[a][n]);
                }
            }
        }
#pragma unroll
        for (int a = 0; a < AT; ++a)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float v = acc[a][n];
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
                if (lane == 0 && k0 + a < r && n < b) C[(size_t)(k0 + a) * b + n] = v;
            }
    }
}

// R = W H for up to NB columns: a lane owns F features of a segment and adds up its atoms' contributions
// h (s q + s z) in registers; the waves of a workgroup and the workgroups of a segment take different atoms and
// are added in a fixed order (LDS, then slabs).
template <int NB, int CH, typename T>
__global__ __launch_bounds__(256) void dict4_product_few_kernel(int d, int r, int b, int group, int groups,
                                                                 const uint32_t* __restrict__ codes,
                                                                 const uint32_t* __restrict__ scales,
                                                                 const T* __restrict__ H, int ldh, float* __restrict__ R,
                                                                 int ldr, int atoms_per_wg, float* __restrict__ slab) {
    constexpr int F = 8 * CH, SEG = 64 * F;
    __shared__ float part[3][NB][SEG];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int words = groups * (group / 8);
    const int w0 = blockIdx.x * (SEG / 8) + lane * CH;
    const bool there = w0 < words;
    const int ka = blockIdx.y * atoms_per_wg, kb = min(r, ka + atoms_per_wg);
    float acc[F][NB], zacc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        zacc[n] = 0.f;
#pragma unroll
        for (int f = 0; f < F; ++f) acc[f][n] = 0.f;
    }
    const int g = there ? (w0 * 8) / group : 0;
    if (there)
#pragma unroll 4
        for (int k = ka + wave; k < kb; k += 4) {
            uint32_t cw[CH];
            const uint32_t* src = codes + (size_t)k * words + w0;
            if constexpr (CH == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(src);
                cw[0] = v.x; cw[1] = v.y; cw[2] = v.z; cw[3] = v.w;
            } else if constexpr (CH == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(src);
                cw[0] = v.x; cw[1] = v.y;
            } else {
                cw[0] = *src;
            }
            const uint32_t sc = scales[(size_t)k * groups + g];
            float hs[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                hs[n] = word_scale(sc) * load_val(H + (size_t)k * ldh + min(n, b - 1));
                zacc[n] = fmaf(word_offset(sc), hs[n], zacc[n]);
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float q[8];
                word_entries(cw[c], q);
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int n = 0; n < NB; ++n) acc[8 * c + j][n] = fmaf(q[j], hs[n], acc[8 * c + j][n]);
            }
        }
    if (wave > 0)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int f = 0; f < F; ++f) part[wave - 1][n][f * 64 + lane] = acc[f][n] + zacc[n];
    __syncthreads();
    if (wave == 0 && there) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const float v = ((acc[f][n] + zacc[n]) + part[0][n][f * 64 + lane]) + (part[1][n][f * 64 + lane] + part[2][n][f * 64 + lane]);
                const int i = w0 * 8 + f;
                if (i < d && n < b) {
                    if (slab) slab[((size_t)blockIdx.y * b + n) * d + i] = v;
                    else R[(size_t)i * ldr + n] = v;
                }
            }
        }
    }
}

// R[i][n] = sum over the slabs z of slab[z][n][i], in order
__global__ __launch_bounds__(256) void dict4_product_few_reduce_kernel(int d, int b, int splits,
                                                                        const float* __restrict__ slab,
                                                                        float* __restrict__ R, int ldr) {
    __shared__ float part[4][64];
    const int o = threadIdx.x & 63, g = threadIdx.x >> 6;
    const size_t e = (size_t)blockIdx.x * 64 + o, all = (size_t)d * b;
    float s = 0.f;
    if (e < all)
        for (int z = g; z < splits; z += 4) s += slab[(size_t)z * all + e];
    part[g][o] = s;
    __syncthreads();
    if (g == 0 && e < all) {
        const int n = (int)(e / d), i = (int)(e % d);
        R[(size_t)i * ldr + n] = (part[0][o] + part[1][o]) + (part[2][o] + part[3][o]);
    }
}

// ------------------------------------------------------------------------------------------- many columns
// 128 x 128 output tiles on the bfloat16 matrix pipe (32x32x16), exact to float32's rounding: a float32 value
// is the sum of three bfloat16 pieces (8 + 8 + 8 bits), a bfloat16 one is its own piece.
//  correlate: the whole numbers q + z (|q + z| <= 255) are bfloat16 values; a group's products are summed on
//             their own (exactly, but for the float32 accumulation) and multiplied by the group's scale.
//  product:   s (q + z) has at most 16 significant bits: two bfloat16 pieces hold it exactly; of the six
//             products of pieces the last (2^-24) is left out.
// LDS tiles are [row][32 k] with a row stride of 80 bytes (16-byte reads of 16 rows touch every bank once).
constexpr int BM = 128, BN = 128, BK = 32, LROW = 40;      // LROW in bfloat16 values
constexpr int LTILE = 128 * LROW;

struct ManyParams {
    const uint32_t* codes;
    const uint32_t* scales;
    const void* X;           // the float operand: [k][n]
    float* out;              // [m][n]
    float* slab;             // [split][m][n], or null
    int M, N, K;             // rows of the output, its columns, contraction length
    int ldx, ldo;
    int group, groups, words;
    int tiles_m, k_per_split;
    int vec;                 // 16-byte loads of X allowed
};

template <typename T>
__device__ __forceinline__ void load_quad(const ManyParams& p, int k, int n, float (&v)[4]) {
    const T* src = (const T*)p.X + (size_t)k * p.ldx + n;
    v[0] = v[1] = v[2] = v[3] = 0.f;
    if (k >= p.K) return;
    if (p.vec && n + 3 < p.N) {
        if constexpr (sizeof(T) == 4) {
            const float4 f = *reinterpret_cast<const float4*>(src);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(src);
            v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) v[j] = load_val(src + j);
    }
}

template <bool PROD, typename T, int G>
__global__ __launch_bounds__(256) void dict4_many_kernel(ManyParams p) {
    constexpr int PX = sizeof(T) == 4 ? 3 : 1;        // pieces of the float operand
    constexpr int PW = PROD ? 2 : 1;                   // pieces of the weights
    extern __shared__ __align__(16) uint16_t lds[];
    uint16_t* la = lds;                                // [2][PW][128][LROW]
    uint16_t* lb = lds + 2 * PW * LTILE;               // [2][PX][128][LROW]
    float* lscale = (float*)(lb + 2 * PX * LTILE);     // [2][128] (correlate)
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int m0 = (blockIdx.x % p.tiles_m) * BM, n0 = (blockIdx.x / p.tiles_m) * BN;
    const int kbeg = blockIdx.y * p.k_per_split, kend = min(PROD ? p.K : p.words * 8, kbeg + p.k_per_split);
    const int steps = (kend - kbeg + BK - 1) / BK;
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    // the 4 x 4 block of X that this thread stages, and its part of the weights
    const int xk = (lane & 7) * 4, xn = (wave * 8 + (lane >> 3)) * 4;

    float xv[4][4];
    uint32_t cw[2], cs[2];
    auto fetch = [&](int step) {
        const int k = kbeg + step * BK;
#pragma unroll
        for (int j = 0; j < 4; ++j) load_quad<T>(p, k + xk + j, n0 + xn, xv[j]);
        if constexpr (!PROD) {
            const int m = m0 + (t >> 1), w = k / 8 + (t & 1) * 2;
            cw[0] = cw[1] = cs[0] = 0;
            if (m < p.M) {
                const uint2 v = *reinterpret_cast<const uint2*>(p.codes + (size_t)m * p.words + w);
                cw[0] = v.x; cw[1] = v.y;
                cs[0] = p.scales[(size_t)m * p.groups + k / G];
            }
        } else {
            const int w = m0 / 8 + (t & 15);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int kk = k + (t >> 4) * 2 + j;
                cw[j] = cs[j] = 0;
                if (kk < p.K && w < p.words) {
                    cw[j] = p.codes[(size_t)kk * p.words + w];
                    cs[j] = p.scales[(size_t)kk * p.groups + (w * 8) / G];
                }
            }
        }
    };
    auto stage = [&](int buf) {
        uint16_t* b = lb + buf * PX * LTILE;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v0 = xv[0][j], v1 = xv[1][j], v2 = xv[2][j], v3 = xv[3][j];
#pragma unroll
            for (int q = 0; q < PX; ++q) {
                const uint32_t a = pack_bf16(v0, v1), c = pack_bf16(v2, v3);
                *reinterpret_cast<uint2*>(b + q * LTILE + (xn + j) * LROW + xk) = make_uint2(a, c);
                v0 -= bf16_lo(a); v1 -= bf16_hi(a); v2 -= bf16_lo(c); v3 -= bf16_hi(c);
            }
        }
        uint16_t* a = la + buf * PW * LTILE;
        if constexpr (!PROD) {
            const float z = word_offset(cs[0]);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float q[8];
                word_entries(cw[c], q);
                uint4 v;
                v.x = pack_bf16(q[0] + z, q[1] + z); v.y = pack_bf16(q[2] + z, q[3] + z);
                v.z = pack_bf16(q[4] + z, q[5] + z); v.w = pack_bf16(q[6] + z, q[7] + z);
                *reinterpret_cast<uint4*>(a + (t >> 1) * LROW + ((t & 1) * 2 + c) * 8) = v;
            }
            if ((t & 1) == 0) lscale[buf * 128 + (t >> 1)] = word_scale(cs[0]);
        } else {
            float q0[8], q1[8];
            word_entries(cw[0], q0);
            word_entries(cw[1], q1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v0 = word_scale(cs[0]) * (q0[j] + word_offset(cs[0]));
                const float v1 = word_scale(cs[1]) * (q1[j] + word_offset(cs[1]));
                const uint32_t hi = pack_bf16(v0, v1);
                const uint32_t lo = pack_bf16(v0 - bf16_lo(hi), v1 - bf16_hi(hi));
                *reinterpret_cast<uint32_t*>(a + ((t & 15) * 8 + j) * LROW + (t >> 4) * 2) = hi;
                *reinterpret_cast<uint32_t*>(a + LTILE + ((t & 15) * 8 + j) * LROW + (t >> 4) * 2) = lo;
            }
        }
    };

    f32x16 acc[2][2], part[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = part[i][j][e] = 0.f;

    fetch(0);
    stage(0);
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1;
        __syncthreads();
        if (s + 1 < steps) fetch(s + 1);
        const uint16_t* a = la + buf * PW * LTILE;
        const uint16_t* b = lb + buf * PX * LTILE;
        const int at = (lane & 31) * LROW + (lane >> 5) * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            bf16x8 fa[PW][2], fb[PX][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int q = 0; q < PW; ++q)
                    fa[q][i] = *reinterpret_cast<const bf16x8*>(a + q * LTILE + (wm + i * 32) * LROW + at + h * 16);
#pragma unroll
                for (int q = 0; q < PX; ++q)
                    fb[q][i] = *reinterpret_cast<const bf16x8*>(b + q * LTILE + (wn + i * 32) * LROW + at + h * 16);
            }
            // smallest products first
#pragma unroll
            for (int qx = PX - 1; qx >= 0; --qx)
#pragma unroll
                for (int qw = PW - 1; qw >= 0; --qw) {
                    if (qx + qw > 2) continue;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            if constexpr (PROD)
                                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[qw][i], fb[qx][j], acc[i][j], 0, 0, 0);
                            else
                                part[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[qw][i], fb[qx][j], part[i][j], 0, 0, 0);
                        }
                }
        }
        if constexpr (!PROD) {
            const int k = kbeg + s * BK + BK;
            if (k % G == 0 || s + 1 == steps) {           // the group ends: its scale
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float sc = lscale[buf * 128 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            acc[i][j][e] = fmaf(sc, part[i][j][e], acc[i][j][e]);
                            part[i][j][e] = 0.f;
                        }
                    }
            }
        }
        if (s + 1 < steps) stage(buf ^ 1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = n0 + wn + j * 32 + (lane & 31);
            if (n >= p.N) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
                if (m >= p.M) continue;
                if (p.slab) p.slab[((size_t)blockIdx.y * p.M + m) * p.N + n] = acc[i][j][e];
                else p.out[(size_t)m * p.ldo + n] = acc[i][j][e];
            }
        }
}

__global__ __launch_bounds__(256) void dict4_many_reduce_kernel(size_t mn, int N, int splits,
                                                                 const float* __restrict__ slab, float* __restrict__ out,
                                                                 int ldo) {
    for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < mn; e += (size_t)gridDim.x * 256) {
        float s = 0.f;
        for (int z = 0; z < splits; ++z) s += slab[(size_t)z * mn + e];
        out[(e / N) * (size_t)ldo + e % N] = s;
    }
}

// ------------------------------------------------------------------------------------------- launches
constexpr int MOST_COLS = 2147483647 - 1024;    // tile arithmetic in int
constexpr int FEW = 8;           // columns up to which the few-column kernels run

struct FewPlan { int nb, ch; };
FewPlan few_plan(int d, int b) {
    FewPlan f;
    f.nb = b <= 1 ? 1 : b <= 2 ? 2 : b <= 4 ? 4 : 8;
    f.ch = f.nb <= 2 ? 4 : f.nb == 4 ? 2 : 1;
    while (f.ch > 1 && d <= 64 * 8 * (f.ch / 2)) f.ch /= 2;         // one segment is enough with narrower lanes
    return f;
}
int product_few_splits(int d, int r, int ch) {
    const int segs = (d + 512 * ch - 1) / (512 * ch);
    int splits = std::max(1, 512 / segs);
    splits = std::min(splits, (r + 63) / 64);                       // 16 atoms a wave at least
    return std::max(1, splits);
}
int many_splits(int M, int N, int steps, int least) {
    const long long tiles = (long long)((M + BM - 1) / BM) * ((N + BN - 1) / BN);
    if (tiles >= 256) return 1;
    long long s = 512 / tiles;
    s = std::min<long long>(s, steps / least);
    return (int)std::max<long long>(1, s);
}

template <int NB, int CH, typename T>
int correlate_few(onmf_ctx* c, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales,
                  const T* X, int ldx, float* C, hipStream_t s) {
    constexpr int AT = 4, SEG = 512 * CH;
    const int segs = (d + SEG - 1) / SEG, groups = (d + group - 1) / group;
    const int staged = std::min(segs, std::max(1, (int)(65536 / (sizeof(float) * SEG * NB))));
    const size_t bytes = sizeof(float) * (size_t)staged * SEG * NB;
    static LdsLimit lim;
    ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)dict4_correlate_few_kernel<NB, CH, AT, T>, bytes));
    const int chunks = (r + 4 * AT - 1) / (4 * AT);
    hipLaunchKernelGGL((dict4_correlate_few_kernel<NB, CH, AT, T>), dim3(std::min(chunks, 1024)), dim3(256), bytes, s, d, r,
                       b, group, groups, codes, scales, X, ldx, C, staged);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

template <int NB, int CH, typename T>
int product_few(onmf_ctx* c, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales, const T* H,
                int ldh, float* R, int ldr, float* ws, hipStream_t s) {
    const int groups = (d + group - 1) / group, segs = (d + 512 * CH - 1) / (512 * CH);
    int splits = product_few_splits(d, r, CH);
    const int per = (r + splits - 1) / splits;
    splits = (r + per - 1) / per;
    float* slab = splits > 1 ? ws : nullptr;
    hipLaunchKernelGGL((dict4_product_few_kernel<NB, CH, T>), dim3(segs, splits), dim3(256), 0, s, d, r, b, group, groups,
                       codes, scales, H, ldh, R, ldr, per, slab);
    HIP_TRY(c, hipGetLastError());
    if (slab) {
        hipLaunchKernelGGL(dict4_product_few_reduce_kernel, dim3(((size_t)d * b + 63) / 64), dim3(256), 0, s, d, b, splits,
                           slab, R, ldr);
        HIP_TRY(c, hipGetLastError());
    }
    return ONMF_OK;
}

template <bool PROD, typename T, int G>
int many(onmf_ctx* c, ManyParams p, float* ws, hipStream_t s) {
    constexpr int PX = sizeof(T) == 4 ? 3 : 1, PW = PROD ? 2 : 1;
    const size_t bytes = sizeof(uint16_t) * 2 * (PX + PW) * LTILE + (PROD ? 0 : 2 * 128 * sizeof(float));
    static LdsLimit lim;
    ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)dict4_many_kernel<PROD, T, G>, bytes));
    const int unit = PROD ? BK : std::max(BK, G);                   // a split never cuts a group
    const int units = ((PROD ? p.K : p.words * 8) + unit - 1) / unit;
    int splits = many_splits(p.M, p.N, units, std::max(1, 128 / unit));
    const int per = (units + splits - 1) / splits;
    splits = (units + per - 1) / per;
    p.k_per_split = per * unit;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.slab = splits > 1 ? ws : nullptr;
    const int tiles_n = (p.N + BN - 1) / BN;
    hipLaunchKernelGGL((dict4_many_kernel<PROD, T, G>), dim3(p.tiles_m * tiles_n, splits), dim3(256), bytes, s, p);
    HIP_TRY(c, hipGetLastError());
    if (p.slab) {
        const size_t mn = (size_t)p.M * p.N;
        hipLaunchKernelGGL(dict4_many_reduce_kernel, dim3((unsigned)std::min<size_t>((mn + 255) / 256, 4096)), dim3(256), 0, s,
                           mn, p.N, splits, p.slab, p.out, p.ldo);
        HIP_TRY(c, hipGetLastError());
    }
    return ONMF_OK;
}

int check4(onmf_ctx* c, const char* what, int d, int r, int group, const void* codes, const void* scales) {
    if (d <= 0 || r <= 0 || !codes || !scales || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3))
        return onmf_fail(c, ONMF_ERR_ARG, "%s: bad arguments (d=%d r=%d; codes must be aligned to 16 bytes)", what, d, r);
    if (group != 32 && group != 64 && group != 128)
        return onmf_fail(c, ONMF_ERR_ARG, "%s: a group is 32, 64 or 128 features, not %d", what, group);
    if (d > (1 << 18)) return onmf_fail(c, ONMF_ERR_ARG, "%s: d=%d is more than 2^18 features", what, d);
    return ONMF_OK;
}

template <typename T>
int correlate_t(onmf_ctx* c, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales, const T* X,
                int ldx, float* C, float* ws, hipStream_t s) {
    if (b <= FEW) {
        const FewPlan f = few_plan(d, b);
#define FEW_CASE(NB, CH) if (f.nb == NB && f.ch == CH) return correlate_few<NB, CH, T>(c, d, r, b, group, codes, scales, X, ldx, C, s)
        FEW_CASE(1, 1); FEW_CASE(1, 2); FEW_CASE(1, 4); FEW_CASE(2, 1); FEW_CASE(2, 2); FEW_CASE(2, 4);
        FEW_CASE(4, 1); FEW_CASE(4, 2); FEW_CASE(8, 1);
#undef FEW_CASE
    }
    ManyParams p = {};
    p.codes = codes; p.scales = scales; p.X = X; p.out = C;
    p.M = r; p.N = b; p.K = d; p.ldx = ldx; p.ldo = b;
    p.group = group; p.groups = (d + group - 1) / group; p.words = p.groups * (group / 8);
    p.vec = ((uintptr_t)X & (4 * sizeof(T) - 1)) == 0 && (ldx & 3) == 0;
    if (group == 32) return many<false, T, 32>(c, p, ws, s);
    if (group == 64) return many<false, T, 64>(c, p, ws, s);
    return many<false, T, 128>(c, p, ws, s);
}

template <typename T>
int product_t(onmf_ctx* c, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales, const T* H,
              int ldh, float* R, int ldr, float* ws, hipStream_t s) {
    if (b <= FEW) {
        const FewPlan f = few_plan(d, b);
#define FEW_CASE(NB, CH) if (f.nb == NB && f.ch == CH) return product_few<NB, CH, T>(c, d, r, b, group, codes, scales, H, ldh, R, ldr, ws, s)
        FEW_CASE(1, 1); FEW_CASE(1, 2); FEW_CASE(1, 4); FEW_CASE(2, 1); FEW_CASE(2, 2); FEW_CASE(2, 4);
        FEW_CASE(4, 1); FEW_CASE(4, 2); FEW_CASE(8, 1);
#undef FEW_CASE
    }
    ManyParams p = {};
    p.codes = codes; p.scales = scales; p.X = H; p.out = R;
    p.M = d; p.N = b; p.K = r; p.ldx = ldh; p.ldo = ldr;
    p.group = group; p.groups = (d + group - 1) / group; p.words = p.groups * (group / 8);
    p.vec = ((uintptr_t)H & (4 * sizeof(T) - 1)) == 0 && (ldh & 3) == 0;
    if (group == 32) return many<true, T, 32>(c, p, ws, s);
    if (group == 64) return many<true, T, 64>(c, p, ws, s);
    return many<true, T, 128>(c, p, ws, s);
}

}  // namespace

extern "C" {

size_t onmf_dict4_workspace(int which, int d, int r, int b, int group) {
    if (d <= 0 || r <= 0 || b <= 0 || (group != 32 && group != 64 && group != 128)) return 0;
    size_t floats = 0;
    if (b <= FEW) {
        if (which == ONMF_DICT4_PRODUCT) {
            const int splits = product_few_splits(d, r, few_plan(d, b).ch);
            if (splits > 1) floats = (size_t)splits * d * b;
        }
    } else {
        const bool prod = which == ONMF_DICT4_PRODUCT;
        const int unit = prod ? BK : std::max(BK, group);
        const int K = prod ? r : (d + group - 1) / group * group;
        const int M = prod ? d : r;
        const int splits = many_splits(M, b, (K + unit - 1) / unit, std::max(1, 128 / unit));
        if (splits > 1) floats = (size_t)splits * M * b;
    }
    return floats * sizeof(float);
}

int onmf_dict4_pack(onmf_ctx* c, int d, int r, int group, const float* W, void* codes, int32_t* scales, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check4(c, "dict4_pack", d, r, group, codes, scales));
    if (!W) return onmf_fail(c, ONMF_ERR_ARG, "dict4_pack: W is null");
    ONMF_ENTER(c);
    const int groups = (d + group - 1) / group;
    hipLaunchKernelGGL(dict4_pack_kernel, dim3((r + 255) / 256, groups), dim3(256), 0, (hipStream_t)stream, d, r, group,
                       groups, W, (uint32_t*)codes, (uint32_t*)scales);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

int onmf_dict4_unpack(onmf_ctx* c, int d, int r, int group, const void* codes, const int32_t* scales, float* W,
                      void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check4(c, "dict4_unpack", d, r, group, codes, scales));
    if (!W) return onmf_fail(c, ONMF_ERR_ARG, "dict4_unpack: W is null");
    ONMF_ENTER(c);
    const int groups = (d + group - 1) / group;
    hipLaunchKernelGGL(dict4_unpack_kernel, dim3((r + 255) / 256, (d + 7) / 8), dim3(256), 0, (hipStream_t)stream, d, r, group,
                       groups, (const uint32_t*)codes, (const uint32_t*)scales, W);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

int onmf_dict4_correlate(onmf_ctx* c, int d, int r, int b, int group, const void* codes, const int32_t* scales,
                         const void* X, int x_type, int ldx, float* C, void* ws, size_t ws_bytes, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check4(c, "dict4_correlate", d, r, group, codes, scales));
    if (b <= 0 || b > MOST_COLS || !X || !C || ldx < b || (x_type != ONMF_TYPE_F32 && x_type != ONMF_TYPE_BF16))
        return onmf_fail(c, ONMF_ERR_ARG, "dict4_correlate: bad arguments (b=%d ldx=%d type=%d)", b, ldx, x_type);
    const size_t need = onmf_dict4_workspace(ONMF_DICT4_CORRELATE, d, r, b, group);
    if (ws_bytes < need || (need && !ws))
        return onmf_fail(c, ONMF_ERR_ARG, "dict4_correlate: workspace of %zu bytes, %zu needed", ws_bytes, need);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const uint32_t *cw = (const uint32_t*)codes, *sc = (const uint32_t*)scales;
    return x_type == T_F32 ? correlate_t<float>(c, d, r, b, group, cw, sc, (const float*)X, ldx, C, (float*)ws, s)
                           : correlate_t<uint16_t>(c, d, r, b, group, cw, sc, (const uint16_t*)X, ldx, C, (float*)ws, s);
}

int onmf_dict4_product(onmf_ctx* c, int d, int r, int b, int group, const void* codes, const int32_t* scales,
                       const void* H, int h_type, int ldh, float* R, int ldr, void* ws, size_t ws_bytes, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check4(c, "dict4_product", d, r, group, codes, scales));
    if (b <= 0 || b > MOST_COLS || !H || !R || ldh < b || ldr < b || (h_type != ONMF_TYPE_F32 && h_type != ONMF_TYPE_BF16))
        return onmf_fail(c, ONMF_ERR_ARG, "dict4_product: bad arguments (b=%d ldh=%d ldr=%d type=%d)", b, ldh, ldr, h_type);
    const size_t need = onmf_dict4_workspace(ONMF_DICT4_PRODUCT, d, r, b, group);
    if (ws_bytes < need || (need && !ws))
        return onmf_fail(c, ONMF_ERR_ARG, "dict4_product: workspace of %zu bytes, %zu needed", ws_bytes, need);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const uint32_t *cw = (const uint32_t*)codes, *sc = (const uint32_t*)scales;
    return h_type == T_F32 ? product_t<float>(c, d, r, b, group, cw, sc, (const float*)H, ldh, R, ldr, (float*)ws, s)
                           : product_t<uint16_t>(c, d, r, b, group, cw, sc, (const uint16_t*)H, ldh, R, ldr, (float*)ws, s);
}

}  // extern "C"
