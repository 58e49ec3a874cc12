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
#include <cmath>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
// rows of any length: pairs that need no more alignment than their entries (the memory pipe takes them as they lie)
typedef float f32x2_any __attribute__((ext_vector_type(2), aligned(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

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

// Bytes as they are: v_cvt_f32_ubyte<n> takes each where it lies (seeing through the mask, the compiler extracts
// the four bits anew, an instruction more an entry).
__device__ __forceinline__ void whole_bytes(uint32_t& v) { asm("" : "+v"(v)); }

// the eight whole numbers q of a word
__device__ __forceinline__ void word_entries(uint32_t w, float (&q)[8]) {
    uint32_t e = w & 0x0f0f0f0fu, o = (w >> 4) & 0x0f0f0f0fu;     // bytes of e: entries 0 4 1 5, of o: 2 6 3 7
    whole_bytes(e);
    whole_bytes(o);
    q[0] = (float)(e & 0xff);
    q[4] = (float)((e >> 8) & 0xff);
    q[1] = (float)((e >> 16) & 0xff);
    q[5] = (float)(e >> 24);
    q[2] = (float)(o & 0xff);
    q[6] = (float)((o >> 8) & 0xff);
    q[3] = (float)((o >> 16) & 0xff);
    q[7] = (float)(o >> 24);
}

// W^T X multiplies the whole numbers q + z by the columns and adds up 32 features before the scale comes in: up to 32 * 255
// times the largest |x|, which float32 need not hold where it holds the result.  The whole numbers (the one column's kernel: x)
// are therefore shrunk by 2^14, exactly, and the finished sums grown again: what is added up lies within s (q + |z|) |x|.
constexpr float SHRINK = 0x1p-14f, GROW = 0x1p14f;

// ------------------------------------------------------------------------------------------- packing
// smallest bfloat16 >= v (v >= 0, finite), as float
__device__ __forceinline__ float bf16_up(double v) {
    float f = (float)v;
    uint32_t u = __float_as_uint(f);
    if ((double)f < v) ++u;
    if (u & 0xffffu) u = (u & 0xffff0000u) + 0x10000u;
    return __uint_as_float(u);
}

// 64 atoms of a group a workgroup: a lane an atom, so that reads of W (row-major) coalesce, and a quarter of its features
// a wave, all on their way together.  The scale spans the group's range in 15 steps (14 where rounding both ends to the
// grid would need a 16th) and is rounded UP to bfloat16, so no entry is clipped and the error is at most s / 2.  An
// entry next to a rounding border falls on its own side: v times the reciprocal (1 ulp) is within 255.5 (2^-23 + 2^-24)
// = 4.6e-5 of the quotient, and only where it lies that near to a half is the quotient itself taken, in double.
// Bound by memory (d=4096 r=32768, 606 MB: 140 us; one thread a group and all quotients in double 585).
template <int FEATURES>
__global__ __launch_bounds__(256) void dict4_pack_kernel(int d, int r, int groups, const float* __restrict__ W,
                                                          uint32_t* __restrict__ codes, uint32_t* __restrict__ scales) {
    constexpr int EACH = FEATURES / 4;
    __shared__ float ends[2][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = blockIdx.x * 64 + lane, g = blockIdx.y;
    const int i0 = g * FEATURES + wave * EACH, n = min(EACH, d - i0);        // (n: this wave's, or none)
    const float most = __int_as_float(0x7f800000);
    const float* src = W + (size_t)i0 * r + min(k, r - 1);
    float v[EACH], lo = most, hi = -most;
#pragma unroll
    for (int j = 0; j < EACH; ++j) v[j] = j < n ? src[(size_t)j * r] : 0.f;
#pragma unroll
    for (int j = 0; j < EACH; ++j)
        if (j < n) {
            if (!(fabsf(v[j]) < most)) lo = -most;       // a NaN or an infinity: the whole group reads NaN
            lo = fminf(lo, v[j]);
            hi = fmaxf(hi, v[j]);
        }
    ends[0][wave][lane] = lo;
    ends[1][wave][lane] = hi;
    __syncthreads();
    if (k >= r) return;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        lo = fminf(lo, ends[0][w][lane]);
        hi = fmaxf(hi, ends[1][w][lane]);
    }
    uint32_t word[EACH / 8], sc;
#pragma unroll
    for (int w = 0; w < EACH / 8; ++w) word[w] = 0;
    if (lo == -most) {
        sc = 0x7fc00000u;
    } else {
        const double range = (double)hi - (double)lo;
        const double floor_ = fmax(fabs((double)lo), fabs((double)hi)) / 255.0;
        float s = bf16_up(fmax(range / 15.0, floor_));
        if (rint((double)hi / (double)s) - rint((double)lo / (double)s) > 15.0) s = bf16_up(fmax(range / 14.0, floor_));
        if (!(s >= 1.17549435e-38f)) {     // nothing but (next to) zeros
            sc = 0;
        } else {
            const float z = (float)rint((double)lo / (double)s), inv = __builtin_amdgcn_rcpf(s);
            sc = __float_as_uint(s) | ((uint32_t)(int)z & 0xffffu);
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                const float f = v[j] * inv;
                float q = rintf(f);
                if (fabsf(f - q) > 0.4999f) q = (float)rint((double)v[j] / (double)s);
                if (j < n) word[j / 8] |= (uint32_t)(int)(q - z) << (4 * ((j % 8 >> 1) + 4 * (j & 1)));
            }
        }
    }
    uint32_t* out = codes + ((size_t)k * groups + g) * (FEATURES / 8) + wave * (EACH / 8);
    if constexpr (EACH == 32) *reinterpret_cast<uint4*>(out) = make_uint4(word[0], word[1], word[2], word[3]);
    else if constexpr (EACH == 16) *reinterpret_cast<uint2*>(out) = make_uint2(word[0], word[1]);
    else out[0] = word[0];
    if (wave == 0) scales[(size_t)k * groups + g] = sc;
}

// One thread per four words (32 features, of one group); neighbouring threads take neighbouring atoms (W's fast index).
// Bound by memory (d=4096 r=32768, 606 MB: 149 us).
__global__ __launch_bounds__(256) void dict4_unpack_kernel(int d, int r, int group, int groups,
                                                            const uint32_t* __restrict__ codes,
                                                            const uint32_t* __restrict__ scales, float* __restrict__ W) {
    const int k = blockIdx.x * 256 + threadIdx.x, w = blockIdx.y * 4;
    if (k >= r) return;
    const uint32_t sc = scales[(size_t)k * groups + (w * 8) / group];
    const float s = word_scale(sc), z = word_offset(sc);
    const uint4 v = *reinterpret_cast<const uint4*>(codes + (size_t)k * groups * (group / 8) + w);
    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        float q[8];
        word_entries(words[u], q);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if ((w + u) * 8 + j < d) W[(size_t)((w + u) * 8 + j) * r + k] = s * (q[j] + z);
    }
}

// ------------------------------------------------------------------------------------------- few columns
// C = W^T x for one column: bound by reading the codes once (d=4096 r=32768, 71 MB: 17 us, 4.2 TB/s; d=441 r=25 3 us, a
// launch).  A lane owns F = 8 CH consecutive features of a segment of 64 F; x is staged in LDS as float and a
// segment's F values are held in registers while AT atoms stream past.  An entry costs an extraction (0.4), a
// conversion and a fused multiply-add; z is taken once a group, with the sum of its features.
// LDS: quad q (of F / 4) of lane l of segment g at [((g * F/4 + q) * 64 + l) * 4].
template <int CH, int AT, typename T>
__global__ __launch_bounds__(256) void dict4_correlate_one_kernel(int d, int r, int group, int groups,
                                                                   const uint32_t* __restrict__ codes,
                                                                   const uint32_t* __restrict__ scales,
                                                                   const T* __restrict__ X, int ldx,
                                                                   float* __restrict__ C, int segs_staged) {
    constexpr int F = 8 * CH, SEG = 64 * F;
    extern __shared__ __align__(16) float xs[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int segs = (d + SEG - 1) / SEG;
    const int words = groups * (group / 8);
    const int chunks = (r + 4 * AT - 1) / (4 * AT);
    bool first = true;
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int k0 = chunk * 4 * AT + wave * AT;
        float acc[AT];
#pragma unroll
        for (int a = 0; a < AT; ++a) acc[a] = 0.f;
        for (int s0 = 0; s0 < segs; s0 += segs_staged) {
            if (first || segs_staged < segs) {          // the whole of x fits: staged once
                __syncthreads();
                const int i0 = s0 * SEG, in = min(segs_staged, segs - s0) * SEG;
#pragma unroll 4
                for (int i = threadIdx.x; i < in; i += 256) {        // (features behind the last: its value, not used)
                    const float x = load_val(X + (size_t)min(i0 + i, d - 1) * ldx), v = i0 + i < d ? x * SHRINK : 0.f;
                    const int g = i / SEG, l = (i % SEG) / F, f = i % F;
                    xs[((g * (F / 4) + (f >> 2)) * 64 + l) * 4 + (f & 3)] = v;
                }
                __syncthreads();
                first = false;
            }
            const int sn = min(segs_staged, segs - s0);
            for (int g = 0; g < sn; ++g) {
                const int w0 = (s0 + g) * (SEG / 8) + lane * CH;       // this lane's first word
                if (w0 >= words) continue;                               // padding of the last segment
                float x[F], sum = 0.f;
#pragma unroll
                for (int q = 0; q < F / 4; ++q) {
                    const float4 v = *reinterpret_cast<const float4*>(&xs[((g * (F / 4) + q) * 64 + lane) * 4]);
                    x[4 * q + 0] = v.x; x[4 * q + 1] = v.y; x[4 * q + 2] = v.z; x[4 * q + 3] = v.w;
                    sum += (v.x + v.y) + (v.z + v.w);
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
                    float t = word_offset(sc[a]) * sum;
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        float q[8];
                        word_entries(cw[a][c], q);
#pragma unroll
                        for (int j = 0; j < 8; ++j) t = fmaf(q[j], x[8 * c + j], t);
                    }
                    acc[a] = fmaf(word_scale(sc[a]), t, acc[a]);
                }
            }
        }
#pragma unroll
        for (int a = 0; a < AT; ++a) {
            float v = acc[a];
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
            if (lane == 0 && k0 + a < r) C[k0 + a] = v * GROW;
        }
    }
}

// R = W H for one or two columns (d=8192 r=16384, 75 MB with the scales: 20 and 27 us; d=1024 r=256 5 us, one launch):
// bound by instructions, 1.4 + NB an entry, and by the codes' way from memory.  A lane owns F features of a segment and
// adds up its atoms' contributions h (s q + s z) in registers; the NW waves of a workgroup take different atoms, AT at
// a time, and are added in LDS, workgroups of the same segment in slabs; both in a fixed order.
template <int NB, int CH, int NW, typename T>
__global__ __launch_bounds__(64 * NW) void dict4_product_few_kernel(int d, int r, int b, int group, int groups,
                                                                     const uint32_t* __restrict__ codes,
                                                                     const uint32_t* __restrict__ scales,
                                                                     const T* __restrict__ H, int ldh, float* __restrict__ R,
                                                                     int ldr, int atoms_per_wg, float* __restrict__ slab) {
    constexpr int F = 8 * CH, SEG = 64 * F, AT = 8;
    __shared__ float part[NW][NB][SEG];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int words = groups * (group / 8);
    const int w0 = min((int)(blockIdx.x * (SEG / 8) + lane * CH), words - CH);      // (features behind the last are not stored)
    const int ka = blockIdx.y * atoms_per_wg, kb = min(r, ka + atoms_per_wg);
    float acc[F][NB], zacc[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        zacc[n] = 0.f;
#pragma unroll
        for (int f = 0; f < F; ++f) acc[f][n] = 0.f;
    }
    const int g = w0 * 8 / group;
    for (int k0 = ka + wave * AT; k0 < kb; k0 += NW * AT) {
        uint32_t cw[AT][CH], sc[AT];
        float h[AT][NB];
#pragma unroll
        for (int a = 0; a < AT; ++a) {
            const int k = min(k0 + a, kb - 1);
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
            sc[a] = scales[(size_t)k * groups + g];
#pragma unroll
            for (int n = 0; n < NB; ++n) h[a][n] = load_val(H + (size_t)k * ldh + min(n, b - 1));
        }
#pragma unroll
        for (int a = 0; a < AT; ++a) {
            float hs[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) h[a][n] = k0 + a < kb ? h[a][n] : 0.f;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                hs[n] = word_scale(sc[a]) * h[a][n];
                zacc[n] = fmaf(word_offset(sc[a]), hs[n], zacc[n]);
            }
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float q[8];
                word_entries(cw[a][c], q);
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int n = 0; n < NB; ++n) acc[8 * c + j][n] = fmaf(q[j], hs[n], acc[8 * c + j][n]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int f = 0; f < F; ++f) part[wave][n][f * 64 + lane] = acc[f][n] + zacc[n];
    __syncthreads();
    for (int e = threadIdx.x; e < NB * SEG; e += 64 * NW) {
        const int n = e / SEG, at = e % SEG, i = blockIdx.x * SEG + (at & 63) * F + (at >> 6);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += part[w][n][at];
        if (i < d && n < b) {
            if (slab) slab[((size_t)blockIdx.y * d + i) * b + n] = v;
            else R[(size_t)i * ldr + n] = v;
        }
    }
}

// R = W H for a few to 1024 columns on the matrix pipe (16x16x32 bfloat16).  A lane takes the words of eight atoms: the
// eight nibbles at one place are the operand of one row at eight consecutive steps of the contraction, so a tile's
// 16 rows are the features at that place of the words of 16 lanes, and nothing has to be turned round.  An entry
// s (q + z) has at most 16 significant bits: its upper half and the rest are bfloat16 values exactly.  Per weight
// 5.4 vector instructions whatever the number of columns, against 1.4 + one a column on the vector pipe: they are
// the bound (d=8192 r=16384 b=7 39 us, b=32 56 us; the codes and scales are 75 MB).
// The waves of a workgroup take different atoms of the same 128 CW features and are added in LDS, workgroups of
// the same features in slabs; both in a fixed order.
template <int NT, int CW, typename T>
__global__ __launch_bounds__(256, 2) void dict4_product_tile_kernel(int d, int r, int b, int group, int groups,
                                                                  const uint32_t* __restrict__ codes,
                                                                  const uint32_t* __restrict__ scales,
                                                                  const T* __restrict__ H, int ldh, float* __restrict__ R,
                                                                  int ldr, int atoms_per_wg, float* __restrict__ slab) {
    constexpr int PX = sizeof(T) == 4 ? 3 : 1, TILES = 8 * CW * NT;
    extern __shared__ __align__(16) float part[];             // [4 waves][TILES][64 lanes][4]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, kg = lane >> 4;
    const int words = groups * (group / 8);
    const int c0 = blockIdx.z * 16 * NT, cols = min(16 * NT, b - c0);
    const int w0 = min((int)(blockIdx.x * 16 + m) * CW, words - CW);           // (rows behind the last are not stored)
    const int g = w0 * 8 / group;
    const int ka = blockIdx.y * atoms_per_wg, kb = min(r, ka + atoms_per_wg);
    f32x4 acc[CW][8][NT];
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[c][j][n] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Raw { uint32_t cw[8][CW], sc[8]; float h[8][NT]; };
    auto fetch = [&](int k0, Raw& x) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = min(k0 + kg * 8 + j, r - 1);
            const uint32_t* src = codes + (size_t)k * words + w0;
            if constexpr (CW == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(src);
                x.cw[j][0] = v.x; x.cw[j][1] = v.y;
            } else {
                x.cw[j][0] = *src;
            }
            x.sc[j] = scales[(size_t)k * groups + g];
#pragma unroll
            for (int n = 0; n < NT; ++n) x.h[j][n] = load_val(H + (size_t)k * ldh + c0 + min(16 * n + m, cols - 1));
        }
    };
    auto compute = [&](int k0, Raw& x) {
        uint4 fb[NT][PX];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k0 + kg * 8 + j < kb ? x.h[j][n] : 0.f;
#pragma unroll
            for (int q = 0; q < PX; ++q) {
                uint32_t u[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                    v[2 * j] -= bf16_lo(u[j]);
                    v[2 * j + 1] -= bf16_hi(u[j]);
                }
                fb[n][q] = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
        float s[8], zs[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            s[j] = word_scale(x.sc[j]);
            zs[j] = s[j] * word_offset(x.sc[j]);
        }
#pragma unroll
        for (int c = 0; c < CW; ++c)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t nib[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    nib[j] = (half ? x.cw[j][c] >> 4 : x.cw[j][c]) & 0x0f0f0f0fu;
                    whole_bytes(nib[j]);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int entry = 2 * half + (q >> 1) + 4 * (q & 1);       // bytes: entries 0 4 1 5, then 2 6 3 7
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float v0 = fmaf((float)((nib[2 * j] >> (8 * q)) & 0xff), s[2 * j], zs[2 * j]);
                        const float v1 = fmaf((float)((nib[2 * j + 1] >> (8 * q)) & 0xff), s[2 * j + 1], zs[2 * j + 1]);
                        const uint32_t b0 = __float_as_uint(v0), b1 = __float_as_uint(v1);
                        hi[j] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
                        lo[j] = __builtin_amdgcn_perm(__float_as_uint(v1 - __uint_as_float(b1 & 0xffff0000u)),
                                                      __float_as_uint(v0 - __uint_as_float(b0 & 0xffff0000u)), 0x07060302u);
                    }
                    const bf16x8 ahi = __builtin_bit_cast(bf16x8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                    const bf16x8 alo = __builtin_bit_cast(bf16x8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
                    // smallest products first; of the six the last (2^-24) is left out
#pragma unroll
                    for (int qx = PX - 1; qx >= 0; --qx)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const bf16x8 f = __builtin_bit_cast(bf16x8, fb[n][qx]);
                            if (qx < 2) acc[c][entry][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(alo, f, acc[c][entry][n], 0, 0, 0);
                            acc[c][entry][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ahi, f, acc[c][entry][n], 0, 0, 0);
                        }
                    // (here and now: all entries unpacked first would fill the registers)
#pragma unroll
                    for (int n = 0; n < NT; ++n) asm volatile("" : "+v"(acc[c][entry][n]));
                }
            }
    };
    Raw even, odd;
    int k0 = ka + wave * 32;
    if (k0 < kb) fetch(k0, even);
    while (k0 < kb) {
        if (k0 + 128 < kb) fetch(k0 + 128, odd);
        compute(k0, even);
        k0 += 128;
        if (k0 >= kb) break;
        if (k0 + 128 < kb) fetch(k0 + 128, even);
        compute(k0, odd);
        k0 += 128;
    }
#pragma unroll
    for (int c = 0; c < CW; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                *reinterpret_cast<f32x4*>(part + ((size_t)(wave * TILES + (c * 8 + j) * NT + n) * 64 + lane) * 4) = acc[c][j][n];
    __syncthreads();
#pragma unroll 4
    for (int ti = wave; ti < TILES; ti += 4) {
        f32x4 v = *reinterpret_cast<const f32x4*>(part + ((size_t)ti * 64 + lane) * 4);
#pragma unroll
        for (int w = 1; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(part + ((size_t)(w * TILES + ti) * 64 + lane) * 4);
        const int n = ti % NT * 16 + (lane & 15), j = ti / NT % 8, c = ti / NT / 8;
        if (n >= cols) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = (((int)blockIdx.x * 16 + 4 * (lane >> 4) + e) * CW + c) * 8 + j;
            if (i >= d) continue;
            if (slab) slab[((size_t)blockIdx.y * d + i) * b + c0 + n] = v[e];
            else R[(size_t)i * ldr + c0 + n] = v[e];
        }
    }
}

// out[m][n] = sum over the slabs z of slab[z][m][n], four threads an entry, in a fixed order; bound by reading them
// (22 slabs of 16384 x 64: 22 us, 4.2 TB/s)
__global__ __launch_bounds__(256) void dict4_reduce_kernel(size_t mn, int N, int splits, const float* __restrict__ slab,
                                                            float* __restrict__ out, int ldo) {
    __shared__ float part[4][64];
    const int o = threadIdx.x & 63, g = threadIdx.x >> 6;
    for (size_t base = (size_t)blockIdx.x * 64; base < mn; base += (size_t)gridDim.x * 64) {
        const size_t e = base + o;
        float s = 0.f;
        if (e < mn) {
#pragma unroll 8
            for (int z = g; z < splits; z += 4) s += slab[(size_t)z * mn + e];
        }
        part[g][o] = s;
        __syncthreads();
        if (g == 0 && e < mn) out[(e / N) * (size_t)ldo + e % N] = (part[0][o] + part[1][o]) + (part[2][o] + part[3][o]);
        __syncthreads();
    }
}

// C = W^T X for a few to 512 columns on the matrix pipe (16x16x32 bfloat16), straight from the nibbles.  The result is
// computed with X as the rows' operand and W as the columns': a lane's operand is one word (eight features of the atom
// l % 16, at word l / 16 of a step's four), its part of the sum belongs to that same atom, and the group's scale, which
// the lane has, is multiplied to it; the whole numbers q + z themselves are bfloat16 values.  A workgroup keeps
// `per` features of X in LDS, already cut into bfloat16 pieces in the operand's order, and its waves take 32 atoms at a
// time past it; ranges of features are added up in slabs.  A lane loads 16 bytes, four words of 128 features, two
// blocks ahead; the 4 x 4 words of the lanes l % 16 + 16 j change places in four instructions.  Bound by its vector
// instructions (3 an entry for up to 16 columns) and, with more columns, the operand reads from LDS and the slabs
// (float32, d=8192 r=16384: b=8 58 us and 5 for adding up, b=32 54 and 8, b=64 69 and 22).
template <int NT, typename T>
__global__ __launch_bounds__(512) void dict4_correlate_tile_kernel(int d, int r, int b, int group, int groups,
                                                                      const uint32_t* __restrict__ codes,
                                                                      const uint32_t* __restrict__ scales,
                                                                      const T* __restrict__ X, int ldx, float* __restrict__ C,
                                                                      int per, float* __restrict__ slab) {
    constexpr int PX = sizeof(T) == 4 ? 3 : 1, AT = 2;
    extern __shared__ __align__(16) uint4 xop[];              // [step of 32][NT][PX][64 lanes]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), m = lane & 15, kq = lane >> 4;
    const int words = groups * (group / 8);
    const int c0 = blockIdx.z * 16 * NT, cols = min(16 * NT, b - c0);
    const int f0 = blockIdx.y * per, f1 = min(d, f0 + per), blocks = (f1 - f0 + 127) / 128;
#pragma unroll 2
    for (int e = t; e < blocks * 4 * NT * 64; e += 512) {
        const int at = e >> 6, n = at % NT * 16 + m, k0 = f0 + at / NT * 32 + 8 * kq;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = load_val(X + (size_t)min(k0 + j, d - 1) * ldx + c0 + min(n, cols - 1));
            v[j] = k0 + j < d ? x : 0.f;
        }
#pragma unroll
        for (int q = 0; q < PX; ++q) {
            uint32_t u[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                v[2 * j] -= bf16_lo(u[j]);
                v[2 * j + 1] -= bf16_hi(u[j]);
            }
            xop[(at * PX + q) * 64 + lane] = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
    __syncthreads();
    const int tiles = (r + 16 * AT - 1) / (16 * AT), stride = gridDim.x * 8;
    struct Raw { uint4 cw[AT]; uint32_t sc[AT][4]; };
    // (atoms behind the last one are the last one, words behind a row's last one its last ones, where X is zero)
    auto fetch = [&](int tile, int blk, Raw& x) {
        const int f = f0 + blk * 128;
#pragma unroll
        for (int a = 0; a < AT; ++a) {
            const int k = min(tile * 16 * AT + 16 * a + m, r - 1);
            x.cw[a] = *reinterpret_cast<const uint4*>(codes + (size_t)k * words + min(f / 8 + 4 * kq, words - 4));
#pragma unroll
            for (int j = 0; j < 4; ++j) x.sc[a][j] = scales[(size_t)k * groups + min((f + 32 * j) / group, groups - 1)];
        }
    };
    f32x4 acc[AT][NT];
    auto compute = [&](int tile, int blk, Raw& x) {
        if (blk == 0)
#pragma unroll
            for (int a = 0; a < AT; ++a)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[a][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        uint32_t w[AT][4];
#pragma unroll
        for (int a = 0; a < AT; ++a) {
            // word 4 row + j in place j of a row of lanes -> word 4 j + row
            const auto p0 = __builtin_amdgcn_permlane32_swap(x.cw[a].x, x.cw[a].z, false, false);
            const auto p1 = __builtin_amdgcn_permlane32_swap(x.cw[a].y, x.cw[a].w, false, false);
            const auto q0 = __builtin_amdgcn_permlane16_swap(p0[0], p1[0], false, false);
            const auto q1 = __builtin_amdgcn_permlane16_swap(p0[1], p1[1], false, false);
            w[a][0] = q0[0]; w[a][1] = q0[1]; w[a][2] = q1[0]; w[a][3] = q1[1];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bf16x8 xo[NT][PX];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int q = 0; q < PX; ++q)
                    xo[n][q] = __builtin_bit_cast(bf16x8, xop[(((blk * 4 + j) * NT + n) * PX + q) * 64 + lane]);
#pragma unroll
            for (int a = 0; a < AT; ++a) {
                const float s = word_scale(x.sc[a][j]), z = word_offset(x.sc[a][j]) * SHRINK;
                float q[8];
                word_entries(w[a][j], q);
#pragma unroll
                for (int i = 0; i < 8; ++i) q[i] = fmaf(q[i], SHRINK, z);
                const bf16x8 wo = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16(q[0], q[1]), pack_bf16(q[2], q[3]),
                                                                        pack_bf16(q[4], q[5]), pack_bf16(q[6], q[7])));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    f32x4 part = f32x4{0.f, 0.f, 0.f, 0.f};
                    // smallest products first
#pragma unroll
                    for (int p = PX - 1; p >= 0; --p) part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xo[n][p], wo, part, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][n][e] = fmaf(s, part[e], acc[a][n][e]);
                }
            }
        }
        if (blk != blocks - 1) return;
        float* out = slab ? slab + (size_t)blockIdx.y * r * b : C;
#pragma unroll
        for (int a = 0; a < AT; ++a) {
            const int k = tile * 16 * AT + 16 * a + m;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int col = 16 * n + 4 * kq;
                float* dst = out + (size_t)k * b + c0 + col;
                if (k < r && col + 4 <= cols) *reinterpret_cast<f32x4_any*>(dst) = acc[a][n] * GROW;
                else if (k < r)
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (col + e < cols) dst[e] = acc[a][n][e] * GROW;
            }
        }
    };
    int tile = blockIdx.x * 8 + wave, blk = 0;                // ... of the loads that are sent for next
    auto ahead = [&]() {
        if (++blk == blocks) {
            blk = 0;
            tile += stride;
        }
    };
    Raw even, odd;
    int ct = tile, cb = 0;                                    // ... and of those that are computed
    auto after = [&]() {
        if (++cb == blocks) {
            cb = 0;
            ct += stride;
        }
    };
    if (tile < tiles) fetch(tile, blk, even);
    ahead();
    if (tile < tiles) fetch(tile, blk, odd);
    ahead();
    while (ct < tiles) {
        compute(ct, cb, even);
        after();
        if (tile < tiles) fetch(tile, blk, even);
        ahead();
        if (ct >= tiles) break;
        compute(ct, cb, odd);
        after();
        if (tile < tiles) fetch(tile, blk, odd);
        ahead();
    }
}

// The same for results so small that a launch counts as much as the work: a workgroup owns 16 atoms, its NW waves share the
// steps of 32 features, DEPTH of them on their way, each cutting its part of X into pieces itself, and add up in LDS
// (d=441 r=72 b=3 3.4 us, of which a launch is 2.5; by ranges and slabs 7.4).
template <int NT, int NW, typename T>
__global__ __launch_bounds__(64 * NW) void dict4_correlate_wave_kernel(int d, int r, int b, int group, int groups,
                                                                       const uint32_t* __restrict__ codes,
                                                                       const uint32_t* __restrict__ scales,
                                                                       const T* __restrict__ X, int ldx, float* __restrict__ C) {
    constexpr int PX = sizeof(T) == 4 ? 3 : 1, DEPTH = NT == 1 ? 4 : NT == 2 ? 3 : 2;
    __shared__ __align__(16) f32x4 part[NW][NT][64];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), m = lane & 15, kq = lane >> 4;
    const int words = groups * (group / 8), steps = (d + 31) / 32;
    const int k = min((int)blockIdx.x * 16 + m, r - 1);                       // (atoms behind the last one are not stored)
    const uint32_t* code = codes + (size_t)k * words + kq;
    const uint32_t* scale = scales + (size_t)k * groups;
    struct Raw { uint32_t w, sc; float x[NT][8]; };
    auto fetch = [&](int s, Raw& v) {
        v.w = code[4 * s];
        v.sc = scale[32 * s / group];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v.x[n][j] = load_val(X + (size_t)min(32 * s + 8 * kq + j, d - 1) * ldx + min(16 * n + m, b - 1));
    };
    f32x4 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int s, Raw& v) {
        const float sc = word_scale(v.sc), z = word_offset(v.sc) * SHRINK;
        float q[8];
        word_entries(v.w, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = fmaf(q[i], SHRINK, z);
        const bf16x8 wo = __builtin_bit_cast(bf16x8, make_uint4(pack_bf16(q[0], q[1]), pack_bf16(q[2], q[3]),
                                                                pack_bf16(q[4], q[5]), pack_bf16(q[6], q[7])));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float x[8];
            uint4 xo[PX];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 32 * s + 8 * kq + j < d ? v.x[n][j] : 0.f;
#pragma unroll
            for (int p = 0; p < PX; ++p) {
                uint32_t u[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u[j] = pack_bf16(x[2 * j], x[2 * j + 1]);
                    x[2 * j] -= bf16_lo(u[j]);
                    x[2 * j + 1] -= bf16_hi(u[j]);
                }
                xo[p] = make_uint4(u[0], u[1], u[2], u[3]);
            }
            f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = PX - 1; p >= 0; --p)
                sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xo[p]), wo, sum, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = fmaf(sc, sum[e], acc[n][e]);
        }
    };
    Raw raw[DEPTH];
#pragma unroll
    for (int j = 0; j < DEPTH; ++j)
        if (wave + j * NW < steps) fetch(wave + j * NW, raw[j]);
    for (int s = wave; s < steps; s += DEPTH * NW)
#pragma unroll
        for (int j = 0; j < DEPTH; ++j)
            if (s + j * NW < steps) {
                compute(s + j * NW, raw[j]);
                if (s + (j + DEPTH) * NW < steps) fetch(s + (j + DEPTH) * NW, raw[j]);
            }
#pragma unroll
    for (int n = 0; n < NT; ++n) part[wave][n][lane] = acc[n];
    __syncthreads();
    for (int e = t; e < NT * 256; e += 64 * NW) {
        const int n = e >> 8, l = (e >> 2) & 63, atom = blockIdx.x * 16 + (l & 15), col = 16 * n + 4 * (l >> 4) + (e & 3);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) v += part[w][n][l][e & 3];
        if (atom < r && col < b) C[(size_t)atom * b + col] = v * GROW;
    }
}

// ------------------------------------------------------------------------------------------- many columns
// The bfloat16 matrix pipe (16x16x32), exact to float32's rounding: a float32 value is the sum of three bfloat16
// pieces (8 + 8 + 8 bits), a bfloat16 one is its own piece.
//  correlate: the whole numbers q + z (|q + z| <= 255), shrunk, are bfloat16 values; 32 features' products are summed
//             on their own and multiplied by their group's scale.
//  product:   s (q + z) has at most 16 significant bits: two bfloat16 pieces hold it exactly; of the six
//             products of pieces the last (2^-24) is left out.
// The weights are laid out as bfloat16 rows [piece][m][k] in the workspace first (unpacked in the product's kernel
// itself they cost every 128 columns as many vector instructions as the columns' own split).
// A workgroup owns 16 MT rows and 128 (bfloat16: 256) columns, a wave all its rows and a quarter of its columns, so
// that every column is split into its pieces once and in registers: lane l holds columns 2 (l % 16) and the next, at
// k = 8 (l / 16) .. + 7, the operand of two tiles.  (bfloat16 columns need no split and a wave takes four tiles of
// them, for half the reads of weights from LDS, which bound it before: d=1024 r=256 b=65536 66 -> 54 us.)  The weights
// go from memory to LDS, one step of 32 ahead, in rows of 64 bytes whose 16-byte chunks are permuted by
// (row >> 2) & 3: the 16 rows of an operand read meet every bank once.
// Bound by the matrix pipe: W^T X d=1024 r=256 b=65536 float32 100 us, 1.03 PFLOP/s of the three products; W H 162 us,
// 1.06 of five; with few columns by what a step waits for its loads.
constexpr int BK = 32;

// correlate's weights: [k][features, padded to whole groups with zeros] whole numbers, and the scales as floats [group][k];
// bound by writing them (d=6492 r=9202, 157 MB: 35 us)
__global__ __launch_bounds__(256) void dict4_lay_correlate_kernel(int d, int r, int words, int group, int groups,
                                                                   const uint32_t* __restrict__ codes,
                                                                   const uint32_t* __restrict__ scales,
                                                                   uint4* __restrict__ A, float* __restrict__ S) {
    const size_t all = (size_t)r * words;
    for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (size_t)gridDim.x * 256) {
        const int k = (int)(e / words), w = (int)(e % words), g = w * 8 / group;
        const uint32_t sc = scales[(size_t)k * groups + g];
        const float z = word_offset(sc) * SHRINK;
        float q[8];
        word_entries(codes[e], q);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = w * 8 + j < d ? fmaf(q[j], SHRINK, z) : 0.f;
        A[e] = make_uint4(pack_bf16(q[0], q[1]), pack_bf16(q[2], q[3]), pack_bf16(q[4], q[5]), pack_bf16(q[6], q[7]));
        if (w * 8 % group == 0) S[(size_t)g * r + k] = word_scale(sc);
    }
}

// the product's weights: [piece][feature][atoms, padded to kp with zeros]; 128 features x 64 atoms a workgroup,
// turned round in LDS (d=1200 r=100 6 us; bound by writing them where they are many, 4 bytes a weight)
__global__ __launch_bounds__(256) void dict4_lay_product_kernel(int d, int r, int words, int group, int groups, int kp,
                                                                 const uint32_t* __restrict__ codes,
                                                                 const uint32_t* __restrict__ scales,
                                                                 uint16_t* __restrict__ A) {
    __shared__ __align__(16) uint16_t tile[2][128][64 + 8];
    const int t = threadIdx.x, w0 = blockIdx.y * 16, k0 = blockIdx.x * 64;
    const int w = w0 + (t & 15), k = k0 + (t >> 4) * 4;
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool there = k + j < r && w < words;
        const uint32_t sc = there ? scales[(size_t)(k + j) * groups + w * 8 / group] : 0;
        word_entries(there ? codes[(size_t)(k + j) * words + w] : 0, v[j]);
#pragma unroll
        for (int f = 0; f < 8; ++f) v[j][f] = word_scale(sc) * (v[j][f] + word_offset(sc));
    }
#pragma unroll
    for (int f = 0; f < 8; ++f) {
        const uint32_t a = pack_bf16(v[0][f], v[1][f]), b = pack_bf16(v[2][f], v[3][f]);
        const uint32_t c = pack_bf16(v[0][f] - bf16_lo(a), v[1][f] - bf16_hi(a)), e = pack_bf16(v[2][f] - bf16_lo(b), v[3][f] - bf16_hi(b));
        *reinterpret_cast<uint2*>(&tile[0][(t & 15) * 8 + f][(t >> 4) * 4]) = make_uint2(a, b);
        *reinterpret_cast<uint2*>(&tile[1][(t & 15) * 8 + f][(t >> 4) * 4]) = make_uint2(c, e);
    }
    __syncthreads();
#pragma unroll
    for (int e = t; e < 2 * 128 * 8; e += 256) {
        const int piece = e >> 10, f = (e >> 3) & 127, c = (e & 7) * 8;
        const int i = w0 * 8 + f;
        if (i < d && k0 + c < kp)
            *reinterpret_cast<uint4*>(A + ((size_t)piece * d + i) * kp + k0 + c) = *reinterpret_cast<const uint4*>(&tile[piece][f][c]);
    }
}

struct ManyParams {
    const uint16_t* A;       // [piece][M][kp] bfloat16
    const float* S;          // correlate: [group][M]
    const void* X;           // the float operand: [k][n]
    float* out;              // [m][n]
    float* slab;             // [split][m][n], or null
    int M, N, K, kp;         // rows of the output, its columns, contraction length and that of A's rows
    int ldx, ldo, group;
    int tiles_m, tiles, k_per_split;
};

// A wave's columns in sixteens, as many as a lane loads at once: two float32 values or four bfloat16 ones.
template <typename T> constexpr int COLUMN_TILES = sizeof(T) == 4 ? 2 : 4;
template <typename T> constexpr int COLUMN_PIECES = sizeof(T) == 4 ? 3 : 1;

// 32 rows of a wave's columns on their way to the matrix pipe.  OFF: 32 bits where 32 rows of X lie within them.
template <typename T, typename OFF>
struct Columns {
    static constexpr int CT = COLUMN_TILES<T>, PX = COLUMN_PIECES<T>;
    const char* X;
    int N, K, ldx, kl, na, late;
    bool some_late;
    u32x2_any xr[8];

    __device__ __forceinline__ Columns(const void* X_, int N_, int K_, int ldx_, int lane)
        : X((const char*)X_), N(N_), K(K_), ldx(ldx_), kl(8 * (lane >> 4)) {}
    // Columns behind the last one are not stored.  A lane that has some reads the last CT columns, its own first among
    // them at place `late`.
    __device__ __forceinline__ void place(int n0, int lane) {
        na = min(n0 + CT * (lane & 15), N - CT);
        late = min(n0 + CT * (lane & 15) - na, CT - 1);
        some_late = __any(late);
    }
    // rows k .. k + 31 (k < K); those behind the last one are the last one (the weights are zero there)
    __device__ __forceinline__ void fetch(int k) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            xr[j] = *reinterpret_cast<const u32x2_any*>(X + (size_t)k * ldx * sizeof(T) +
                                                        ((OFF)min(kl + j, K - 1 - k) * (OFF)ldx + (OFF)na) * (OFF)sizeof(T));
    }
    __device__ __forceinline__ void split(uint4 (&fb)[CT][PX]) {
        if (some_late)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint64_t v = ((uint64_t)xr[j][1] << 32 | xr[j][0]) >> (late * (64 / CT));
                xr[j][0] = (uint32_t)v;
                xr[j][1] = (uint32_t)(v >> 32);
            }
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            uint32_t u[4];
            if constexpr (PX == 1) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    u[j] = __builtin_amdgcn_perm(xr[2 * j + 1][c / 2], xr[2 * j][c / 2], c % 2 ? 0x07060302u : 0x05040100u);
                fb[c][0] = make_uint4(u[0], u[1], u[2], u[3]);
            } else {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(xr[j][c]);
#pragma unroll
                for (int q = 0; q < PX; ++q) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        u[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                        v[2 * j] -= bf16_lo(u[j]);
                        v[2 * j + 1] -= bf16_hi(u[j]);
                    }
                    fb[c][q] = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
        }
    }
};

// A step of 32 of the contraction for 16 MT rows: the weights' operands at `a` (1024 bytes a piece and sixteen rows),
// correlate's scales at `s`.
template <bool PROD, int MT, int CT, int PX>
__device__ __forceinline__ void row_tiles(const char* a, const float* s, int lane, const uint4 (&fb)[CT][PX], f32x4 (&acc)[MT][CT]) {
    constexpr int PW = PROD ? 2 : 1;
    const int op = (lane & 15) * 64 + (((lane >> 4) ^ ((lane >> 2) & 3)) * 16);
    // the next tile's weights and scales are read while this one's are used
    bf16x8 fa[2][PW];
    f32x4 sc[2];
    auto operand = [&](int i) {
#pragma unroll
        for (int q = 0; q < PW; ++q) fa[i & 1][q] = *reinterpret_cast<const bf16x8*>(a + (q * MT + i) * 1024 + op);
        if constexpr (!PROD) sc[i & 1] = *reinterpret_cast<const f32x4*>(s + 16 * i + 4 * (lane >> 4));
    };
    operand(0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if (i + 1 < MT) operand(i + 1);
        f32x4 part[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) part[c] = PROD ? acc[i][c] : f32x4{0.f, 0.f, 0.f, 0.f};
        // smallest products first
#pragma unroll
        for (int qx = PX - 1; qx >= 0; --qx)
#pragma unroll
            for (int qw = PW - 1; qw >= 0; --qw) {
                if (qx + qw > 2) continue;
#pragma unroll
                for (int c = 0; c < CT; ++c)
                    part[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i & 1][qw], __builtin_bit_cast(bf16x8, fb[c][qx]),
                                                                      part[c], 0, 0, 0);
            }
        if constexpr (PROD) {
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[i][c] = part[c];
        } else {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][c][e] = fmaf(sc[i & 1][e], part[c][e], acc[i][c][e]);
            // (here and now: put off to the step's end, the tiles' sums would fill the registers)
#pragma unroll
            for (int c = 0; c < CT; ++c) asm volatile("" : "+v"(acc[i][c]));
        }
    }
}

template <bool PROD, int MT, int CT>
__device__ __forceinline__ void store_tiles(float* out, int ldo, int M, int N, int m0, int n0, int lane, const f32x4 (&acc)[MT][CT]) {
    const int n = n0 + CT * (lane & 15);
    if (n >= N) return;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = m0 + 16 * i + 4 * (lane >> 4) + e;
            if (m >= M) continue;
            float* dst = out + (size_t)m * ldo + n;
            float v[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) v[c] = PROD ? acc[i][c][e] : acc[i][c][e] * GROW;
            if (n + CT <= N) {
                if constexpr (CT == 2) *reinterpret_cast<f32x2_any*>(dst) = f32x2_any{v[0], v[1]};
                else *reinterpret_cast<f32x4_any*>(dst) = f32x4_any{v[0], v[1], v[2], v[3]};
            } else
#pragma unroll
                for (int c = 0; c < CT - 1; ++c)
                    if (n + c < N) dst[c] = v[c];
        }
}

template <bool PROD, typename T, int MT, typename OFF>
__global__ __launch_bounds__(256, 2) void dict4_many_kernel(ManyParams p) {
    constexpr int PX = COLUMN_PIECES<T>, CT = COLUMN_TILES<T>;
    constexpr int PW = PROD ? 2 : 1;                   // pieces of the weights
    constexpr int ROWS = PW * 16 * MT, STAGE = ROWS * 64;
    constexpr int SROWS = PROD ? 0 : (16 * MT + 63) / 64 * 64;
    extern __shared__ __align__(16) char lds[];       // [2][STAGE], then float [2][SROWS]
    float* lscale = (float*)(lds + 2 * STAGE);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // row tiles of the same columns follow each other on one XCD
    const int at = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (at >= p.tiles) return;
    const int m0 = (at % p.tiles_m) * 16 * MT, n0 = (at / p.tiles_m) * 64 * CT + wave * 16 * CT;
    const int kbeg = blockIdx.y * p.k_per_split, kend = min(p.K, kbeg + p.k_per_split);
    const int steps = (kend - kbeg + BK - 1) / BK;

    // 16 rows of weights a load: a base for the wave and 32 bits a lane (rows behind the last one are the last one)
    constexpr int LOADS = (ROWS / 16 + 3) / 4;
    const char* base[LOADS];
    uint32_t off[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int row = (j * 4 + wave) * 16, piece = row / (16 * MT);
        const int first = min(m0 + row - piece * 16 * MT, p.M - 1);
        base[j] = (const char*)(p.A + ((size_t)piece * p.M + first) * p.kp);
        off[j] = (uint32_t)(min(first + (lane >> 2), p.M - 1) - first) * (uint32_t)p.kp * 2 + (((lane & 3) ^ ((lane >> 4) & 3)) * 16);
    }
    const uint32_t soff = PROD ? 0 : (uint32_t)min(m0 + t, p.M - 1) * 4;
    auto fetch_a = [&](int k, int buf) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            if (ROWS % 64 == 0 || (j * 4 + wave) * 16 < ROWS)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base[j] + (size_t)k * 2 + off[j]),
                                                 (__attribute__((address_space(3))) void*)(lds + buf * STAGE + (j * 4 + wave) * 1024),
                                                 16, 0, 0);
        if constexpr (!PROD)
            if (wave * 64 < 16 * MT)               // (by way of a register the wave would wait for it here)
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void*)((const char*)(p.S + (size_t)(k / p.group) * p.M) + soff),
                    (__attribute__((address_space(3))) void*)(lscale + buf * SROWS + wave * 64), 4, 0, 0);
    };
    Columns<T, OFF> x(p.X, p.N, p.K, p.ldx, lane);
    uint4 fb[CT][PX];
    f32x4 acc[MT][CT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    x.place(n0, lane);
    fetch_a(kbeg, 0);
    x.fetch(kbeg);
    x.split(fb);
    for (int s = 0; s < steps; ++s) {
        const int buf = s & 1, k = kbeg + s * BK;
        // (this step's weights have come - a barrier by itself waits for no load to LDS, and that the columns' loads, sent behind
        // them, were waited for is the compiler's choice - and all waves are done with the last step's)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < steps) {
            fetch_a(k + BK, buf ^ 1);
            x.fetch(k + BK);
        }
        row_tiles<PROD, MT>(lds + buf * STAGE, lscale + buf * SROWS, lane, fb, acc);
        if (s + 1 < steps) x.split(fb);
    }
    if (p.slab) store_tiles<PROD>(p.slab + (size_t)blockIdx.y * p.M * p.N, p.N, p.M, p.N, m0, n0, lane, acc);
    else store_tiles<PROD>(p.out, p.ldo, p.M, p.N, m0, n0, lane, acc);
}

// The same for a contraction so short that a workgroup keeps all its rows' weights in LDS: it unpacks them there itself, and
// its four waves take one set of columns after the other past them, each at its own pace, the next step's columns on
// their way.  One launch, no workspace.  (W H float32 d=1200 r=100 b=8192 22 us, 39 MB of results; laid out
// first and multiplied in a second launch 26.)
struct ResidentParams {
    const uint32_t *codes, *scales;
    const void* X;
    float* out;
    int M, N, K, d, r;
    int ldx, ldo, group, groups;
    int tiles_m, parts;
};
template <bool PROD, typename T, int MT, typename OFF>
__global__ __launch_bounds__(256, 2) void dict4_resident_kernel(ResidentParams p) {
    constexpr int PX = COLUMN_PIECES<T>, CT = COLUMN_TILES<T>, PW = PROD ? 2 : 1, ROWS = 16 * MT, STAGE = PW * ROWS * 64;
    extern __shared__ __align__(16) char lds[];       // [step][piece][row][32 values], then float [group][row]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // row tiles of the same columns follow each other on one XCD
    const int at = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (at >= p.tiles_m * p.parts) return;
    const int m0 = at % p.tiles_m * ROWS, part = at / p.tiles_m;
    const int steps = (p.K + BK - 1) / BK, words = p.groups * (p.group / 8);
    float* lscale = (float*)(lds + steps * STAGE);
    // a value's place: chunks of 8 are permuted by the row, as above
    auto cell = [&](int piece, int row, int k) {
        return lds + (k / BK) * STAGE + (piece * ROWS + row) * 64 + ((((k & 31) >> 3) ^ ((row >> 2) & 3)) * 16) + (k & 7) * 2;
    };
    if constexpr (PROD) {
        // words of four atoms: eight rows, turned round
        for (int e = t; e < steps * 8 * 2 * MT; e += 256) {
            const int w = m0 / 8 + e % (2 * MT), k = e / (2 * MT) * 4;
            float v[4][8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool there = k + j < p.r && w < words;
                const uint32_t sc = there ? p.scales[(size_t)(k + j) * p.groups + w * 8 / p.group] : 0;
                word_entries(there ? p.codes[(size_t)(k + j) * words + w] : 0, v[j]);
#pragma unroll
                for (int f = 0; f < 8; ++f) v[j][f] = word_scale(sc) * (v[j][f] + word_offset(sc));
            }
#pragma unroll
            for (int f = 0; f < 8; ++f) {
                const uint32_t a = pack_bf16(v[0][f], v[1][f]), b = pack_bf16(v[2][f], v[3][f]);
                const int row = e % (2 * MT) * 8 + f;
                *reinterpret_cast<uint2*>(cell(0, row, k)) = make_uint2(a, b);
                *reinterpret_cast<uint2*>(cell(1, row, k)) = make_uint2(pack_bf16(v[0][f] - bf16_lo(a), v[1][f] - bf16_hi(a)),
                                                                         pack_bf16(v[2][f] - bf16_lo(b), v[3][f] - bf16_hi(b)));
            }
        }
    } else {
        for (int e = t; e < ROWS * steps * 4; e += 256) {
            const int row = e / (steps * 4), w = e % (steps * 4), k = m0 + row;
            uint32_t u[4] = {0, 0, 0, 0};
            if (k < p.r) {
                const uint32_t sc = p.scales[(size_t)k * p.groups + w * 8 / p.group];
                const float z = word_offset(sc) * SHRINK;
                float q[8];
                word_entries(p.codes[(size_t)k * words + w], q);
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = w * 8 + j < p.d ? fmaf(q[j], SHRINK, z) : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = pack_bf16(q[2 * j], q[2 * j + 1]);
                if (w * 8 % p.group == 0) lscale[w * 8 / p.group * ROWS + row] = word_scale(sc);
            }
            *reinterpret_cast<uint4*>(cell(0, row, w * 8)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
    __syncthreads();
    const int sets = (p.N + 16 * CT - 1) / (16 * CT), stride = p.parts * 4;
    int set = part * 4 + wave;
    if (set >= sets) return;
    Columns<T, OFF> x(p.X, p.N, p.K, p.ldx, lane);
    x.place(set * 16 * CT, lane);
    x.fetch(0);
    for (; set < sets; set += stride) {
        f32x4 acc[MT][CT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < steps; ++s) {
            uint4 fb[CT][PX];
            x.split(fb);
            if (s + 1 < steps) {
                x.fetch((s + 1) * BK);
            } else if (set + stride < sets) {
                x.place((set + stride) * 16 * CT, lane);
                x.fetch(0);
            }
            row_tiles<PROD, MT>(lds + s * STAGE, lscale + s * BK / p.group * ROWS, lane, fb, acc);
        }
        store_tiles<PROD>(p.out, p.ldo, p.M, p.N, m0, set * 16 * CT, lane, acc);
    }
}

// ------------------------------------------------------------------------------------------- launches
constexpr int MOST_COLS = 2147483647 - 1024;    // tile arithmetic in int
constexpr int FEW_PRODUCT = 2;              // columns up to which the product's vector kernel runs
// ... and the tile kernels, a block of columns in the grid for every 32 (product) or 64.  With more columns the weights
// are better laid out once (us, tile and many columns' kernels: W H, d=8192 r=16384 b=192 340 and 507, b=1000 1337
// and 1270, d=1024 r=1024 b=512 18.6 and 27.6; W^T X, float32, d=8192 r=16384 b=128 173 and 222, b=256 420 and
// 314, d=4096 r=256 b=384 16.6 and 21.4, bfloat16, d=8192 r=16384 b=512 413 and 461).
constexpr int TILE_PRODUCT = 1024;
constexpr size_t RESIDENT_BYTES = 150 * 1024;
int most_tile_columns(int d, int r, bool wide) { return !wide || (long long)d * r <= 1 << 20 ? 512 : 192; }     // (the correlate's)

// words a lane of the vector kernels: one segment is enough with narrower lanes where there are few features
int words_a_lane(int d) { return d <= 512 ? 1 : d <= 1024 ? 2 : 4; }
// The vector kernel's split of the atoms.  Up to 512 atoms one workgroup of 16 waves takes them all, in one launch
// with nothing to add up behind it.
struct FewProduct { bool one; int ch, segs, splits, per; };
FewProduct product_few_plan(int d, int r) {
    FewProduct q;
    q.one = r <= 512;
    q.ch = q.one ? 1 : words_a_lane(d);
    q.segs = (d + 512 * q.ch - 1) / (512 * q.ch);
    const int splits = q.one ? 1 : std::max(1, std::min(1024 / q.segs, r / 128));      // 32 atoms a wave at least
    q.per = ((r + splits - 1) / splits + 31) / 32 * 32;
    q.splits = (r + q.per - 1) / q.per;
    return q;
}
// Rows of a workgroup's tile (in sixteens) and pieces of the contraction for a product with many columns: the pair with
// the least time by a model of what a step of 32 was measured to take with w workgroups a CU - 0.45 to 0.6 us until its
// loads have come, for every set of workgroups that are resident together, and for every sixteen rows (and one for the
// columns' split) 0.05 to 0.09 us of matrix and vector instructions - and of the pieces' way through memory at
// 4 TB/s.  (W^T X, d=6492 r=9202 b=73 float32: tiles of 32, 64, 128, 256 rows in one piece 237, 194, 236, 382 us, in
// pieces for two workgroups a CU 142, 98, 91, 119.)
struct ManyPlan { int mt, tiles_m, tiles_n, splits, per; size_t a_bytes, s_bytes, slab_bytes; double cost; };
ManyPlan many_plan(bool prod, int d, int r, int b, int group, bool wide) {
    ManyPlan q;
    const int M = prod ? d : r;
    const int kp = prod ? (r + BK - 1) / BK * BK : (d + group - 1) / group * group;
    const int steps = ((prod ? r : d) + BK - 1) / BK;
    const int cols = 64 * (wide ? COLUMN_TILES<float> : COLUMN_TILES<uint16_t>);
    q.tiles_n = (b + cols - 1) / cols;
    double best = -1;
    for (int mt = prod || !wide ? 8 : 16; mt >= 2; mt /= 2) {       // (what LDS and the registers hold)
        const int tiles_m = (M + 16 * mt - 1) / (16 * mt), resident = mt == 16 || (mt == 8 && !wide) ? 2 : mt == 8 || !wide ? 3 : 4;
        const double tiles = (double)tiles_m * q.tiles_n;
        const double row = prod ? (wide ? 0.09 : 0.085) : (wide ? 0.07 : 0.05), own = wide ? 0.6 : 0.45;
        for (int target = 0; target <= 1024; target += 256) {
            const int want = (int)std::max(1.0, std::min(target / tiles, steps / 2.0));
            const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
            const double w = std::ceil(tiles * splits / 256);
            // (256 rows alone on the chip: 0.01 more; with other sets behind it the columns that it saves count as much)
            const double each = row + (mt == 16 && w <= 2 ? 0.01 : 0.0);
            double cost = per * (own * std::ceil(w / resident) + each * w * (mt + 1));
            if (splits > 1) cost += 3.0 + 2e-6 * splits * M * b;
            if (best >= 0 && cost >= best) continue;
            best = q.cost = cost;
            q.mt = mt;
            q.tiles_m = tiles_m;
            q.per = per;
            q.splits = splits;
        }
    }
    q.a_bytes = ((size_t)(prod ? 2 : 1) * M * kp * 2 + 255) & ~(size_t)255;
    q.s_bytes = prod ? 0 : ((size_t)(kp / group) * r * sizeof(float) + 255) & ~(size_t)255;
    q.slab_bytes = q.splits > 1 ? (size_t)q.splits * M * b * sizeof(float) : 0;
    return q;
}

int add_slabs(onmf_ctx* c, size_t mn, int N, int splits, const float* slab, float* out, int ldo, hipStream_t s) {
    hipLaunchKernelGGL(dict4_reduce_kernel, dim3((unsigned)std::min<size_t>((mn + 63) / 64, 16384)), dim3(256), 0, s, mn, N,
                       splits, slab, out, ldo);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

template <int CH, typename T>
int correlate_one(onmf_ctx* c, int d, int r, int group, const uint32_t* codes, const uint32_t* scales, const T* X, int ldx,
                  float* C, hipStream_t s) {
    constexpr int AT = 4, SEG = 512 * CH;
    const int segs = (d + SEG - 1) / SEG, groups = (d + group - 1) / group;
    const int staged = std::min(segs, (int)(65536 / (sizeof(float) * SEG)));
    const int chunks = (r + 4 * AT - 1) / (4 * AT);
    hipLaunchKernelGGL((dict4_correlate_one_kernel<CH, AT, T>), dim3(std::min(chunks, 1024)), dim3(256),
                       sizeof(float) * (size_t)staged * SEG, s, d, r, group, groups, codes, scales, X, ldx, C, staged);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

template <int NB, int CH, int NW, typename T>
int product_few(onmf_ctx* c, const FewProduct& q, int d, int r, int b, int group, const uint32_t* codes,
                const uint32_t* scales, const T* H, int ldh, float* R, int ldr, float* ws, hipStream_t s) {
    float* slab = q.splits > 1 ? ws : nullptr;
    hipLaunchKernelGGL((dict4_product_few_kernel<NB, CH, NW, T>), dim3(q.segs, q.splits), dim3(64 * NW), 0, s, d, r, b, group,
                       (d + group - 1) / group, codes, scales, H, ldh, R, ldr, q.per, slab);
    HIP_TRY(c, hipGetLastError());
    return slab ? add_slabs(c, (size_t)d * b, b, q.splits, slab, R, ldr, s) : ONMF_OK;
}

// The tile kernel's split of the atoms: two workgroups a CU (what its registers allow), 128 atoms (a step of each wave) at least.
struct TilePlan { int nt, cw, blocks, splits, per, zs; };
TilePlan product_tile_plan(int d, int r, int b, int group) {
    TilePlan q;
    q.nt = b <= 16 ? 1 : 2;
    // (two words a lane where there are weights enough, one for half the sums to add up where not: d=441 r=256 b=7
    // 7.6 and 5.4 us, d=8192 r=16384 b=7 37 and 48)
    q.cw = q.nt == 1 && (long long)d * r > 1 << 23 ? 2 : 1;
    q.zs = (b + 16 * q.nt - 1) / (16 * q.nt);
    const int words = (d + group - 1) / group * (group / 8), steps = (r + 127) / 128;
    q.blocks = (words + 16 * q.cw - 1) / (16 * q.cw);
    double best = -1;
    for (int target = 0; target <= 512; target += 256) {
        const int want = std::max(1, std::min(steps, target / (q.blocks * q.zs)));
        const int per = (steps + want - 1) / want, splits = (steps + per - 1) / per;
        const double w = (double)q.blocks * q.zs * splits;
        double cost = std::ceil(w / 512) * per * (w > 256 ? 3.0 : 2.0);
        if (splits > 1) cost += 4.0 + 2.5e-6 * splits * d * b;
        if (best >= 0 && cost >= best) continue;
        best = cost;
        q.per = per * 128;
        q.splits = splits;
    }
    return q;
}
template <int NT, int CW, typename T>
int product_tile(onmf_ctx* c, const TilePlan& q, int d, int r, int b, int group, const uint32_t* codes,
                 const uint32_t* scales, const T* H, int ldh, float* R, int ldr, float* ws, hipStream_t s) {
    constexpr size_t bytes = 4 * 8 * CW * NT * 64 * 4 * sizeof(float);
    static LdsLimit lim;
    ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)dict4_product_tile_kernel<NT, CW, T>, bytes));
    float* slab = q.splits > 1 ? ws : nullptr;
    hipLaunchKernelGGL((dict4_product_tile_kernel<NT, CW, T>), dim3(q.blocks, q.splits, q.zs), dim3(256), bytes, s, d, r, b, group,
                       (d + group - 1) / group, codes, scales, H, ldh, R, ldr, q.per, slab);
    HIP_TRY(c, hipGetLastError());
    return slab ? add_slabs(c, (size_t)d * b, b, q.splits, slab, R, ldr, s) : ONMF_OK;
}

// The correlate's tile kernel: a workgroup a CU, ranges of features that fit in its LDS and more of them (down to
// 128 features) where there are not atoms enough.  `one`: little enough for the kernel with one launch, whose
// workgroups take 1.2 us for 16 steps of 32 features and 16 columns (float32, three columns, us, one launch and ranges:
// d=441 r=72 3.5 and 7.4, d=1024 r=4096 5.4 and 11.6, d=1024 r=16384 15.0 and 11.9, d=8192 r=72 21.4 and 10.8).
struct RangePlan { bool one; int nt, per, splits, parts, zs; };
RangePlan correlate_tile_plan(int d, int r, int b, bool wide) {
    RangePlan q;
    q.nt = b <= 16 ? 1 : b <= 32 ? 2 : 4;
    q.zs = (b + 16 * q.nt - 1) / (16 * q.nt);
    const int blocks = (d + 127) / 128, most = 144 * 1024 / (4 * 1024 * q.nt * (wide ? 3 : 1)), waves = (r + 255) / 256;
    q.one = b <= 64 && d <= 4096 / q.nt && (long long)((d + 31) / 32) * ((r + 15) / 16) <= 16384;
    const int least = (blocks + most - 1) / most;
    const int want = std::max(least, std::min(256 / (waves * q.zs), blocks));
    const int each = (blocks + want - 1) / want;
    q.per = each * 128;
    q.splits = (blocks + each - 1) / each;
    q.parts = std::max(1, std::min(waves, 256 / (q.splits * q.zs)));
    return q;
}
template <int NT, typename T>
int correlate_wave(onmf_ctx* c, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales, const T* X, int ldx,
                   float* C, hipStream_t s) {
    const dim3 grid((r + 15) / 16);
    const int groups = (d + group - 1) / group;
    if (d <= 256)
        hipLaunchKernelGGL((dict4_correlate_wave_kernel<NT, 4, T>), grid, dim3(256), 0, s, d, r, b, group, groups, codes, scales,
                           X, ldx, C);
    else
        hipLaunchKernelGGL((dict4_correlate_wave_kernel<NT, 16, T>), grid, dim3(1024), 0, s, d, r, b, group, groups, codes, scales,
                           X, ldx, C);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}
template <int NT, typename T>
int correlate_tile(onmf_ctx* c, const RangePlan& q, int d, int r, int b, int group, const uint32_t* codes,
                   const uint32_t* scales, const T* X, int ldx, float* C, float* ws, hipStream_t s) {
    const size_t bytes = (size_t)q.per / 32 * NT * (sizeof(T) == 4 ? 3 : 1) * 1024;
    static LdsLimit lim;
    ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)dict4_correlate_tile_kernel<NT, T>, bytes));
    float* slab = q.splits > 1 ? ws : nullptr;
    hipLaunchKernelGGL((dict4_correlate_tile_kernel<NT, T>), dim3(q.parts, q.splits, q.zs), dim3(512), bytes, s, d, r, b, group,
                       (d + group - 1) / group, codes, scales, X, ldx, C, q.per, slab);
    HIP_TRY(c, hipGetLastError());
    return slab ? add_slabs(c, (size_t)r * b, b, q.splits, slab, C, b, s) : ONMF_OK;
}

template <bool PROD, typename T>
int many(onmf_ctx* c, const ManyPlan& q, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales, const T* X, int ldx,
         float* out, int ldo, char* ws, hipStream_t s) {
    const int groups = (d + group - 1) / group, words = groups * (group / 8);
    ManyParams p;
    p.A = (const uint16_t*)ws;
    p.S = (const float*)(ws + q.a_bytes);
    p.slab = q.splits > 1 ? (float*)(ws + q.a_bytes + q.s_bytes) : nullptr;
    p.X = X; p.out = out; p.ldx = ldx; p.ldo = ldo; p.group = group;
    p.M = PROD ? d : r; p.N = b; p.K = PROD ? r : d;
    p.kp = PROD ? (r + BK - 1) / BK * BK : words * 8;
    p.tiles_m = q.tiles_m; p.tiles = q.tiles_m * q.tiles_n; p.k_per_split = q.per * BK;
    if constexpr (PROD)
        hipLaunchKernelGGL(dict4_lay_product_kernel, dim3((p.kp + 63) / 64, (words + 15) / 16), dim3(256), 0, s, d, r, words, group,
                           groups, p.kp, codes, scales, (uint16_t*)ws);
    else
        hipLaunchKernelGGL(dict4_lay_correlate_kernel, dim3((unsigned)std::min<size_t>(((size_t)r * words + 255) / 256, 8192)),
                           dim3(256), 0, s, d, r, words, group, groups, codes, scales, (uint4*)ws, (float*)(ws + q.a_bytes));
    HIP_TRY(c, hipGetLastError());
    const dim3 grid((p.tiles + 7) / 8 * 8, q.splits);
    const bool near = ((size_t)BK * ldx + b) * sizeof(T) < ((size_t)1 << 32);
#define MANY_CASE(MT)                                                                                                    \
    if (q.mt == MT) {                                                                                                    \
        const size_t bytes = 2 * ((PROD ? 2 : 1) * 16 * MT * 64 + (PROD ? 0 : (16 * MT + 63) / 64 * 64 * sizeof(float)));  \
        if (near) hipLaunchKernelGGL((dict4_many_kernel<PROD, T, MT, uint32_t>), grid, dim3(256), bytes, s, p);          \
        else hipLaunchKernelGGL((dict4_many_kernel<PROD, T, MT, uint64_t>), grid, dim3(256), bytes, s, p);               \
    }
    if constexpr (!PROD && sizeof(T) == 4) { MANY_CASE(16) }
    MANY_CASE(8) MANY_CASE(4) MANY_CASE(2)
#undef MANY_CASE
    HIP_TRY(c, hipGetLastError());
    if (p.slab) return add_slabs(c, (size_t)p.M * p.N, p.N, q.splits, p.slab, p.out, p.ldo, s);
    return ONMF_OK;
}

// Rows of a resident workgroup's tile, or none where the two launches of the many columns' kernel take less by their model
// (with 8 us for the first of them and its latency, the weights' way at 4 TB/s and the result's at 8).  A step takes
// a wave `own` and `row` for every sixteen rows, half as long again with two workgroups a CU; before that come the
// launch and the unpacking.  (us, resident and many: W H float32 d=1200 r=100 b=8192 22 and 25.5, d=1024 r=256
// b=2000 13.3 and 18.4, b=60000 170 and 153; bfloat16 d=441 r=100 b=5001 8.7 and 13.6; W^T X bfloat16 d=441 r=100
// b=16384 12.4 and 16.6, float32 d=1024 r=256 b=520 24 and 16.)
struct ResidentPlan { int mt, tiles_m, parts; size_t bytes; };
ResidentPlan resident_plan(const ManyPlan& many, bool prod, int d, int r, int b, int group, bool wide) {
    ResidentPlan q;
    q.mt = 0;
    const int M = prod ? d : r, K = prod ? r : d, steps = (K + BK - 1) / BK;
    const int cols = 16 * (wide ? COLUMN_TILES<float> : COLUMN_TILES<uint16_t>);
    const int sets = (b + cols - 1) / cols;
    const double own = wide ? (prod ? 0.5 : 0.35) : 0.26, row = prod && !wide ? 0.16 : 0.145;
    double best = many.cost + 8.0 + (prod ? 4.5 : 2.5) * d * r / 4e6 + 4.0 * M * b / 8e6;
    for (int mt = wide ? 8 : 4; mt >= 2; mt /= 2) {            // (what the registers hold)
        const size_t scale_bytes = prod ? 0 : sizeof(float) * ((steps * BK + group - 1) / group) * 16 * mt;
        const size_t bytes = (size_t)steps * (prod ? 2 : 1) * 16 * mt * 64 + scale_bytes;
        if (bytes > RESIDENT_BYTES) continue;
        const int tiles_m = (M + 16 * mt - 1) / (16 * mt), resident = bytes > RESIDENT_BYTES / 2 ? 1 : 2;
        const double waves = (double)sets * tiles_m, step = (own + row * mt) * (waves > 1024 && resident == 2 ? 1.5 : 1.0);
        const double cost = 3.5 + bytes / 40e3 + std::ceil(waves / (1024 * resident)) * steps * step;
        if (cost >= best) continue;
        best = cost;
        q.mt = mt;
        q.bytes = bytes;
        q.tiles_m = tiles_m;
        q.parts = std::min((sets + 3) / 4, std::max(1, 256 * resident / tiles_m));
    }
    return q;
}
template <bool PROD, typename T>
int resident(onmf_ctx* c, const ResidentPlan& q, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales,
             const T* X, int ldx, float* out, int ldo, hipStream_t s) {
    ResidentParams p;
    p.codes = codes; p.scales = scales; p.X = X; p.out = out; p.ldx = ldx; p.ldo = ldo; p.group = group;
    p.groups = (d + group - 1) / group; p.d = d; p.r = r;
    p.M = PROD ? d : r; p.N = b; p.K = PROD ? r : d; p.tiles_m = q.tiles_m; p.parts = q.parts;
    const dim3 grid((q.tiles_m * q.parts + 7) / 8 * 8);
    const bool near = ((size_t)BK * ldx + b) * sizeof(T) < ((size_t)1 << 32);
#define RESIDENT_CASE(MT, OFF)                                                                                           \
    {                                                                                                                    \
        static LdsLimit lim;                                                                                             \
        ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)dict4_resident_kernel<PROD, T, MT, OFF>, q.bytes));            \
        hipLaunchKernelGGL((dict4_resident_kernel<PROD, T, MT, OFF>), grid, dim3(256), q.bytes, s, p);                     \
    }
#define RESIDENT_CASES(MT) if (q.mt == MT) { if (near) RESIDENT_CASE(MT, uint32_t) else RESIDENT_CASE(MT, uint64_t) }
    if constexpr (sizeof(T) == 4) { RESIDENT_CASES(8) }
    RESIDENT_CASES(4) RESIDENT_CASES(2)
#undef RESIDENT_CASES
#undef RESIDENT_CASE
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

int check4(onmf_ctx* c, const char* what, int d, int r, int group, const void* codes, const void* scales) {
    if (d <= 0 || r <= 0 || !codes || !scales || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3))
        return onmf_fail(c, ONMF_ERR_ARG, "%s: bad arguments (d=%d r=%d; codes must be aligned to 16 bytes)", what, d, r);
    if (group != 32 && group != 64 && group != 128)
        return onmf_fail(c, ONMF_ERR_ARG, "%s: a group is 32, 64 or 128 features, not %d", what, group);
    if (d > (1 << 18) || r > MOST_COLS)
        return onmf_fail(c, ONMF_ERR_ARG, "%s: d=%d is more than 2^18 features, or r=%d more atoms than an int counts", what, d, r);
    return ONMF_OK;
}

size_t workspace_of(bool prod, int d, int r, int b, int group, bool wide) {
    int splits = 1;
    if (prod && b <= FEW_PRODUCT) splits = product_few_plan(d, r).splits;
    else if (prod && b <= TILE_PRODUCT) splits = product_tile_plan(d, r, b, group).splits;
    else if (!prod && b == 1) splits = 1;
    else if (!prod && b <= most_tile_columns(d, r, wide)) {
        const RangePlan q = correlate_tile_plan(d, r, b, wide);
        splits = q.one ? 1 : q.splits;
    } else {
        const ManyPlan q = many_plan(prod, d, r, b, group, wide);
        if (!resident_plan(q, prod, d, r, b, group, wide).mt) return q.a_bytes + q.s_bytes + q.slab_bytes;
    }
    return splits > 1 ? (size_t)splits * (prod ? d : r) * b * sizeof(float) : 0;
}

template <typename T>
int correlate_t(onmf_ctx* c, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales, const T* X,
                int ldx, float* C, float* ws, hipStream_t s) {
    if (b == 1) {
        const int ch = words_a_lane(d);
        if (ch == 1) return correlate_one<1, T>(c, d, r, group, codes, scales, X, ldx, C, s);
        if (ch == 2) return correlate_one<2, T>(c, d, r, group, codes, scales, X, ldx, C, s);
        return correlate_one<4, T>(c, d, r, group, codes, scales, X, ldx, C, s);
    }
    if (b <= most_tile_columns(d, r, sizeof(T) == 4)) {
        const RangePlan q = correlate_tile_plan(d, r, b, sizeof(T) == 4);
        if (q.one && q.nt == 1) return correlate_wave<1, T>(c, d, r, b, group, codes, scales, X, ldx, C, s);
        if (q.one && q.nt == 2) return correlate_wave<2, T>(c, d, r, b, group, codes, scales, X, ldx, C, s);
        if (q.one) return correlate_wave<4, T>(c, d, r, b, group, codes, scales, X, ldx, C, s);
        if (q.nt == 1) return correlate_tile<1, T>(c, q, d, r, b, group, codes, scales, X, ldx, C, ws, s);
        if (q.nt == 2) return correlate_tile<2, T>(c, q, d, r, b, group, codes, scales, X, ldx, C, ws, s);
        return correlate_tile<4, T>(c, q, d, r, b, group, codes, scales, X, ldx, C, ws, s);
    }
    const ManyPlan m = many_plan(false, d, r, b, group, sizeof(T) == 4);
    const ResidentPlan q = resident_plan(m, false, d, r, b, group, sizeof(T) == 4);
    if (q.mt) return resident<false, T>(c, q, d, r, b, group, codes, scales, X, ldx, C, b, s);
    return many<false, T>(c, m, d, r, b, group, codes, scales, X, ldx, C, b, (char*)ws, s);
}

template <typename T>
int product_t(onmf_ctx* c, int d, int r, int b, int group, const uint32_t* codes, const uint32_t* scales, const T* H,
              int ldh, float* R, int ldr, float* ws, hipStream_t s) {
    if (b <= FEW_PRODUCT) {
        const FewProduct q = product_few_plan(d, r);
#define FEW_CASE(NB, CH) \
    if (b <= NB && q.ch == CH && !q.one) return product_few<NB, CH, 4, T>(c, q, d, r, b, group, codes, scales, H, ldh, R, ldr, ws, s)
        if (q.one && b == 1) return product_few<1, 1, 16, T>(c, q, d, r, b, group, codes, scales, H, ldh, R, ldr, ws, s);
        if (q.one) return product_few<2, 1, 16, T>(c, q, d, r, b, group, codes, scales, H, ldh, R, ldr, ws, s);
        FEW_CASE(1, 1); FEW_CASE(1, 2); FEW_CASE(1, 4); FEW_CASE(2, 1); FEW_CASE(2, 2); FEW_CASE(2, 4);
#undef FEW_CASE
    }
    if (b <= TILE_PRODUCT) {
        const TilePlan q = product_tile_plan(d, r, b, group);
        if (q.nt == 1 && q.cw == 1) return product_tile<1, 1, T>(c, q, d, r, b, group, codes, scales, H, ldh, R, ldr, ws, s);
        if (q.nt == 1) return product_tile<1, 2, T>(c, q, d, r, b, group, codes, scales, H, ldh, R, ldr, ws, s);
        return product_tile<2, 1, T>(c, q, d, r, b, group, codes, scales, H, ldh, R, ldr, ws, s);
    }
    const ManyPlan m = many_plan(true, d, r, b, group, sizeof(T) == 4);
    const ResidentPlan q = resident_plan(m, true, d, r, b, group, sizeof(T) == 4);
    if (q.mt) return resident<true, T>(c, q, d, r, b, group, codes, scales, H, ldh, R, ldr, s);
    return many<true, T>(c, m, d, r, b, group, codes, scales, H, ldh, R, ldr, (char*)ws, s);
}

}  // namespace

extern "C" {

size_t onmf_dict4_workspace(int which, int d, int r, int b, int group) {
    if (d <= 0 || r <= 0 || b <= 0 || (group != 32 && group != 64 && group != 128)) return 0;
    if (d > (1 << 18) || r > MOST_COLS || b > MOST_COLS) return 0;              // sizes that the calls refuse
    size_t need = 0;                                    // enough for either type of the columns
    for (const bool wide : {false, true}) need = std::max(need, workspace_of(which == ONMF_DICT4_PRODUCT, d, r, b, group, wide));
    return need;
}

int onmf_dict4_pack(onmf_ctx* c, int d, int r, int group, const float* W, void* codes, int32_t* scales, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check4(c, "dict4_pack", d, r, group, codes, scales));
    if (!W) return onmf_fail(c, ONMF_ERR_ARG, "dict4_pack: W is null");
    ONMF_ENTER(c);
    const int groups = (d + group - 1) / group;
    const dim3 grid((r + 63) / 64, groups);
    const auto kernel = group == 128 ? dict4_pack_kernel<128> : group == 64 ? dict4_pack_kernel<64> : dict4_pack_kernel<32>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, d, r, groups, W, (uint32_t*)codes, (uint32_t*)scales);
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
    hipLaunchKernelGGL(dict4_unpack_kernel, dim3((r + 255) / 256, (d + 31) / 32), dim3(256), 0, (hipStream_t)stream, d, r, group,
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
    const size_t need = workspace_of(false, d, r, b, group, x_type == T_F32);
    if (ws_bytes < need || (need && !ws) || ((uintptr_t)ws & 15))
        return onmf_fail(c, ONMF_ERR_ARG, "dict4_correlate: workspace of %zu bytes, %zu needed, aligned to 16", ws_bytes, need);
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
    const size_t need = workspace_of(true, d, r, b, group, h_type == T_F32);
    if (ws_bytes < need || (need && !ws) || ((uintptr_t)ws & 15))
        return onmf_fail(c, ONMF_ERR_ARG, "dict4_product: workspace of %zu bytes, %zu needed, aligned to 16", ws_bytes, need);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const uint32_t *cw = (const uint32_t*)codes, *sc = (const uint32_t*)scales;
    return h_type == T_F32 ? product_t<float>(c, d, r, b, group, cw, sc, (const float*)H, ldh, R, ldr, (float*)ws, s)
                           : product_t<uint16_t>(c, d, r, b, group, cw, sc, (const uint16_t*)H, ldh, R, ldr, (float*)ws, s);
}

}  // extern "C"
