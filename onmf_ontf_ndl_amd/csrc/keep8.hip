// Columns held in 8 bits and what the dictionary's update needs of them, on gfx950.
//
// Format: 128 consecutive columns of a row share a scale s = max |v| / 127 (float32, by the reciprocal of 127, as float
// arrays are divided by a number on the GPU); an entry stands for s q, q = rint(v / s) in -127..127.  codes is
// [row][padded columns] int8 (rows padded to whole groups with zeros), scales [row][group].  A minibatch X and its code H
// put away this way take a quarter of their room, and the sums H H^T and H X^T - the gradient to the dictionary is
// W (H H^T) - X H^T - run on the 8-bit matrix pipe: inside a group the products of whole numbers add up exactly in int32.
#include "common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef double f64x2_any __attribute__((ext_vector_type(2), aligned(8)));
// rows of any length: vectors that need no more alignment than their entries (the memory pipe takes them as they lie)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

namespace {

constexpr int GROUP = 128;
constexpr size_t MOST_GROUPS = ((size_t)1 << 29) - 32;      // eight threads a group, fewer than 2^32 in a launch
constexpr int MOST_COLS = 1 << 28;       // eight rows' codes lie within 32 bits
constexpr int MOST_ROWS = 2147483647 - 1024;    // tile arithmetic in int

__device__ __forceinline__ float bf16_to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float load_val(const float* p) { return *p; }
__device__ __forceinline__ float load_val(const uint16_t* p) { return bf16_to_f32(*p); }

// ------------------------------------------------------------------------------------------- put away
// Whole q nearest to v / s with ties to even, decided exactly: the remainder v - s q is a multiple of half an
// ulp of s and below 2^24 of them, so the fused multiply-add gives it without rounding and a quotient next to
// a half falls on its own side whatever the reciprocal's rounding.
__device__ __forceinline__ float nearest(float v, float s, float q) {
    const float rest = 2.f * fmaf(-q, s, v);
    const bool odd = ((int)q & 1) != 0;
    if (rest > s || (rest == s && odd)) q += 1.f;
    else if (rest < -s || (rest == -s && odd)) q -= 1.f;
    return q;
}

// the largest value of 16 lanes, in all of them
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));      // lanes 1 apart
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));      // 2
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));     // the halves of 8
    return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));  // the halves of 16
}

// row and group of the first of the groups a thread handles, moved on one at a time (one division a thread)
struct GroupAt {
    uint32_t row, g, groups;
    __device__ __forceinline__ GroupAt(uint32_t at, uint32_t n) : row(at / n), g(at % n), groups(n) {}
    __device__ __forceinline__ void next() { if (++g == groups) { g = 0; ++row; } }
};

// 16 lanes per group, eight columns a lane, U groups a lane (their loads are on their way together).  Bound by
// memory: 5 bytes a float32 entry, 3 a bfloat16 one (1024 x 65536: float32 60 us, 5.6 TB/s, bfloat16 43, 4.7).
template <typename T, int U>
__global__ __launch_bounds__(256) void keep8_kernel(size_t all, int n, int groups, const T* __restrict__ X, int ldx,
                                                     int8_t* __restrict__ codes, float* __restrict__ scales) {
    const int lane = threadIdx.x & 15;
    const size_t first = ((size_t)blockIdx.x * 16 + (threadIdx.x >> 4)) * U;
    if (first >= all) return;
    GroupAt at((uint32_t)first, (uint32_t)groups);
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u, at.next()) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u][j] = 0.f;
        if (first + u >= all) continue;
        const int c = (int)at.g * GROUP + lane * 8;
        const T* src = X + (size_t)at.row * ldx + c;
        if (c + 7 < n) {
            if constexpr (sizeof(T) == 4) {
                const f32x4_any f = reinterpret_cast<const f32x4_any*>(src)[0], h = reinterpret_cast<const f32x4_any*>(src)[1];
                v[u][0] = f.x; v[u][1] = f.y; v[u][2] = f.z; v[u][3] = f.w;
                v[u][4] = h.x; v[u][5] = h.y; v[u][6] = h.z; v[u][7] = h.w;
            } else {
                const u32x4_any p = *reinterpret_cast<const u32x4_any*>(src);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[u][2 * j] = __uint_as_float(p[j] << 16);
                    v[u][2 * j + 1] = __uint_as_float(p[j] & 0xffff0000u);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < n) v[u][j] = load_val(src + j);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (first + u >= all) break;
        // the largest magnitude by its bits: a NaN's are above an infinity's, an infinity's above all others
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[u][j]) & 0x7fffffffu);
        most = max16(most);
        float s = __uint_as_float(most) * (1.f / 127.f);
        float q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = 0.f;
        if (most >= 0x7f800000u) {
            s = __uint_as_float(0x7fc00000u);            // a NaN or an infinity: the whole group reads NaN
        } else if (s < 1.17549435e-38f) {
            s = 0.f;                                       // nothing but (next to) zeros
        } else {
            // v times the reciprocal (1 ulp) is within 127 (2^-23 + 2^-24) = 2.3e-5 of the quotient: only where it lies
            // that near to a half is the remainder asked
            const float inv = __builtin_amdgcn_rcpf(s);
            float off = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = v[u][j] * inv;
                q[j] = rintf(f);
                off = fmaxf(off, fabsf(f - q[j]));
            }
            if (off > 0.49997f) {
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = nearest(v[u][j], s, q[j]);
            }
        }
        uint32_t word[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) word[j >> 2] |= ((uint32_t)(int)q[j] & 0xff) << (8 * (j & 3));
        // (a row's groups follow one another in both outputs: group `first + u` of all)
        *reinterpret_cast<uint2*>(codes + (first + u) * GROUP + lane * 8) = make_uint2(word[0], word[1]);
        if (lane == 0) scales[first + u] = s;
    }
}

// ------------------------------------------------------------------------------------------- bring back
// 32 lanes per group, four columns a lane, U groups a lane.  Bound by memory, 5 bytes an entry (1024 x 65536: 60 us,
// 5.6 TB/s).
template <int U>
__global__ __launch_bounds__(256) void keep8_expand_kernel(size_t all, int n, int groups, const int8_t* __restrict__ codes,
                                                            const float* __restrict__ scales, float* __restrict__ X,
                                                            int ldx) {
    const int lane = threadIdx.x & 31;
    const size_t first = ((size_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * U;
    if (first >= all) return;
    uint32_t w[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const size_t at = min(first + u, all - 1);
        w[u] = *reinterpret_cast<const uint32_t*>(codes + at * GROUP + lane * 4);
        s[u] = scales[at];
    }
    GroupAt at((uint32_t)first, (uint32_t)groups);
#pragma unroll
    for (int u = 0; u < U; ++u, at.next()) {
        if (first + u >= all) break;
        const int c = (int)at.g * GROUP + lane * 4;
        const f32x4_any v = {s[u] * (float)(int8_t)(w[u] & 0xff), s[u] * (float)(int8_t)((w[u] >> 8) & 0xff),
                             s[u] * (float)(int8_t)((w[u] >> 16) & 0xff), s[u] * (float)(int8_t)(w[u] >> 24)};
        float* dst = X + (size_t)at.row * ldx + c;
        if (c + 3 < n) {
            *reinterpret_cast<f32x4_any*>(dst) = v;
        } else {
            if (c + 0 < n) dst[0] = v.x;
            if (c + 1 < n) dst[1] = v.y;
            if (c + 2 < n) dst[2] = v.z;
            if (c + 3 < n) dst[3] = v.w;
        }
    }
}

// X[:, j] = column idx[j]; a negative index counts from the end, one out of range reads NaN.  Bound by its reads, a byte
// of every 64 that come (8192 columns at random of 1024 x 65536: 68 us).
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
// Tiles of [H H^T | H X^T], one 128-column group of the contraction a step; a workgroup takes a run of groups and
// writes its sums to a slab.  int32 inside a group (at most 128 * 127^2), float32 over a workgroup's run, double
// over the runs.  PRECISE, for the gradient: double over a run too and in its slab (near a stationary dictionary W (H H^T)
// and X H^T nearly cancel: what is rounded to float32 on the way, a run's sums included, is as large as the gradient).
// A wave owns 16 MI x 16 NJ outputs in 16x16x64 tiles (four of X's scales and one of H's a lane
// and tile: half the scale reads of the 32x32 shape).  The codes go from memory straight to LDS, two groups ahead,
// in rows of 128 bytes whose 16-byte chunks are permuted by (row >> 1) & 7, so that the 16 rows of an operand read
// meet every bank once.  Rows behind the last one read the last row's codes; what they give is not stored.
// In float32 H's scale is multiplied to the whole sum and X's with the addition: the two scales' own product may lie beyond
// what float32 holds where the sum does not, and that would make zeros NaN.
// Per group and output three vector instructions (conversion, product with a scale, fused multiply-add) stand against 1/256 of
// a matrix instruction.  Where memory is not the bound, three pipes are, in turn: of a group of a 128 x 256 tile the operands
// are 192 KB from LDS (0.64 us at 128 B a cycle), 1536 vector instructions (0.64 us) and 8.4 MOP (0.43 us), and all waves pass one
// barrier a group, which was measured to take 1.7 us, their sum (d=4096 r=256 n=65536, 146 GOP: 125 us, PRECISE 145 and the
// slabs' 62 MB; d=1024 40 us).
template <int MI, int NJ, int WM_, int WN_, int STAGES> struct Tile {
    static constexpr int mi = MI, nj = NJ, wm = WM_, wn = WN_, stages = STAGES;
    static constexpr int bm = 16 * MI * WM_, bn = 16 * NJ * WN_, waves = WM_ * WN_;
    static constexpr int rows = (bm + bn + 8 * waves - 1) / (8 * waves) * (8 * waves);     // of a stage: every wave loads as many
    // scales come sg groups at a time, sg lanes to a row (more groups than there are stages: see the waits)
    static constexpr int sg = STAGES <= 4 ? 4 : 8, sper = 64 / sg * waves;
    static constexpr int srows = (bm + bn + sper - 1) / sper * sper;
    static_assert(STAGES <= sg && bm % (64 / sg) == 0 && bm % 8 == 0, "");
};

struct SumParams {
    const int8_t *hc, *xc;
    const float *hs, *xs;
    void* slab;               // [split][r][cols], floats; PRECISE: doubles
    int d, r, groups, per_split, splits;
    int tiles_m, tiles_h, tiles;     // tiles along r (rows); column tiles of the H H^T part; all tiles
    int cols_h, cols;         // columns of a slab row: the H H^T part's, all (both multiples of 4)
    // one run holds everything: the results at once, the gradient's as doubles
    double *Ad, *Bd, *diag;   // (diag: A's diagonal once more, or null)
    double w, keep;
    const float *A_in, *B_in;
    float *A, *B;
};

template <typename S, bool PRECISE>
__global__ __launch_bounds__(64 * S::waves) void keep8_sums_kernel(SumParams p) {
    constexpr int STAGES = S::stages, AHEAD = STAGES - 1, STAGE = S::rows * GROUP;
    extern __shared__ __align__(16) int8_t lds[];            // [STAGES][STAGE], then float [2][S::srows][SG]
    float* lsc = (float*)(lds + STAGES * STAGE);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // workgroups of one run share H's codes: they follow each other on one XCD (workgroups go to the XCDs in turn,
    // an eighth of them to each)
    const int at = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int split = at / p.tiles, tile = at % p.tiles;
    if (split >= p.splits) return;
    const int tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const int m0 = tm * S::bm;
    const bool is_h = tn < p.tiles_h;
    const int n0 = (is_h ? tn : tn - p.tiles_h) * S::bn;
    const int N = is_h ? p.r : p.d;
    const int8_t* bc = is_h ? p.hc : p.xc;
    const float* bs = is_h ? p.hs : p.xs;
    const size_t ld = (size_t)p.groups * GROUP;
    const int g0 = split * p.per_split, g1 = min(p.groups, g0 + p.per_split);
    const int wm = (wave % S::wm) * 16 * S::mi, wn = (wave / S::wm) * 16 * S::nj;

    // A wave's loads are eight rows each, dealt out to the waves in turn; scales come SG groups at a time, SG lanes to
    // a row (a row's are 4 bytes a group: taken one group at a time they were as many requests as the codes):
    // [row][SG].  Addresses: a base for the wave and 32 bits a lane.
    constexpr int NW = S::waves, LOADS = S::rows / 8 / NW, SLOADS = S::srows / S::sper, SG = S::sg;
    auto rows_of = [&](int row, int& first, int& last) {         // the matrix row at row `row` of a stage, and the last there is
        const bool of_h = row < S::bm;
        last = of_h ? p.r - 1 : N - 1;
        first = min(of_h ? m0 + row : n0 + row - S::bm, last);
        return of_h;
    };
    const int8_t* base[LOADS];
    uint32_t off[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int row = (j * NW + wave) * 8;
        int first, last;
        base[j] = rows_of(row, first, last) ? p.hc : bc;
        base[j] += (size_t)first * ld;
        off[j] = (uint32_t)(min(first + (lane >> 3), last) - first) * (uint32_t)ld +
                 (((lane & 7) ^ (((row + (lane >> 3)) >> 1) & 7)) * 16);
    }
    const float* sbase[SLOADS];
    uint32_t soff[SLOADS];
#pragma unroll
    for (int j = 0; j < SLOADS; ++j) {
        int first, last;
        sbase[j] = rows_of((j * NW + wave) * (64 / SG), first, last) ? p.hs : bs;
        sbase[j] += (size_t)first * p.groups;
        soff[j] = (uint32_t)(min(first + lane / SG, last) - first) * (uint32_t)p.groups * 4;
    }
    auto fetch = [&](int g, int buf) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base[j] + (size_t)g * GROUP + off[j]),
                                             (__attribute__((address_space(3))) void*)(lds + buf * STAGE + (j * NW + wave) * 1024),
                                             16, 0, 0);
    };
    auto fetch_scales = [&](int g, int half) {
        const uint32_t q = (uint32_t)min(lane % SG, p.groups - 1 - g) * 4;
#pragma unroll
        for (int j = 0; j < SLOADS; ++j)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((const char*)(sbase[j] + g) + (soff[j] + q)),
                                             (__attribute__((address_space(3))) void*)(lsc + half * SG * S::srows + (j * NW + wave) * 64),
                                             4, 0, 0);
    };

    typedef std::conditional_t<PRECISE, double, float> V;
    typedef V V4 __attribute__((ext_vector_type(4)));
    V4 acc[S::mi][S::nj];
#pragma unroll
    for (int i = 0; i < S::mi; ++i)
#pragma unroll
        for (int j = 0; j < S::nj; ++j) acc[i][j] = V4{0, 0, 0, 0};
    // where a lane's operands and scales lie in a stage (whole tiles of 16 rows further on the chunks lie alike)
    const int op0 = (wm + (lane & 15)) * GROUP + (((lane >> 4) ^ ((lane >> 1) & 7)) * 16), op1 = op0 ^ 64;
    const int ba = (S::bm + wn - wm) * GROUP;
    const int sc_h = SG * (wm + (lane & 15)), sc_x = SG * (S::bm + wn + 4 * (lane >> 4));
    // AHEAD groups are on their way while one is computed, and the scales of the next SG.  Loads come back in order:
    // with only what was sent behind this group's codes still out - the codes of the AHEAD - 1 groups behind it, and
    // the scales where a fetch of them lies in between - this one's have arrived; behind the barrier those of all
    // waves have, and all waves are done with the group before, whose place the next one sent for takes.
    const int n = g1 - g0;
    fetch_scales(g0, 0);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (k < n) fetch(g0 + k, k);
    int buf = 0;
    for (int k = 0; k < n; ++k) {
        // (step i sent for scales where i is a multiple of SG and group i + SG is there)
        const int i = (k - 1) & ~(SG - 1);
        const bool scales_out = i >= k - AHEAD && i >= 0 && i + SG < n;
        if (k + AHEAD > n) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else if (scales_out) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((AHEAD - 1) * LOADS + SLOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((AHEAD - 1) * LOADS) : "memory");
        if (k + AHEAD < n) fetch(g0 + k + AHEAD, buf == 0 ? AHEAD : buf - 1);
        if (k % SG == 0 && k + SG < n) fetch_scales(g0 + k + SG, (k / SG + 1) & 1);
        const int8_t* la0 = lds + buf * STAGE + op0;
        const int8_t* la1 = lds + buf * STAGE + op1;
        const float* sa = lsc + (k / SG & 1) * SG * S::srows + k % SG + sc_h;
        const float* sb = lsc + (k / SG & 1) * SG * S::srows + k % SG + sc_x;
        // (X's rows are the matrix instruction's rows and H's its columns: a lane's four values lie side by side in
        // the slab)
        if constexpr (PRECISE) {
            // (X's operands and scales held and H's passed by: what the doubles leave room for)
            i32x4 fb[S::nj][2];
            float xs[S::nj][4];
#pragma unroll
            for (int j = 0; j < S::nj; ++j) {
                fb[j][0] = *reinterpret_cast<const i32x4*>(la0 + ba + 16 * j * GROUP);
                fb[j][1] = *reinterpret_cast<const i32x4*>(la1 + ba + 16 * j * GROUP);
#pragma unroll
                for (int e = 0; e < 4; ++e) xs[j][e] = sb[SG * (16 * j + e)];
            }
#pragma unroll
            for (int i = 0; i < S::mi; ++i) {
                const i32x4 fa0 = *reinterpret_cast<const i32x4*>(la0 + 16 * i * GROUP);
                const i32x4 fa1 = *reinterpret_cast<const i32x4*>(la1 + 16 * i * GROUP);
                const double hs = (double)sa[SG * 16 * i];
                i32x4 part[S::nj];
#pragma unroll
                for (int j = 0; j < S::nj; ++j) part[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j][0], fa0, i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < S::nj; ++j) part[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j][1], fa1, part[j], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < S::nj; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][j][e] = fma((double)xs[j][e] * hs, (double)part[j][e], acc[i][j][e]);
                    asm volatile("" : "+v"(acc[i][j]));
                }
            }
        } else {
            i32x4 fa[S::mi][2];
            float hs[S::mi];
#pragma unroll
            for (int i = 0; i < S::mi; ++i) {
                fa[i][0] = *reinterpret_cast<const i32x4*>(la0 + 16 * i * GROUP);
                fa[i][1] = *reinterpret_cast<const i32x4*>(la1 + 16 * i * GROUP);
                hs[i] = sa[SG * 16 * i];
            }
#pragma unroll
            for (int j = 0; j < S::nj; ++j) {
                const i32x4 fb0 = *reinterpret_cast<const i32x4*>(la0 + ba + 16 * j * GROUP);
                const i32x4 fb1 = *reinterpret_cast<const i32x4*>(la1 + ba + 16 * j * GROUP);
                float xs[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) xs[e] = sb[SG * (16 * j + e)];
                i32x4 part[S::mi];
#pragma unroll
                for (int i = 0; i < S::mi; ++i) part[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb0, fa[i][0], i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < S::mi; ++i) part[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb1, fa[i][1], part[i], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < S::mi; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(xs[e], hs[i] * (float)part[i][e], acc[i][j][e]);
            }
        }
        buf = buf == AHEAD ? 0 : buf + 1;
    }
    if (p.splits == 1) {
        const float* in = is_h ? p.A_in : p.B_in;
        float* out = is_h ? p.A : p.B;
#pragma unroll
        for (int i = 0; i < S::mi; ++i) {
            const int m = m0 + wm + 16 * i + (lane & 15);
            if (m >= p.r) continue;
#pragma unroll
            for (int j = 0; j < S::nj; ++j) {
                const int n = n0 + wn + 16 * j + 4 * (lane >> 4);
                const size_t at = (size_t)m * N + n;
                if constexpr (PRECISE) {
                    double* dst = (is_h ? p.Ad : p.Bd) + at;
                    if (p.diag && is_h)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (n + e == m) p.diag[m] = acc[i][j][e];
                    if (n + 4 <= N) {
                        reinterpret_cast<f64x2_any*>(dst)[0] = f64x2_any{acc[i][j][0], acc[i][j][1]};
                        reinterpret_cast<f64x2_any*>(dst)[1] = f64x2_any{acc[i][j][2], acc[i][j][3]};
                    } else
#pragma unroll
                        for (int e = 0; e < 3; ++e)
                            if (n + e < N) dst[e] = acc[i][j][e];
                } else if (n + 3 < N) {
                    f32x4_any v = {0.f, 0.f, 0.f, 0.f};
                    if (in) v = *reinterpret_cast<const f32x4_any*>(in + at);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (float)(p.w * (double)acc[i][j][e] + p.keep * (double)v[e]);
                    *reinterpret_cast<f32x4_any*>(out + at) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (n + e >= N) continue;
                        out[at + e] = (float)(p.w * (double)acc[i][j][e] + (in ? p.keep * (double)in[at + e] : 0.0));
                    }
                }
            }
        }
        return;
    }
    V* out = (V*)p.slab + (size_t)split * p.r * p.cols + (is_h ? 0 : p.cols_h);
#pragma unroll
    for (int i = 0; i < S::mi; ++i) {
        const int m = m0 + wm + 16 * i + (lane & 15);
        if (m >= p.r) continue;
#pragma unroll
        for (int j = 0; j < S::nj; ++j) {
            const int n = n0 + wn + 16 * j + 4 * (lane >> 4);
            if (n >= N) continue;                        // (rows of the slab are padded to whole quads)
            V* dst = out + (size_t)m * p.cols + n;
            if constexpr (PRECISE) {
                reinterpret_cast<f64x2*>(dst)[0] = f64x2{acc[i][j][0], acc[i][j][1]};
                reinterpret_cast<f64x2*>(dst)[1] = f64x2{acc[i][j][2], acc[i][j][3]};
            } else {
                *reinterpret_cast<f32x4*>(dst) = acc[i][j];
            }
        }
    }
}

// sum over the slabs of four neighbouring entries, in double and in a fixed order: the ZL threads of an entry take
// every ZL-th slab and are added in turn
template <int ZL>
__device__ __forceinline__ void sum_slabs(const float* src, size_t stride, int splits, int z0, double (&s)[4]) {
    s[0] = s[1] = s[2] = s[3] = 0.0;
#pragma unroll 8
    for (int z = z0; z < splits; z += ZL) {
        const float4 v = *reinterpret_cast<const float4*>(src + (size_t)z * stride);
        s[0] += (double)v.x; s[1] += (double)v.y; s[2] += (double)v.z; s[3] += (double)v.w;
    }
}
template <int ZL>
__device__ __forceinline__ void sum_slabs(const double* src, size_t stride, int splits, int z0, double (&s)[4]) {
    s[0] = s[1] = s[2] = s[3] = 0.0;
#pragma unroll 4
    for (int z = z0; z < splits; z += ZL) {
        const f64x2* at = reinterpret_cast<const f64x2*>(src + (size_t)z * stride);
        const f64x2 v = at[0], u = at[1];
        s[0] += v.x; s[1] += v.y; s[2] += u.x; s[3] += u.y;
    }
}

// A = keep A_in + w sum, B = keep B_in + w sum; from slabs of doubles (the gradient) the sums themselves to Ad and Bd.  Bound
// by reading the slabs (d=4096 r=256 n=65536 8.7 us, doubles 12.5).
template <int ZL, typename V>
__global__ __launch_bounds__(256) void keep8_reduce_kernel(int d, int r, int cols_h, int cols, int splits,
                                                            const V* __restrict__ slab, double w, double keep,
                                                            const float* A_in, const float* B_in, float* A, float* B,
                                                            double* __restrict__ Ad, double* __restrict__ Bd,
                                                            double* __restrict__ diag) {
    constexpr int Q = 256 / ZL;
    __shared__ double part[ZL][Q][4];
    const int q = threadIdx.x % Q, z0 = threadIdx.x / Q;
    const int quads = cols / 4;
    const size_t all = (size_t)r * quads, one = (size_t)r * cols;
    const size_t e = (size_t)blockIdx.x * Q + q;
    const int k = e < all ? (int)(e / quads) : 0, c = e < all ? (int)(e % quads) * 4 : 0;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    if (e < all) sum_slabs<ZL>(slab + (size_t)k * cols + c, one, splits, z0, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) part[z0][q][j] = s[j];
    __syncthreads();
    if (z0 != 0 || e >= all) return;
    const bool is_h = c < cols_h;
    const int n0 = is_h ? c : c - cols_h, N = is_h ? r : d;
    const float* in = is_h ? A_in : B_in;
    float* out = is_h ? A : B;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (n0 + j >= N) break;
        double v = part[0][q][j];
#pragma unroll
        for (int z = 1; z < ZL; ++z) v += part[z][q][j];
        const size_t at = (size_t)k * N + n0 + j;
        if constexpr (sizeof(V) == 8) {
            (is_h ? Ad : Bd)[at] = v;
            if (diag && is_h && n0 + j == k) diag[k] = v;
        } else out[at] = (float)(w * v + (in ? keep * (double)in[at] : 0.0));
    }
}

// dW[i][k] = sum_j W[i][j] A[j][k] - B[k][i] in double, rounded once: near a stationary dictionary the two terms
// nearly cancel.  A workgroup owns a 32 x 32 tile, its NW waves share the sum over j in sixteens and add up in LDS.  A
// wave loads the double matrix pipe's operands (16x16x4) straight into registers, the next sixteen while these are
// computed: four neighbours of W a lane, at j = 16 s + 4 (l / 16) + i in the i-th instruction, and rows of A.  Output
// row 4 e + l / 16.  Bound by the double matrix pipe where r is large (d=4096 r=256 19.5 us; r=1024 182, 47 TFLOP/s).
template <int NW> struct GradientLds { double part[NW][32][32], tb[32][33]; };
template <int NW, bool REST>                          // REST: only entries that are NaN so far
__device__ __forceinline__ void gradient_tile(GradientLds<NW>& lds, int i0, int k0, int d, int r, const float* __restrict__ W,
                                              const double* __restrict__ A, const double* __restrict__ B, float* __restrict__ dW) {
    auto& part = lds.part;
    auto& tb = lds.tb;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), m = lane & 15, quad = lane >> 4;
    for (int e = t; e < 1024; e += 64 * NW) {
        const int k = k0 + (e >> 5), i = i0 + (e & 31);
        tb[e & 31][e >> 5] = (k < r && i < d) ? B[(size_t)k * d + i] : 0.0;
    }
    // (rows and columns behind the last ones are the last ones and not stored, behind the last j the weight is zero)
    const float* row[2] = {W + (size_t)min(i0 + m, d - 1) * r, W + (size_t)min(i0 + 16 + m, d - 1) * r};
    const int col[2] = {min(k0 + m, r - 1), min(k0 + 16 + m, r - 1)};
    struct Step { f32x4_any w[2]; double a[4][2]; };
    auto fetch = [&](int j0, Step& v) {
        const int j = j0 + 4 * quad;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (j0 + 16 <= r) v.w[h] = *reinterpret_cast<const f32x4_any*>(row[h] + j);
            else
#pragma unroll
                for (int i = 0; i < 4; ++i) v.w[h][i] = j + i < r ? row[h][j + i] : 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) v.a[i][h] = A[(size_t)min(j + i, r - 1) * r + col[h]];
        }
    };
    f64x4 acc[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) acc[h][0] = acc[h][1] = f64x4{0.0, 0.0, 0.0, 0.0};
    auto compute = [&](const Step& v) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    acc[h][c] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)v.w[h][i], v.a[i][c], acc[h][c], 0, 0, 0);
    };
    Step even, odd;
    int j0 = wave * 16;
    if (j0 < r) fetch(j0, even);
    while (j0 < r) {
        if (j0 + 16 * NW < r) fetch(j0 + 16 * NW, odd);
        compute(even);
        j0 += 16 * NW;
        if (j0 >= r) break;
        if (j0 + 16 * NW < r) fetch(j0 + 16 * NW, even);
        compute(odd);
        j0 += 16 * NW;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[wave][16 * h + 4 * e + quad][16 * c + m] = acc[h][c][e];
    __syncthreads();
    for (int e = t; e < 1024; e += 64 * NW) {
        const int i = e >> 5, k = e & 31;
        double v = part[0][i][k];
#pragma unroll
        for (int z = 1; z < NW; ++z) v += part[z][i][k];
        if (i0 + i >= d || k0 + k >= r) continue;
        float* dst = dW + (size_t)(i0 + i) * r + k0 + k;
        if (!REST || *dst != *dst) *dst = (float)(v - tb[i][k]);
    }
}
template <int NW>
__global__ __launch_bounds__(64 * NW) void keep8_gradient_kernel(int d, int r, const float* __restrict__ W,
                                                                  const double* __restrict__ A, const double* __restrict__ B,
                                                                  float* __restrict__ dW) {
    __shared__ GradientLds<NW> lds;
    gradient_tile<NW, false>(lds, blockIdx.y * 32, blockIdx.x * 32, d, r, W, A, B, dW);
}
// Behind the product by digits (below): 64 x 64 entries a workgroup, if the mark of their tile is set, and of those what was left
// as NaN.  (Where none is set, d=8192 r=1024: 5 us; a workgroup for every 32 x 32 8.6.)
constexpr int LEFT = 64;
__global__ __launch_bounds__(256) void keep8_left_kernel(int d, int r, const float* __restrict__ W, const double* __restrict__ A,
                                                          const double* __restrict__ B, float* __restrict__ dW,
                                                          const int* __restrict__ marks, int tile, int across) {
    __shared__ GradientLds<4> lds;
    const int i1 = blockIdx.y * LEFT, k1 = blockIdx.x * LEFT;
    if (!marks[i1 / tile * across + k1 / tile]) return;
    for (int i0 = i1; i0 < min(d, i1 + LEFT); i0 += 32)
        for (int k0 = k1; k0 < min(r, k1 + LEFT); k0 += 32) {
            gradient_tile<4, true>(lds, i0, k0, d, r, W, A, B, dW);
            __syncthreads();
        }
}

// The same on the 8-bit matrix pipe, where r is large.  Atoms are balanced first, by c_j = 2^floor(log2(A_jj) / 2): the terms
// W_ij c_j and A_jk / c_j have the same products, no term of A's row k is then above twice the square root of A_kk, and what an atom
// weighs does not depend on how its scale is shared between W and H (one that no column uses weighs nothing).  Each row x of
// the balanced W and A (which is symmetric) is rounded to whole numbers N of 31 bits, x = p 2^-31 N with a power of two p of at
// most about twice the largest |x|, and N = sum_t q_t 2^(8 (3 - t)) cut into four digits of 8 bits.  Products of digits
// add up exactly in int32, those of one weight, t + u = 0..4, in one sum; they meet in double.
// What this is off by: half a unit of each x times the other's |x|, and of 2^62 a term what is left out (t + u > 4, below
// 2^23 (1 + 2^-8)), |error| <= 2^-32 (p_w S_a + p_a S_w) + 2^-38.9 r p_w p_a with the rows' sums S of magnitudes.  An entry is kept
// where that is at most 2^-25 (|W A| + |B|), half a float32 step of the terms; where it is not - a row's small terms count because
// its large ones meet zeros of A or cancel - it is left as NaN and its tile marked, for the double pipe to compute anew.  So
// every entry depends on its own row and column alone.  Bound by the matrix pipe (d=4096 r=1024: the thirteen products 55 us,
// 2.0 POP/s, the digits 10, the look at the marks 4.5; on the double matrix pipe 182.  Where nothing is held, a dictionary of both
// signs or codes that never meet, both are run: 280 us of the whole gradient instead of 84).
constexpr int DIGITS = 4, SUMS = 5;
constexpr int MOST_DIGIT_ROWS = 32767;           // 4 products of 128 x 128 add up below 2^31

// c_j of A_jj as a power of two; 0 for an atom without code, 1 for one that is not finite (its row of A says so)
__device__ __forceinline__ double balance(double diag, bool inverse) {
    const int hi = __double2hiint(diag);              // (a sum of squares of scales is no subnormal number and not negative)
    if (diag == 0.0) return inverse ? 1.0 : 0.0;
    if (hi >= 0x7ff00000) return 1.0;
    const int c = ((hi >> 20) - 1023) >> 1;
    return __hiloint2double((1023 + (inverse ? -c : c)) << 20, 0);
}

// digits[t][row][kp], zeros behind column r, the powers of two and the sums of magnitudes: W's d rows, then A's r; a wave a
// row, whose first 1024 entries are held in registers between finding the power and cutting.  The product's marks are
// taken back.  Bound by its vector instructions and the reading of W and A (d=4096 r=1024, 46 MB: 10 us).
__global__ __launch_bounds__(256) void keep8_digits_kernel(int d, int r, int kp, const float* __restrict__ W,
                                                            const double* __restrict__ A, const double* __restrict__ diag,
                                                            int8_t* __restrict__ digits, double* __restrict__ powers,
                                                            double* __restrict__ sums, int* __restrict__ marks, int n_marks) {
    constexpr int HELD = 4;
    for (int e = blockIdx.x * 256 + threadIdx.x; e < n_marks; e += gridDim.x * 256) marks[e] = 0;
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= d + r) return;
    // four neighbours, balanced (those behind column r - 1 are zeros)
    auto values = [&](int k, double (&v)[4]) {
        auto take = [&](const auto* src, bool inverse) {
            typedef std::remove_cv_t<std::remove_reference_t<decltype(*src)>> V;
            typedef V V4 __attribute__((ext_vector_type(4), aligned(sizeof(V))));
            typedef double D4 __attribute__((ext_vector_type(4), aligned(8)));
            if (k + 4 <= r) {
                const V4 x = *reinterpret_cast<const V4*>(src + k);
                const D4 c = *reinterpret_cast<const D4*>(diag + k);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = (double)x[j] * balance(c[j], inverse);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = k + j < r ? (double)src[k + j] * balance(diag[k + j], inverse) : 0.0;
            }
        };
        if (row < d) take(W + (size_t)row * r, false);
        else take(A + (size_t)(row - d) * r, true);
    };
    double most = 0.0, sum = 0.0, held[HELD][4];
    auto look = [&](const double (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            most = fmax(most, fabs(v[j]));
            sum += fabs(v[j]);
        }
    };
#pragma unroll
    for (int q = 0; q < HELD; ++q)
        if (lane * 4 + 256 * q < r) {
            values(lane * 4 + 256 * q, held[q]);
            look(held[q]);
        }
    for (int k = lane * 4 + 256 * HELD; k < r; k += 256) {
        double v[4];
        values(k, v);
        look(v);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        most = fmax(most, __shfl_xor(most, o, 64));
        sum += __shfl_xor(sum, o, 64);
    }
    const bool fine = sum <= 1.7976931348623157e308;  // (a NaN or an infinity anywhere is in the sum)
    int e = 0;                                        // most <= 127/128 2^e: the first digit is at most 127
    if (fine && frexp(most, &e) > 127.0 / 128.0) ++e;
    if (lane == 0) {
        powers[row] = !fine ? (double)__int_as_float(0x7fc00000) : most > 0.0 ? ldexp(1.0, e) : 0.0;
        sums[row] = sum;
    }
    const double scale = fine ? ldexp(1.0, 31 - e) : 0.0;
    const size_t plane = (size_t)(d + r) * kp;
    auto cut = [&](int k, const double (&v)[4]) {
        // N's digits of 8 bits with their signs: with a half of each but the first added the carries are where they
        // belong, and the bytes' upper bits the other way round are the digits
        uint32_t n[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) n[j] = fine ? ((uint32_t)(int)rint(v[j] * scale) + 0x00808080u) ^ 0x00808080u : 0u;
#pragma unroll
        for (int t = 0; t < DIGITS; ++t) {
            const uint32_t at = 3 - t, pick = at | (4 + at) << 8 | 0x0c0c0000u;      // byte `at` of both (12: zero)
            const uint32_t lo = __builtin_amdgcn_perm(n[1], n[0], pick), hi = __builtin_amdgcn_perm(n[3], n[2], pick);
            *reinterpret_cast<uint32_t*>(digits + t * plane + (size_t)row * kp + k) = lo | hi << 16;
        }
    };
#pragma unroll
    for (int q = 0; q < HELD; ++q) {
        const int k = lane * 4 + 256 * q;
        if (k >= kp) continue;
        if (k >= r)
#pragma unroll
            for (int j = 0; j < 4; ++j) held[q][j] = 0.0;
        cut(k, held[q]);
    }
    for (int k = lane * 4 + 256 * HELD; k < kp; k += 256) {
        double v[4];
        values(k, v);
        cut(k, v);
    }
}

// A tile of 16 MI WM columns of dW (A's rows are the matrix instruction's rows) and 16 NJ WN rows; 64 of the contraction a
// step, the next step's digits on their way to LDS, in rows of 64 bytes whose chunks are permuted by (row >> 2) & 3.
template <int MI, int NJ, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void keep8_digit_product_kernel(int d, int r, int kp, const int8_t* __restrict__ digits,
                                                                            const double* __restrict__ powers,
                                                                            const double* __restrict__ sums,
                                                                            const double* __restrict__ B, float* __restrict__ dW,
                                                                            int* __restrict__ marks) {
    constexpr int NW = WM * WN, BM = 16 * MI * WM, BN = 16 * NJ * WN, BLOCKS = DIGITS * (BM + BN) / 16, LOADS = BLOCKS / NW;
    constexpr int STAGE = BLOCKS * 1024;
    static_assert(BLOCKS % NW == 0 && BM % 16 == 0, "");
    extern __shared__ __align__(16) int8_t lds[];      // [2][digit][BM rows of A, BN rows of W][64]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int k0 = blockIdx.x * BM, i0 = blockIdx.y * BN;
    const int wm = wave % WM * 16 * MI, wn = wave / WM * 16 * NJ;
    const size_t plane = (size_t)(d + r) * kp;
    const int8_t* src[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {                  // (rows behind the last one are the last one and not stored)
        const int block = j * NW + wave, t = block / ((BM + BN) / 16), at = block % ((BM + BN) / 16) * 16 + (lane >> 2);
        const int row = at < BM ? d + min(k0 + at, r - 1) : min(i0 + at - BM, d - 1);
        src[j] = digits + t * plane + (size_t)row * kp + ((lane & 3) ^ ((lane >> 4) & 3)) * 16;
    }
    auto fetch = [&](int k, int buf) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[j] + k),
                                             (__attribute__((address_space(3))) void*)(lds + buf * STAGE + (j * NW + wave) * 1024),
                                             16, 0, 0);
    };
    i32x4 acc[SUMS][MI][NJ];
#pragma unroll
    for (int t = 0; t < SUMS; ++t)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[t][i][j] = i32x4{0, 0, 0, 0};
    const int op = (lane & 15) * 64 + (((lane >> 4) ^ ((lane >> 2) & 3)) * 16);
    fetch(0, 0);
    for (int k = 0, buf = 0; k < kp; k += 64, buf ^= 1) {
        // (this step's digits have come, all waves are done with the step before, whose place the next one's take)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (k + 64 < kp) fetch(k + 64, buf ^ 1);
        const int8_t* base = lds + buf * STAGE + op;
        i32x4 fb[DIGITS][NJ];
#pragma unroll
        for (int t = 0; t < DIGITS; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[t][j] = *reinterpret_cast<const i32x4*>(base + (t * (BM + BN) + BM + wn + 16 * j) * 64);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            i32x4 fa[DIGITS];
#pragma unroll
            for (int t = 0; t < DIGITS; ++t) fa[t] = *reinterpret_cast<const i32x4*>(base + (t * (BM + BN) + wm + 16 * i) * 64);
#pragma unroll
            for (int t = 0; t < DIGITS; ++t)
#pragma unroll
                for (int u = 0; u < DIGITS && t + u < SUMS; ++u)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        acc[t + u][i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[t], fb[u][j], acc[t + u][i][j], 0, 0, 0);
        }
    }
    bool unheld = false;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int i = i0 + wn + 16 * j + (lane & 15);
        if (i >= d) continue;
        const double pi = powers[i], si = sums[i];
#pragma unroll
        for (int m = 0; m < MI; ++m) {
            const int k = k0 + wm + 16 * m + 4 * (lane >> 4);
            f32x4_any out;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                double v = (double)acc[SUMS - 1][m][j][e];
#pragma unroll
                for (int t = SUMS - 2; t >= 0; --t) v = v * 0x1p-8 + (double)acc[t][m][j][e];
                const int kk = min(k + e, r - 1);
                const double pk = powers[d + kk], b = B[(size_t)kk * d + i];
                v = v * 0x1p-14 * pi * pk;
                const double off = 0x1p-32 * (pi * sums[d + kk] + pk * si) + 0x1.13p-39 * r * pi * pk;
                const bool held = off <= 0x1p-25 * (fabs(v) + fabs(b));
                unheld = unheld || !held;
                out[e] = held ? (float)(v - b) : __int_as_float(0x7fc00000);
            }
            float* dst = dW + (size_t)i * r + k;
            if (k + 4 <= r) *reinterpret_cast<f32x4_any*>(dst) = out;
            else
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (k + e < r) dst[e] = out[e];
        }
    }
    if (unheld) marks[blockIdx.y * gridDim.x + blockIdx.x] = 1;
}

// The same gradient by way of the residual, dW = (W H - X) H^T, for up to 128 columns: with n < r / 2 of them it is
// less work than W (H H^T), and one launch.  A workgroup owns 16 rows.  Its waves share the atoms of W H (double matrix
// pipe: row l % 16 of W and 16 columns of H at k = 16 s + 4 (l / 16) + j in the j-th instruction, so that a lane
// loads four neighbours of W and words of four codes; the scale of an atom goes with W, one exact double product),
// add up in LDS and take X off; then they share the atoms of the result, with the residual's operands in registers and the
// scale of an atom on its sum.  TILES sixteens of columns (1, 4 or 8), NW waves.  Bound by the double matrix pipe of the
// CUs that have rows (d=2372 r=581 n=2 9.6 us, n=128 30; by the sums 60).
template <int TILES, int NW>
__global__ __launch_bounds__(64 * NW) void keep8_residual_kernel(int d, int r, const float* __restrict__ W,
                                                                  const int8_t* __restrict__ xc, const float* __restrict__ xs,
                                                                  const int8_t* __restrict__ hc, const float* __restrict__ hs,
                                                                  float* __restrict__ dW) {
    constexpr int N = 16 * TILES, WORDS = (TILES + 3) / 4, LINE = N + 2;
    extern __shared__ __align__(16) double sums[];        // [NW][16][N], then the residual [16][LINE]
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, quad = lane >> 4;
    const int i0 = blockIdx.x * 16;
    const float* wrow = W + (size_t)min(i0 + c, d - 1) * r;
    struct Step { float w[4], s[4]; uint32_t h[4][WORDS]; };
    auto fetch = [&](int k0, Step& v) {                   // (atoms behind the last one: the last one's, with weight 0)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = min(k0 + 4 * quad + j, r - 1);
            v.w[j] = wrow[k];
            v.s[j] = hs[k];
            const int8_t* code = hc + (size_t)k * GROUP;
#pragma unroll
            for (int u = 0; u < WORDS; ++u)
                v.h[j][u] = TILES == 1 ? (uint32_t)(int)code[c] : *reinterpret_cast<const uint32_t*>(code + 64 * u + 4 * c);
        }
    };
    f64x4 acc[TILES];
#pragma unroll
    for (int q = 0; q < TILES; ++q) acc[q] = f64x4{0.0, 0.0, 0.0, 0.0};
    Step now, next;
    if (wave * 16 < r) fetch(wave * 16, now);
    for (int k0 = wave * 16; k0 < r; k0 += 16 * NW) {
        if (k0 + 16 * NW < r) fetch(k0 + 16 * NW, next);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double a = k0 + 4 * quad + j < r ? (double)now.w[j] * (double)now.s[j] : 0.0;
#pragma unroll
            for (int q = 0; q < TILES; ++q) {
                const int code = TILES == 1 ? (int)now.h[j][0] : (int)(int8_t)(now.h[j][q / 4] >> (8 * (q % 4)));
                acc[q] = __builtin_amdgcn_mfma_f64_16x16x4f64(a, (double)code, acc[q], 0, 0, 0);
            }
        }
        if (k0 + 16 * NW < r) now = next;
    }
#pragma unroll
    for (int q = 0; q < TILES; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sums[(wave * 16 + 4 * e + quad) * N + (TILES == 1 ? c : 64 * (q / 4) + 4 * c + q % 4)] = acc[q][e];
    __syncthreads();
    constexpr int EACH = (16 * N + 64 * NW - 1) / (64 * NW);
    double rest[EACH];
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
        const int e = t + q * 64 * NW, row = min(i0 + e / N, d - 1);
        if (e >= 16 * N) continue;
        double v = sums[e];
#pragma unroll
        for (int z = 1; z < NW; ++z) v += sums[z * 16 * N + e];
        rest[q] = v - (double)xs[row] * (double)xc[(size_t)row * GROUP + e % N];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
        const int e = t + q * 64 * NW;
        if (e < 16 * N) sums[e / N * LINE + e % N] = rest[q];
    }
    __syncthreads();
    // instruction 16 u + j (one tile: j) contracts over the columns 64 u + 16 (l / 16) + j (4 (l / 16) + j)
    constexpr int STEPS = N / 4, RUN = TILES == 1 ? 4 : 16;
    double res[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) res[s] = sums[c * LINE + s / RUN * 64 + quad * RUN + s % RUN];
    for (int k0 = wave * 16; k0 < r; k0 += 16 * NW) {
        const int k = min(k0 + c, r - 1);
        const int8_t* code = hc + (size_t)k * GROUP + quad * RUN;
        const double scale = (double)hs[k];
        uint32_t h[STEPS / 4];
        if constexpr (TILES == 1) h[0] = *reinterpret_cast<const uint32_t*>(code);
        else
#pragma unroll
            for (int u = 0; u < WORDS; ++u) {
                const uint4 v = *reinterpret_cast<const uint4*>(code + 64 * u);
                h[4 * u] = v.x; h[4 * u + 1] = v.y; h[4 * u + 2] = v.z; h[4 * u + 3] = v.w;
            }
        f64x4 sum = f64x4{0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            sum = __builtin_amdgcn_mfma_f64_16x16x4f64(res[s], (double)(int)(int8_t)(h[s / 4] >> (8 * (s % 4))), sum, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = i0 + 4 * e + quad;
            if (i < d && k0 + c < r) dW[(size_t)i * r + k0 + c] = (float)(scale * sum[e]);
        }
    }
}

// ------------------------------------------------------------------------------------------- launches
using Wide = Tile<4, 2, 4, 4, 3>;       // 256 x 128
using Middle = Tile<4, 2, 2, 8, 3>;     // 128 x 256
using Narrow = Tile<4, 2, 1, 8, 3>;     // 64 x 256
using Slim = Tile<2, 2, 1, 4, 6>;       // 32 x 128

struct SumPlan { int tile, bm, bn, tiles_m, tiles_h, tiles_x, cols_h, cols, splits, per; double cost; };
// The tile and the number of runs with the least time by what was measured of them: a tile's own time (us: filling the ring,
// writing the sums), what a group takes it - its operations, or with the chip full its codes' way from the caches at
// 8 TB/s - and, with several runs, a second launch and the slabs' way through memory at 4 TB/s.  One workgroup a CU.
// (us: d=8192 r=64 n=1000 64 x 256 13.2, 32 x 128 6.4; d=8192 r=256 n=1000 256 x 128 20, 64 x 256 12; d=4096 r=256
// n=65536 256 x 128 125, 64 x 256 180; d=1200 r=100 n=8191 in runs of four groups 17.3, of two 20.3.)
// Sums in double (the gradient's): a group that waits for no codes takes a third more (27 groups in 64 x 256 37 us), and an
// entry of a slab a quarter (whole gradient, us: d=290 r=876 n=3335 in one run 59.6, in three 49.9; d=4096 r=256 n=65536
// 256 x 128 176, 128 x 256 178; d=1024 66 and 66).
SumPlan sum_plan(int d, int r, int n, bool precise) {
    static constexpr struct { int bm, bn, rows; double own, group; } kind[4] = {{Slim::bm, Slim::bn, Slim::rows, 2.4, 0.5},
                                                                                 {Narrow::bm, Narrow::bn, Narrow::rows, 5.0, 0.87},
                                                                                 {Middle::bm, Middle::bn, Middle::rows, 7.0, 1.25},
                                                                                 {Wide::bm, Wide::bn, Wide::rows, 9.6, 1.2}};
    SumPlan q;
    const int groups = (n + GROUP - 1) / GROUP;
    q.cols_h = (r + 3) & ~3;
    q.cols = q.cols_h + ((d + 3) & ~3);
    double best = -1;
    for (int i = 0; i < 4; ++i) {
        if (i > 0 && r <= kind[i - 1].bm) break;
        const int tiles_m = (r + kind[i].bm - 1) / kind[i].bm, tiles_h = (r + kind[i].bn - 1) / kind[i].bn;
        const int tiles_x = (d + kind[i].bn - 1) / kind[i].bn;
        const double tiles = (double)tiles_m * (tiles_h + tiles_x);
        for (int target = 0; target <= 512; target = target ? 2 * target : 64) {
            const int want = (int)std::max(1.0, std::min(target / tiles, (double)groups));
            const int per = (groups + want - 1) / want, splits = (groups + per - 1) / per;
            const double w = tiles * splits;
            double cost = std::ceil(w / 256) *
                          (kind[i].own + per * std::max(kind[i].group * (precise ? 1.35 : 1.0),
                                                        kind[i].rows * (double)GROUP * std::min(w, 256.0) / 8e6));
            if (splits > 1) cost += 5.0 + (precise ? 2.5e-6 : 2e-6) * splits * r * q.cols;
            if (best >= 0 && cost >= best) continue;
            best = q.cost = cost;
            q.tile = i;
            q.bm = kind[i].bm;
            q.bn = kind[i].bn;
            q.tiles_m = tiles_m;
            q.tiles_h = tiles_h;
            q.tiles_x = tiles_x;
            q.per = per;
            q.splits = splits;
        }
    }
    return q;
}
size_t sums_bytes(const SumPlan& q, int r, bool precise) {
    return q.splits == 1 ? 0 : ((size_t)q.splits * r * q.cols * (precise ? sizeof(double) : sizeof(float)) + 255) & ~(size_t)255;
}

int check8(onmf_ctx* c, const char* what, int d, int n, const void* codes, const void* scales) {
    if (d <= 0 || n <= 0 || !codes || !scales || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 3))
        return onmf_fail(c, ONMF_ERR_ARG, "%s: bad arguments (d=%d n=%d; codes must be aligned to 16 bytes)", what, d, n);
    if (n > MOST_COLS) return onmf_fail(c, ONMF_ERR_ARG, "%s: n=%d is more than 2^28 columns", what, n);
    if (d > MOST_ROWS) return onmf_fail(c, ONMF_ERR_ARG, "%s: %d rows are more than the kernels' int counts", what, d);
    return ONMF_OK;
}

template <typename S, bool PRECISE>
int launch_sums(onmf_ctx* c, const SumParams& p, hipStream_t s) {
    constexpr size_t bytes = S::stages * (size_t)S::rows * GROUP + 2 * (size_t)S::srows * S::sg * sizeof(float);
    static_assert(bytes <= 160 * 1024, "LDS of a compute unit");
    static LdsLimit lim;
    ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)keep8_sums_kernel<S, PRECISE>, bytes));
    hipLaunchKernelGGL((keep8_sums_kernel<S, PRECISE>), dim3((p.tiles * p.splits + 7) / 8 * 8), dim3(64 * S::waves), bytes, s, p);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

template <bool PRECISE>
int launch_tile(onmf_ctx* c, int tile, const SumParams& p, hipStream_t s) {
    switch (tile) {
        case 0: return launch_sums<Slim, PRECISE>(c, p, s);
        case 1: return launch_sums<Narrow, PRECISE>(c, p, s);
        case 2: return launch_sums<Middle, PRECISE>(c, p, s);
        default: return launch_sums<Wide, PRECISE>(c, p, s);
    }
}

// The sums of a minibatch into A and B, or as doubles into Ad and Bd.
int run_sums(onmf_ctx* c, const SumPlan& q, int d, int r, int n, const int8_t* xc, const float* xs, const int8_t* hc, const float* hs,
             void* slab, double w, double keep, const float* A_in, const float* B_in, float* A, float* B, double* Ad,
             double* Bd, double* diag, hipStream_t s) {
    SumParams p;
    p.hc = hc; p.xc = xc; p.hs = hs; p.xs = xs; p.slab = slab;
    p.d = d; p.r = r; p.groups = (n + GROUP - 1) / GROUP; p.per_split = q.per; p.splits = q.splits;
    p.tiles_m = q.tiles_m; p.tiles_h = q.tiles_h; p.tiles = q.tiles_m * (q.tiles_h + q.tiles_x);
    p.cols_h = q.cols_h; p.cols = q.cols;
    p.w = w; p.keep = keep; p.A_in = A_in; p.B_in = B_in; p.A = A; p.B = B;
    p.Ad = Ad; p.Bd = Bd; p.diag = diag;
    ONMF_TRY(Ad ? launch_tile<true>(c, q.tile, p, s) : launch_tile<false>(c, q.tile, p, s));
    if (q.splits == 1) return ONMF_OK;
    // (few entries with many slabs: more threads to an entry)
    const size_t quads = (size_t)r * q.cols / 4;
    auto reduce = [&](auto kernel, int per, const auto* slabs) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((quads + per - 1) / per)), dim3(256), 0, s, d, r, q.cols_h, q.cols, q.splits, slabs,
                           w, keep, A_in, B_in, A, B, Ad, Bd, diag);
    };
    if (Ad && quads < 16384) reduce(keep8_reduce_kernel<16, double>, 16, (const double*)slab);
    else if (Ad) reduce(keep8_reduce_kernel<4, double>, 64, (const double*)slab);
    else if (quads < 16384) reduce(keep8_reduce_kernel<16, float>, 16, (const float*)slab);
    else reduce(keep8_reduce_kernel<4, float>, 64, (const float*)slab);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

// Whole digits take three launches, of which the last, for what they do not hold, mostly ends at once.  Measured (us of the
// whole gradient, n=500, digits and the double pipe): d r^2 = 2.7e8, d=4096 r=256 31.6 and 30.5; 4.3e8 and 4.5e8, d=1200 r=600 37.7
// and 39.7, d=4096 r=330 42 and 46; 5.4e8, d=2048 r=512 36.5 and 42.5; 6.3e8, d=600 r=1024 41 and 54; 4.3e9, d=4096 r=1024 84 and 200.
// With few features cutting A takes longer than the product: d=200 r=1500 48 and 56, d=100 r=2050 68 and 66, d=32 r=4096 147 and 92.
bool by_digits(int d, int r) { return d >= 128 && r <= MOST_DIGIT_ROWS && (double)d * r * r > 4e8; }
int digit_columns(int r) { return (r + 63) & ~63; }
// Rows and columns of a workgroup's tile
int digit_tile(int d, int r) { return (long long)((r + 127) / 128) * ((d + 127) / 128) >= 256 ? 128 : 64; }
struct DigitSpace {
    int8_t* digits;                // [DIGITS][d + r][digit_columns]
    double *powers, *sums;         // [d + r]
    double* diag;                  // [r]
    int* marks;                    // [(d + tile - 1) / tile][(r + tile - 1) / tile]
    int tile, n_marks;
    size_t bytes;
    DigitSpace(int d, int r, char* ws) {
        tile = digit_tile(d, r);
        n_marks = ((d + tile - 1) / tile) * ((r + tile - 1) / tile);
        const size_t planes = ((size_t)DIGITS * ((size_t)d + r) * digit_columns(r) + 255) & ~(size_t)255;
        digits = (int8_t*)ws;
        powers = (double*)(ws + planes);
        sums = powers + d + r;
        diag = sums + d + r;
        marks = (int*)(diag + r);
        bytes = planes + sizeof(double) * (2 * ((size_t)d + r) + r) + sizeof(int) * (size_t)n_marks;
    }
};
size_t digits_bytes(int d, int r) { return by_digits(d, r) ? DigitSpace(d, r, nullptr).bytes : 0; }
template <int MI, int NJ, int WM, int WN>
int launch_digit_product(onmf_ctx* c, int d, int r, const DigitSpace& q, const float* W, const double* A, const double* B, float* dW,
                         hipStream_t s) {
    constexpr int BM = 16 * MI * WM, BN = 16 * NJ * WN;
    static_assert(BM == BN && BM % LEFT == 0, "a mark is a square");
    constexpr size_t bytes = 2 * (size_t)DIGITS * (BM + BN) * 64;
    static LdsLimit lim;
    ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)keep8_digit_product_kernel<MI, NJ, WM, WN>, bytes));
    const dim3 grid((r + BM - 1) / BM, (d + BN - 1) / BN);
    hipLaunchKernelGGL((keep8_digit_product_kernel<MI, NJ, WM, WN>), grid, dim3(64 * WM * WN), bytes, s, d, r, digit_columns(r), q.digits,
                       q.powers, q.sums, B, dW, q.marks);
    HIP_TRY(c, hipGetLastError());
    hipLaunchKernelGGL(keep8_left_kernel, dim3((r + LEFT - 1) / LEFT, (d + LEFT - 1) / LEFT), dim3(256), 0, s, d, r, W, A, B, dW, q.marks, BM,
                       (int)grid.x);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}
int launch_gradient(onmf_ctx* c, int d, int r, const float* W, const double* A, const double* B, float* dW, char* ws, hipStream_t s) {
    if (by_digits(d, r)) {
        const DigitSpace q(d, r, ws);
        hipLaunchKernelGGL(keep8_digits_kernel, dim3((d + r + 3) / 4), dim3(256), 0, s, d, r, digit_columns(r), W, A, q.diag, q.digits,
                           q.powers, q.sums, q.marks, q.n_marks);
        HIP_TRY(c, hipGetLastError());
        if (q.tile == 128) return launch_digit_product<4, 2, 2, 4>(c, d, r, q, W, A, B, dW, s);
        return launch_digit_product<2, 2, 2, 2>(c, d, r, q, W, A, B, dW, s);
    }
    const dim3 grid((r + 31) / 32, (d + 31) / 32);
    // (more waves a tile where there are few tiles and enough of j: d=215 r=1017 15.3 us, with four waves 28; with many
    // tiles the double matrix pipe is what counts: d=8192 r=256 36 us, with eight waves 42)
    if (r > 64 && (size_t)grid.x * grid.y <= 512)
        hipLaunchKernelGGL(keep8_gradient_kernel<8>, grid, dim3(512), 0, s, d, r, W, A, B, dW);
    else
        hipLaunchKernelGGL(keep8_gradient_kernel<4>, grid, dim3(256), 0, s, d, r, W, A, B, dW);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

// The residual costs a workgroup r times the columns that its tiles hold; the sums a launch more and W (H H^T), d r^2
// at 45 TFLOP/s.  In us, from measurements (residual and sums: d=441 r=25 n=128 6.0 and 9; d=2372 r=581 n=2 9.6 and
// 60; d=60 r=1024 n=100 43 and 22; d=65536 r=64 n=128 83 and 49, n=16 24 and 49).
bool by_residual(const SumPlan& q, int d, int r, int n) {
    if (n > GROUP) return false;
    const double residual = 2.5 + std::ceil(d / (n <= 16 ? 8192.0 : 4096.0)) * (1.0 + r * (n <= 16 ? 0.009 : n <= 64 ? 0.023 : 0.04));
    return residual < q.cost + 6.0 + 0.011 * r + 2.0 * d * r * r / 45e6;
}

template <int TILES, int NW>
int launch_residual(onmf_ctx* c, int d, int r, const float* W, const int8_t* xc, const float* xs, const int8_t* hc, const float* hs,
                    float* dW, hipStream_t s) {
    constexpr size_t bytes = (size_t)NW * 16 * 16 * TILES * sizeof(double);
    static_assert(bytes <= 160 * 1024 && NW >= 2, "the residual, with its lines' padding, takes the sums' place");
    static LdsLimit lim;
    ONMF_TRY(onmf_raise_lds_limit(c, lim, (const void*)keep8_residual_kernel<TILES, NW>, bytes));
    hipLaunchKernelGGL((keep8_residual_kernel<TILES, NW>), dim3((d + 15) / 16), dim3(64 * NW), bytes, s, d, r, W, xc, xs, hc, hs, dW);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

// H H^T and H X^T, and the digits behind them
size_t both_sums_bytes(int d, int r) {
    return (sizeof(double) * (size_t)r * ((size_t)r + d) + 255) & ~(size_t)255;
}
size_t gradient_bytes(int d, int r) { return both_sums_bytes(d, r) + digits_bytes(d, r); }

// Groups a thread handles: several where there are enough of them to fill the chip with.
template <typename T>
void launch_keep(size_t all, int n, int groups, const T* X, int ldx, int8_t* codes, float* scales, hipStream_t s) {
    if (all >= 65536)
        hipLaunchKernelGGL((keep8_kernel<T, 2>), dim3((unsigned)((all + 31) / 32)), dim3(256), 0, s, all, n, groups, X, ldx, codes,
                           scales);
    else
        hipLaunchKernelGGL((keep8_kernel<T, 1>), dim3((unsigned)((all + 15) / 16)), dim3(256), 0, s, all, n, groups, X, ldx, codes,
                           scales);
}
void launch_expand(size_t all, int n, int groups, const int8_t* codes, const float* scales, float* X, int ldx, hipStream_t s) {
    if (all >= 65536)
        hipLaunchKernelGGL(keep8_expand_kernel<4>, dim3((unsigned)((all + 31) / 32)), dim3(256), 0, s, all, n, groups, codes, scales,
                           X, ldx);
    else
        hipLaunchKernelGGL(keep8_expand_kernel<1>, dim3((unsigned)((all + 7) / 8)), dim3(256), 0, s, all, n, groups, codes, scales, X,
                           ldx);
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
    const size_t all = (size_t)d * groups;
    if (all > MOST_GROUPS) return onmf_fail(c, ONMF_ERR_ARG, "keep8: %d x %d is more than 2^29 - 32 groups of 128", d, n);
    if (x_type == ONMF_TYPE_F32) launch_keep(all, n, groups, (const float*)X, ldx, codes, scales, s);
    else launch_keep(all, n, groups, (const uint16_t*)X, ldx, codes, scales, s);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

int onmf_keep8_expand(onmf_ctx* c, int d, int n, const int8_t* codes, const float* scales, const int64_t* idx, int b,
                      float* X, int ldx, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check8(c, "keep8_expand", d, n, codes, scales));
    const int cols = idx ? b : n;
    if (!X || cols <= 0 || cols > 2147483647 - 1024 || ldx < cols)
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_expand: bad arguments (b=%d ldx=%d)", b, ldx);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const int groups = (n + GROUP - 1) / GROUP;
    const size_t all = (size_t)d * groups;
    if (idx)
        hipLaunchKernelGGL(keep8_gather_kernel, dim3((b + 255) / 256, std::min(d, 4096)), dim3(256), 0, s, d, n, groups, codes,
                           scales, (const long long*)idx, b, X, ldx);
    else if (all > MOST_GROUPS)
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_expand: %d x %d is more than 2^29 - 32 groups of 128", d, n);
    else
        launch_expand(all, n, groups, codes, scales, X, ldx, s);
    HIP_TRY(c, hipGetLastError());
    return ONMF_OK;
}

size_t onmf_keep8_workspace(int d, int r, int n, int gradient) {
    if (d <= 0 || r <= 0 || n <= 0 || n > MOST_COLS) return 0;                  // sizes that the calls refuse
    if (d > MOST_ROWS || r > MOST_ROWS || (gradient && (d > (1 << 18) || r > (1 << 18)))) return 0;
    const SumPlan q = sum_plan(d, r, n, true);
    if (gradient && by_residual(q, d, r, n)) return 0;
    // slabs for either call's runs
    const size_t slabs = std::max(sums_bytes(q, r, true), sums_bytes(sum_plan(d, r, n, false), r, false));
    return slabs + (gradient ? gradient_bytes(d, r) : 0);
}

int onmf_keep8_aggregate(onmf_ctx* c, int d, int r, int n, const int8_t* x_codes, const float* x_scales,
                         const int8_t* h_codes, const float* h_scales, double w, const float* A_in, const float* B_in,
                         float* A_out, float* B_out, void* ws, size_t ws_bytes, void* stream) {
    if (!c) return ONMF_ERR_ARG;
    ONMF_TRY(check8(c, "keep8_aggregate", d, n, x_codes, x_scales));
    ONMF_TRY(check8(c, "keep8_aggregate", r, n, h_codes, h_scales));
    if (!A_out || !B_out) return onmf_fail(c, ONMF_ERR_ARG, "keep8_aggregate: an output is null");
    const size_t need = onmf_keep8_workspace(d, r, n, 0);
    if ((need && !ws) || ws_bytes < need || ((uintptr_t)ws & 15))
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_aggregate: workspace of %zu bytes, %zu needed, aligned to 16", ws_bytes, need);
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    return run_sums(c, sum_plan(d, r, n, false), d, r, n, x_codes, x_scales, h_codes, h_scales, ws, w, 1.0 - w, A_in, B_in,
                    A_out, B_out, nullptr, nullptr, nullptr, s);
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
    if ((need && !ws) || ws_bytes < need || ((uintptr_t)ws & 15))
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_gradient: workspace of %zu bytes, %zu needed, aligned to 16", ws_bytes, need);
    if (dW < W + (size_t)d * r && W < dW + (size_t)d * r)
        return onmf_fail(c, ONMF_ERR_ARG, "keep8_gradient: dW lies over W, which all of it is computed from");
    ONMF_ENTER(c);
    hipStream_t s = (hipStream_t)stream;
    const SumPlan q = sum_plan(d, r, n, true);
    if (by_residual(q, d, r, n)) {
        if (n <= 16) return launch_residual<1, 16>(c, d, r, W, x_codes, x_scales, h_codes, h_scales, dW, s);
        if (n <= 64) return launch_residual<4, 16>(c, d, r, W, x_codes, x_scales, h_codes, h_scales, dW, s);
        return launch_residual<8, 8>(c, d, r, W, x_codes, x_scales, h_codes, h_scales, dW, s);
    }
    double* A = (double*)((char*)ws + sums_bytes(q, r, true));
    char* rest = (char*)A + both_sums_bytes(d, r);
    ONMF_TRY(run_sums(c, q, d, r, n, x_codes, x_scales, h_codes, h_scales, ws, 1.0, 0.0, nullptr, nullptr, nullptr, nullptr,
                      A, A + (size_t)r * r, by_digits(d, r) ? DigitSpace(d, r, rest).diag : nullptr, s));
    return launch_gradient(c, d, r, W, A, A + (size_t)r * r, dW, rest, s);
}

}  // extern "C"
