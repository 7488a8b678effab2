// The dense layer with its epilogue, forward and backward:
//   z = x w^T + bias,  y = act(z) + residual;
//   dz = dy act'(z),   dx = dz w,  dw = dz^T x,  dbias = sum of dz over the rows.
// x [m, k], w [n, k], y, z, dy, residual [m, n]; float32, float16 or bfloat16, sums in float32.
//
// Three products of the same form, C[i, j] = sum_c A[i, c] B[j, c]:
//   forward  A = x    B = w          both contiguous along the contraction
//   dx       A = dz   B = w^T        B contiguous along j
//   dw       A = dz^T B = x^T        both contiguous along i, j
#include <hip/hip_runtime.h>

#include "train_common.h"
#include "train_kernels.h"

namespace scmiac {
namespace {

using namespace train;

enum { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };
enum { kForward = 0, kDx = 1, kDw = 2 };

constexpr float kInvSqrt2Pi = 0.39894228040143267794f;

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * z)); }      // (good to a step of float32)

// The normal distribution function P(z), and e = exp(-z^2 / 2).  P(-a) = e t q(t), t = 1 / (1 + s a), where q is a polynomial
// fitted to it (least squares of the relative error, the weights raised where that is largest).
// Half types: one for all a, off by 1.8e-6 relative, a hundredth of their rounding, at half the instructions of the error
// function (2000 x 60 -> 5000 in bfloat16, forward and backward, 85 -> 66 us).
// float32: from a = 1 on, off by 8e-8; below it 1/2 + z r(z^2), off by 4e-8, where e t q(t) would lose two bits.  P then has a
// relative error of 1.4e-7 for positive z, 1e-6 down to -3 and 4e-6 down to -9, the last from the exponent's rounding.  (1 + erf
// cancels there: at z = -5 it is off by 4 %.  The complementary error function is as good as this and costs 885 us for 681 at
// 16384 x 4096 -> 120, forward and backward, where backward works out a slope 64 times; with erf 740.)
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    e = fast_exp2(-0.5f * kLog2e * z * z);
    const float a = fabsf(z);
    if constexpr (sizeof(T) == 4) {
        const float t = __builtin_amdgcn_rcpf(fmaf(0.25f, a, 1.f)), zz = z * z;
        float q = -0.045124784111976624f;
        q = fmaf(q, t, 0.1043723002076149f);
        q = fmaf(q, t, -0.01647164486348629f);
        q = fmaf(q, t, 0.08863063901662827f);
        q = fmaf(q, t, 0.07475871592760086f);
        q = fmaf(q, t, 0.09441080689430237f);
        q = fmaf(q, t, 0.09966612607240677f);
        q = fmaf(q, t, 0.09973771125078201f);
        q *= e * t;
        float r = 9.423524170415476e-05f;
        r = fmaf(r, zz, -0.001169353723526001f);
        r = fmaf(r, zz, 0.009967196732759476f);
        r = fmaf(r, zz, -0.06648958474397659f);
        r = fmaf(r, zz, 0.3989422619342804f);
        return a < 1.f ? fmaf(r, z, 0.5f) : z > 0.f ? 1.f - q : q;
    } else {
        const float t = __builtin_amdgcn_rcpf(fmaf(0.27f, a, 1.f));
        float q = -0.06008049888899402f;
        q = fmaf(q, t, 0.15620462423136175f);
        q = fmaf(q, t, -0.021565300509812337f);
        q = fmaf(q, t, 0.11616217791854966f);
        q = fmaf(q, t, 0.09317027342324012f);
        q = fmaf(q, t, 0.10842423982399171f);
        q = fmaf(q, t, 0.10768500957219908f);
        q *= e * t;
        return z > 0.f ? 1.f - q : q;
    }
}

template <typename T>
__device__ __forceinline__ float act_value(int act, float z) {
    switch (act) {
        case kActRelu: return z < 0.f ? 0.f : z;   // (a NaN stays one)
        case kActGelu: {
            float e;
            return z * normal_cdf<T>(z, e);
        }
        case kActSilu: return z * sigmoid(z);
        default: return z;
    }
}
// (z is cut to where the second terms are 0 in float32: at an infinity, which a kept half-precision z may be, they would be NaN)
template <typename T>
__device__ __forceinline__ float act_slope(int act, float z) {
    switch (act) {
        case kActRelu: return z > 0.f ? 1.f : z != z ? z : 0.f;
        case kActGelu: {
            const float c = fminf(fmaxf(z, -30.f), 30.f);
            float e;
            const float p = normal_cdf<T>(z, e);
            return p + c * kInvSqrt2Pi * e;
        }
        case kActSilu: {
            const float s = sigmoid(z), c = fminf(fmaxf(z, -100.f), 100.f);
            return s * (1.f + c * (1.f - s));
        }
        default: return 1.f;
    }
}

// The kept pre-activation.  In the half types it is rounded (the slope of gelu and silu then moves by
// less than their outputs' own rounding); a positive value never becomes zero, where relu's slope jumps.
template <typename T>
__device__ __forceinline__ T keep_z(float z) {
    const T r = from_f32<T>(z);
    if (z > 0.f && to_f32(r) == 0.f) return __builtin_bit_cast(T, (uint16_t)1);
    return r;
}
template <>
__device__ __forceinline__ float keep_z<float>(float z) {
    return z;
}

// A few neighbouring values of one row of the forward product through the epilogue.
template <typename T, int V>
__device__ __forceinline__ void act_values(int act, float (&v)[V]) {
    switch (act) {       // (the same for everybody: the loops stay small)
        case kActRelu:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = act_value<T>(kActRelu, v[e]);
            break;
        case kActGelu:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = act_value<T>(kActGelu, v[e]);
            break;
        case kActSilu:
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = act_value<T>(kActSilu, v[e]);
            break;
        default: break;
    }
}
template <typename T, int V>
__device__ __forceinline__ void slope_values(int act, float (&g)[V], const T (&z)[V]) {
    switch (act) {
        case kActRelu:
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] *= act_slope<T>(kActRelu, to_f32(z[e]));
            break;
        case kActGelu:
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] *= act_slope<T>(kActGelu, to_f32(z[e]));
            break;
        case kActSilu:
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] *= act_slope<T>(kActSilu, to_f32(z[e]));
            break;
        default: break;
    }
}
// V neighbouring elements at p, of which `count` are there
template <typename T, int V>
__device__ __forceinline__ void take_run(T (&v)[V], const T* __restrict__ p, long long count) {
    if (count >= V) {
        __builtin_memcpy(v, p, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = e < count ? p[e] : T(0);
    }
}
template <typename T, int V>
__device__ __forceinline__ void add_run(float (&v)[V], const T* __restrict__ p, int count) {
    T in[V];
    take_run<T, V>(in, p, count);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] += to_f32(in[e]);
}
template <typename T, int V, bool kKeep = false>
__device__ __forceinline__ void store_run(const float (&v)[V], T* __restrict__ p, int count) {
    T out[V];
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = kKeep ? keep_z<T>(v[e]) : from_f32<T>(v[e]);
    if (count >= V) {
        __builtin_memcpy(p, out, sizeof(out));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < count) p[e] = out[e];
    }
}
// v: z without the bias, columns [j, j + count) of row i (count <= V); `added`: the residual there, if there is one
template <typename T, int V>
__device__ __forceinline__ void forward_run(float (&v)[V], const float (&bias)[V], bool has_residual, const T (&added)[V], long long at,
                                            int count, int act, T* __restrict__ y, T* __restrict__ zk) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] += bias[e];
    if (zk) store_run<T, V, true>(v, zk + at, count);
    act_values<T, V>(act, v);
    if (has_residual) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] += to_f32(added[e]);
    }
    store_run<T, V>(v, y + at, count);
}
template <typename T, int V>
__device__ __forceinline__ void forward_out(float (&v)[V], long long i, long long j, int count, long long n, int act,
                                            const T* __restrict__ bias, const T* __restrict__ residual, long long ldr,
                                            T* __restrict__ y, T* __restrict__ zk) {
    float b[V] = {};
    T added[V];
    if (bias) add_run<T, V>(b, bias + j, count);
    if (residual) take_run<T, V>(added, residual + i * ldr + j, count);
    forward_run<T, V>(v, b, residual != nullptr, added, i * n + j, count, act, y, zk);
}

// ------------------------------------------------------------------ tiles of 64 x 64, or 128 x 32, any shape

constexpr int kDepth = 32, kThreads = 256;
constexpr int kTileSize = 4096;      // values of C in either

template <typename T>
struct Lds {
    static constexpr int LD = sizeof(T) == 4 ? kDepth + 4 : kDepth + 8;   // rows start on 16 bytes, four banks apart
    // Where element c of row r of a step lies.  The 16-byte pieces of every eight rows are exchanged differently: an operand
    // that lies across the contraction is written a column of every eighth row at a time.
    static __device__ __forceinline__ int at(int r, int c) { return r * LD + (c ^ (sizeof(T) == 4 ? 4 * ((r >> 3) & 7) : 8 * ((r >> 3) & 3))); }
};

// V neighbouring elements of a row of a step
template <typename T, int V>
__device__ __forceinline__ void put_run(T* lds, int r, int c, const T (&v)[V]) {
    constexpr int kPiece = V * sizeof(T) < 16 ? V : 16 / sizeof(T);
#pragma unroll
    for (int e = 0; e < V; e += kPiece)
        __builtin_memcpy(__builtin_assume_aligned(lds + Lds<T>::at(r, c + e), kPiece * sizeof(T)), v + e, kPiece * sizeof(T));
}

struct TileArgs {
    const void *a, *b;             // forward: x, w;  dx: -, w;  dw: -, x
    const void *z, *dy;
    const void *bias, *residual;
    long long lda, ldb, ldr;
    long long rows, cols, depth;   // of C and of the contraction
    long long n;                   // row length of z, dy, y
    int act, splits, lanes;
    unsigned tiles_i, tiles;       // tiles of C one below the other, and all
    long long split_len;
    void *out, *keep, *dbias;
    float *part, *part_bias;       // [splits][rows][cols], [splits][rows]
};

template <typename T, int TN>
struct TileLds {
    union {
        struct {
            __align__(16) T a[kTileSize / TN * Lds<T>::LD];
            __align__(16) T b[TN * Lds<T>::LD];
        };
        __align__(16) float c[kTileSize];
    };
};

// C leaves through LDS: an accumulator holds one column of four rows a lane, memory wants runs of columns.  A tile of TN
// columns lies row by row, every second group of four rows with its halves (or neighbouring rows) exchanged, so that the
// two halves of a wave, four rows apart, write to different banks.
template <int TN>
__device__ __forceinline__ int place(int row, int col) {
    return TN == 64 ? row * 64 + (col ^ ((row & 4) << 3)) : (row ^ ((row >> 2) & 1)) * 32 + col;
}
template <int TN>
__device__ __forceinline__ void put_quadrant(const f32x16& acc, float* c, int i, int j) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
#pragma unroll
    for (int r = 0; r < 16; ++r) c[place<TN>(i + 8 * (r >> 2) + 4 * half + (r & 3), j + (lane & 31))] = acc[r];
}
// A tile from LDS through the epilogue, eight columns at a time, by kT threads: the same columns every time, so
// that the bias is fetched once, and the residuals of a few rows are fetched before any of them is used.
template <typename T, int OP, int kT, int TN>
__device__ __forceinline__ void tile_out(const TileArgs& p, const float* c, long long i0, long long j0, int t) {
    constexpr int kInRow = TN / 8, kRuns = (kTileSize / 8 + kT - 1) / kT, kBatch = kRuns < 4 ? kRuns : 4;
    const int col = (t % kInRow) * 8;
    const long long j = j0 + col;
    if (j >= p.cols || t >= kTileSize / 8) return;
    const int count = (int)min(8ll, p.cols - j);
    float bias[8] = {};
    if (OP == kForward && p.bias) add_run<T, 8>(bias, static_cast<const T*>(p.bias) + j, count);
    const T* residual = OP == kForward ? static_cast<const T*>(p.residual) : nullptr;
#pragma unroll 1
    for (int r0 = 0; r0 < kRuns; r0 += kBatch) {
        T added[kBatch][8];
        if (residual) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const long long i = i0 + (t + (r0 + u) * kT) / kInRow;
                take_run<T, 8>(added[u], residual + i * p.ldr + j, i < p.rows ? count : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int row = (t + (r0 + u) * kT) / kInRow;
            const long long i = i0 + row;
            if (i >= p.rows) continue;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(c + place<TN>(row, col)), hi = *reinterpret_cast<const f32x4*>(c + place<TN>(row, col + 4));
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (OP == kForward)
                forward_run<T, 8>(v, bias, residual != nullptr, added[u], i * p.n + j, count, p.act, static_cast<T*>(p.out),
                                  static_cast<T*>(p.keep));
            else
                store_run<T, 8>(v, static_cast<T*>(p.out) + i * p.cols + j, count);
        }
    }
}

// Piece `piece` of the work on one product: a tile of C, and within it a split of the contraction.  A group of four waves
// makes a tile, each wave 32 x 32 of it, in steps of 32 along the contraction, fetched one step ahead.  Where the
// pieces are too few to fill the chip, G groups share one: every G-th step each, added up in their order.
template <typename T, int OP, int G, int TN>
__device__ __forceinline__ void tile_product(const TileArgs& p, unsigned piece, TileLds<T, TN>* lds) {
    constexpr int TM = kTileSize / TN;
    constexpr int kRunsA = TM / 64, kRunB = TN / 8;      // runs of eight a thread fetches of A's step; length of its one of B's
    const int group = G == 1 ? 0 : wave_id() / 4, wave = wave_id() % 4;
    const int t = threadIdx.x % kThreads, lane = t & 63;
    T *as = lds[group].a, *bs = lds[group].b;
    const unsigned split = piece / p.tiles, tile = piece - split * p.tiles, tile_j = tile / p.tiles_i;
    const long long i0 = (long long)(tile - tile_j * p.tiles_i) * TM, j0 = (long long)tile_j * TN;
    const long long c_lo = (long long)split * p.split_len;
    const long long c_hi = min(p.depth, c_lo + p.split_len);
    const T* __restrict__ a = static_cast<const T*>(p.a);
    const T* __restrict__ b = static_cast<const T*>(p.b);
    const T* __restrict__ z = static_cast<const T*>(p.z);
    const T* __restrict__ dy = static_cast<const T*>(p.dy);

    // This thread's runs of each operand's step: along the contraction, a few threads a row, or
    // across it, a few threads a column, whichever way its elements lie next to each other.
    constexpr bool kAlongA = OP != kDw, kAlongB = OP == kForward;
    constexpr int kInA = kAlongA ? kDepth / 8 : 8, kInB = kAlongB ? kDepth / kRunB : TN / kRunB;
    const int ca = kAlongA ? (t % kInA) * 8 : t / kInA, ra = kAlongA ? t / kInA : (t % kInA) * 8;
    const int cb = kAlongB ? (t % kInB) * kRunB : t / kInB, rb = kAlongB ? t / kInB : (t % kInB) * kRunB;

    T va[kRunsA][8], vb[kRunB];
    float dsum[kRunsA][8] = {};
    auto load = [&](long long c0) {
#pragma unroll
        for (int u = 0; u < kRunsA; ++u) {
            const long long r = i0 + ra + 64 * u, c = c0 + ca;
            const bool there = r < p.rows && c < c_hi;
            const long long count = there ? (kAlongA ? c_hi - c : p.rows - r) : 0;
            if constexpr (OP == kForward) {
                take_run<T, 8>(va[u], a + r * p.lda + c, count);
            } else {
                const long long at = OP == kDx ? r * p.n + c : c * p.n + r;
                take_run<T, 8>(va[u], dy + at, count);
                float g[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = to_f32(va[u][e]);
                if (p.act != kActNone) {
                    T vz[8];
                    take_run<T, 8>(vz, z + at, count);
                    slope_values(p.act, g, vz);
                    // (dz as the matrix instructions take it: in the half types one rounding more, which makes the errors of
                    // dx and dw 1.45 times those of their own rounding; a second plane of dz would double both products)
#pragma unroll
                    for (int e = 0; e < 8; ++e) va[u][e] = from_f32<T>(g[e]);
                }
                if (OP == kDw) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) dsum[u][e] += g[e];
                }
            }
        }
        {
            const long long r = j0 + rb, c = c0 + cb;
            const long long count = b && r < p.cols && c < c_hi ? (kAlongB ? c_hi - c : p.cols - r) : 0;
            take_run<T, kRunB>(vb, b + (kAlongB ? r * p.ldb + c : c * p.ldb + r), count);
        }
    };

    f32x16 acc = {};
    const int wi = (TN == 64 ? wave & 1 : wave) * 32, wj = TN == 64 ? (wave >> 1) * 32 : 0;     // this wave's part
    const int wr = wi + (lane & 31), wc = wj + (lane & 31), half = lane >> 5;
    load(c_lo + group * kDepth);
    for (long long c0 = c_lo; c0 < c_hi; c0 += G * kDepth) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kRunsA; ++u) {
            if constexpr (kAlongA) {
                put_run<T, 8>(as, ra + 64 * u, ca, va[u]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) as[Lds<T>::at(ra + 64 * u + e, ca)] = va[u][e];
            }
        }
        if constexpr (kAlongB) {
            put_run<T, kRunB>(bs, rb, cb, vb);
        } else {
#pragma unroll
            for (int e = 0; e < kRunB; ++e) bs[Lds<T>::at(rb + e, cb)] = vb[e];
        }
        __syncthreads();
        if (c0 + G * kDepth < c_hi) load(c0 + (G + group) * kDepth);
        if constexpr (sizeof(T) == 4) {
            // the two halves of the wave take four neighbouring steps of the contraction each: any order of them
            // gives the same sum of products, and this one reads 16 bytes a lane
#pragma unroll
            for (int s = 0; s < kDepth / 8; ++s) {
                const f32x4 fa = *reinterpret_cast<const f32x4*>(&as[Lds<T>::at(wr, s * 8 + half * 4)]);
                const f32x4 fb = *reinterpret_cast<const f32x4*>(&bs[Lds<T>::at(wc, s * 8 + half * 4)]);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[q], fb[q], acc, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < kDepth / 16; ++s) {
                if constexpr (__is_same(T, bf16)) {
                    const bf16x8 fa = *reinterpret_cast<const bf16x8*>(&as[Lds<T>::at(wr, s * 16 + half * 8)]);
                    const bf16x8 fb = *reinterpret_cast<const bf16x8*>(&bs[Lds<T>::at(wc, s * 16 + half * 8)]);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb, acc, 0, 0, 0);
                } else {
                    const f16x8 fa = *reinterpret_cast<const f16x8*>(&as[Lds<T>::at(wr, s * 16 + half * 8)]);
                    const f16x8 fb = *reinterpret_cast<const f16x8*>(&bs[Lds<T>::at(wc, s * 16 + half * 8)]);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa, fb, acc, 0, 0, 0);
                }
            }
        }
    }

    const int all = threadIdx.x;
    if (OP == kDw && p.dbias && tile_j == 0) {   // rows of C are the outputs: their sums of dz, from 32 threads of every group
        __syncthreads();
        float* s = lds[group].c;
#pragma unroll
        for (int u = 0; u < kRunsA; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[ca * TM + ra + 64 * u + e] = dsum[u][e];
        __syncthreads();
        if (all < TM && i0 + all < p.rows) {
            float sum = 0.f;
            for (int g = 0; g < G; ++g)
                for (int c = 0; c < kDepth; ++c) sum += lds[g].c[c * TM + all];
            if (p.splits > 1)
                p.part_bias[(long long)split * p.rows + i0 + all] = sum;
            else
                static_cast<T*>(p.dbias)[i0 + all] = from_f32<T>(sum);
        }
    }
    __syncthreads();     // the operands' tiles are read: C's values take their place
    put_quadrant<TN>(acc, lds[group].c, wi, wj);
    __syncthreads();
    float* c = lds[0].c;
    if (G > 1) {
        for (int e = all * 4; e < kTileSize; e += G * kThreads * 4) {
            f32x4 v = *reinterpret_cast<const f32x4*>(c + e);
#pragma unroll
            for (int g = 1; g < G; ++g) v += *reinterpret_cast<const f32x4*>(lds[g].c + e);
            *reinterpret_cast<f32x4*>(c + e) = v;
        }
        __syncthreads();
    }
    if (p.splits > 1) {
        for (int e = all; e < kTileSize; e += G * kThreads) {
            const long long i = i0 + e / TN, j = j0 + e % TN;
            if (i < p.rows && j < p.cols) p.part[((long long)split * p.rows + i) * p.cols + j] = c[place<TN>(e / TN, e % TN)];
        }
    } else if (p.out) {
        tile_out<T, OP, G * kThreads, TN>(p, c, i0, j0, all);
    }
}

template <typename T, int G, int TN>
__global__ __launch_bounds__(kThreads* G) void linear_tile_forward_kernel(TileArgs p) {
    __shared__ TileLds<T, TN> lds[G];
    tile_product<T, kForward, G, TN>(p, blockIdx.x, lds);
}
// both products of the backward pass in one launch, the first pieces_dx blocks on dx
template <typename T, int G, int TN>
__global__ __launch_bounds__(kThreads* G) void linear_tile_backward_kernel(TileArgs dx, unsigned pieces_dx, TileArgs dw) {
    __shared__ TileLds<T, TN> lds[G];
    if (blockIdx.x < pieces_dx)
        tile_product<T, kDx, G, TN>(dx, blockIdx.x, lds);
    else
        tile_product<T, kDw, G, TN>(dw, blockIdx.x - pieces_dx, lds);
}

// Joins the splits of the contraction, in their order.
template <typename T, int OP>
__device__ __forceinline__ void join_splits(const TileArgs& p) {
    const long long total = p.rows * p.cols;
    for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < total; e += (long long)gridDim.x * kThreads) {
        float s = 0.f;
#pragma unroll 8
        for (int q = 0; q < p.splits; ++q) s += p.part[q * total + e];
        float v[1] = {s};
        if (OP == kForward)
            forward_out<T, 1>(v, e / p.cols, e % p.cols, 1, p.n, p.act, static_cast<const T*>(p.bias),
                              static_cast<const T*>(p.residual), p.ldr, static_cast<T*>(p.out), static_cast<T*>(p.keep));
        else if (p.out)
            static_cast<T*>(p.out)[e] = from_f32<T>(s);
    }
    if (OP == kDw && p.dbias)
        for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < p.rows; e += (long long)gridDim.x * kThreads) {
            float s = 0.f;
            for (int q = 0; q < p.splits; ++q) s += p.part_bias[(long long)q * p.rows + e];
            static_cast<T*>(p.dbias)[e] = from_f32<T>(s);
        }
}
template <typename T, int OP>
__global__ __launch_bounds__(kThreads) void linear_join_kernel(TileArgs p) {
    join_splits<T, OP>(p);
}
template <typename T>
__global__ __launch_bounds__(kThreads) void linear_join_backward_kernel(TileArgs dx, TileArgs dw) {
    if (dx.splits > 1) join_splits<T, kDx>(dx);
    if (dw.splits > 1) join_splits<T, kDw>(dw);
}
inline unsigned join_blocks(long long elements) {
    const long long blocks = ceil_div(elements, kThreads);
    return (unsigned)(blocks < 4096 ? blocks : 4096);
}

// Up to this many pieces, four groups of waves share each: there is room on the chip for all of them, and a piece's
// steps, each as long as a fetch from memory takes, become a quarter.  With one group / four, float32:
// 1024 x 480 -> 1024 25.5 / 17.3 us, 256 x 128 -> 30 (four steps) 6.9 / 6.3; but 256 x 50 -> 128 (two) 5.1 / 6.5.
constexpr unsigned kFewPieces = 256;
constexpr int kGroups = 4;
inline bool share_pieces(long long pieces, long long longest) { return pieces <= kFewPieces && longest > 3 * kDepth; }

// Pieces of the contraction, of the least expected time: the products of one launch are cut into pieces of about the same
// number of steps, so many as a piece and the chip then take least for.  With two or more pieces at it, or one of
// four groups, a compute unit makes a step in about 0.75 us in float32 and 0.25 in the half types, and backward
// works out the slopes of 64 x 32 pre-activations besides (four groups of two products, whose pieces are not of one
// length, a third more); a join costs 6 us, and for each of a value's sums its fetch and its way to memory and back.
// Forward in float32, two blocks to a compute unit wherever the depth allows / this rule: 912 x 3499 -> 1098 170 / 100 us,
// 1024 x 1024 -> 1024 35 / 29, 33 x 1802 -> 12 15.5 / 10.3; forward and backward with gelu
// 20 x 3000 -> 1063 48 / 37, 191 x 732 -> 1446 53 / 46, 904 x 108 -> 4686 90 / 88, 2000 x 60 -> 5000 105 / 106
// (gelu by the error function; this rule now 77 and 92).
struct TilePlan {
    int splits;
    long long len;
};
struct TileShape {
    long long rows, cols, depth;
};
template <int N>
void plan_tiles(const TileShape (&of)[N], int tn, int esize, int act, bool backward, TilePlan (&plan)[N]) {
    static const float slope_us[] = {0.f, 0.05f, 0.6f, 0.3f};
    const double step = (esize == 4 ? 0.75 : 0.25) + (backward ? slope_us[act] : 0.f);
    long long tiles[N], steps[N], longest = 1;
    for (int i = 0; i < N; ++i) {
        tiles[i] = ceil_div(of[i].rows, kTileSize / tn) * ceil_div(of[i].cols, tn);
        steps[i] = tiles[i] ? ceil_div(of[i].depth, kDepth) : 0;
        plan[i] = {1, of[i].depth};
        if (steps[i] > longest) longest = steps[i];
    }
    double least = 1e30;
    for (long long s = 1; s <= 1024 && s <= longest; s += 1 + s / 4) {
        const long long len = ceil_div(longest, s);
        long long pieces = 0, work = 0;
        double sums = 0.;
        for (int i = 0; i < N; ++i) {
            const long long c = steps[i] > len ? ceil_div(steps[i], len) : 1;
            pieces += tiles[i] * c, work += tiles[i] * steps[i];
            if (c > 1) sums += (double)c * of[i].rows * of[i].cols;
        }
        double t = s > 1 ? 6.0 + 0.05 * N * s + sums * 2e-6 : 0.0;
        if (pieces <= kFewPieces) {
            t += (N == 2 ? 1.3 : 1.0) * step * round_up(len, kGroups);      // (a piece of up to three steps, by one group: no less)
        } else if (N == 1) {
            const long long at_once = ceil_div(pieces, 256);
            t += step * len * (at_once < 2 ? 2 : at_once);
        } else {
            const double alone = len * (2 * step > 1. ? 2 * step : 1.), all = step * (work / 256. + len);
            t += alone > all ? alone : all;
        }
        if (t >= least) continue;
        least = t;
        for (int i = 0; i < N; ++i) {
            plan[i] = {1, of[i].depth};
            if (steps[i] > len) plan[i] = {(int)ceil_div(steps[i], len), len * kDepth};
        }
    }
}
size_t part_bytes(const TileShape& of, const TilePlan& plan) {
    return plan.splits > 1 ? sizeof(float) * (size_t)plan.splits * ((size_t)of.rows * of.cols + of.rows) : 0;
}

// Columns of a tile for C = A B^T.  With at most 32 columns half of a 64 x 64 tile's arithmetic is for nothing, but its tiles
// are twice as many, which a small A needs more.  Microseconds with 64 and 32 columns:
// float32 forward 10412 x 2000 -> 30 42.5 / 31.0, 1024 x 2000 -> 30 16.4 / 17.2; backward 4096 x 30 -> 4096 97.7 / 75.5,
// 2048 x 30 -> 2048 41.1 / 35.7, 1024 x 30 -> 1024 27.5 / 28.5; bfloat16 62.6 / 53.1, 28.3 / 24.9, 20.6 / 21.6.
inline int tile_width(long long cols, long long size_of_a) { return cols <= 32 && size_of_a >= 2097152 ? 32 : 64; }

// fills in the splits of a product whose partial sums start at ws; returns its number of pieces
unsigned set_tiles(TileArgs& p, int tn, const TilePlan& plan, void* ws) {
    p.splits = plan.splits, p.split_len = plan.len;
    p.part = static_cast<float*>(ws);
    p.part_bias = p.part + (size_t)p.splits * p.rows * p.cols;
    p.tiles_i = (unsigned)ceil_div(p.rows, kTileSize / tn);
    p.tiles = (unsigned)(p.tiles_i * ceil_div(p.cols, tn));
    return p.tiles * (unsigned)p.splits;
}

// ------------------------------------------------------------------ up to eight rows
//
// With a handful of rows the layer is one reading of w: every lane streams 16-byte pieces of w's rows
// past the few rows of x (forward), or of dz (dx), in float32 FMAs.  Bound by that reading: 1 x 4096 -> 16384 in bfloat16
// with silu and residual 24.6 us, 5.5 TB/s.

constexpr int kFewRows = 8;
constexpr int kFewCols = 4;      // rows of w a wave has in hand at a time: each piece of x serves four of w

// y: p.lanes lanes (8 to 64, a power of two, by the length of a row) share kFewCols rows of w.
template <typename T, int M>
__global__ __launch_bounds__(kThreads) void linear_few_rows_kernel(TileArgs p) {
    constexpr int V = Vec16<T>::N;
    const int lane = threadIdx.x & (p.lanes - 1);
    const long long j0 = ((long long)blockIdx.x * (kThreads / p.lanes) + threadIdx.x / p.lanes) * kFewCols;
    const T* __restrict__ x = static_cast<const T*>(p.a);
    const T* __restrict__ w = static_cast<const T*>(p.b);
    const T *xr[M], *wr[kFewCols];
#pragma unroll
    for (int i = 0; i < M; ++i) xr[i] = x + min((long long)i, p.rows - 1) * p.lda;
#pragma unroll
    for (int j = 0; j < kFewCols; ++j) wr[j] = w + min(j0 + j, p.cols - 1) * p.ldb;
    float acc[M][kFewCols] = {};
    const long long pieces = p.depth / V;
#pragma unroll 2
    for (long long c = lane; c < pieces; c += p.lanes) {
        float fw[kFewCols][V];
        Vec16<T> vw[kFewCols], vx[M];
#pragma unroll
        for (int j = 0; j < kFewCols; ++j) vw[j] = load_vec(wr[j] + c * V);
#pragma unroll
        for (int i = 0; i < M; ++i) vx[i] = load_vec(xr[i] + c * V);
#pragma unroll
        for (int j = 0; j < kFewCols; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) fw[j][e] = vw[j].get(e);
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float f = vx[i].get(e);
#pragma unroll
                for (int j = 0; j < kFewCols; ++j) acc[i][j] = fmaf(f, fw[j][e], acc[i][j]);
            }
    }
    const long long c = pieces * V + lane;      // fewer than V left
    if (c < p.depth)
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int j = 0; j < kFewCols; ++j) acc[i][j] = fmaf(to_f32(xr[i][c]), to_f32(wr[j][c]), acc[i][j]);
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < kFewCols; ++j) {
            float z = acc[i][j];
            for (int off = p.lanes >> 1; off; off >>= 1) z += __shfl_xor(z, off);
            acc[i][j] = z;
        }
    if (lane >= M || lane >= p.rows || j0 >= p.cols) return;     // a lane for each row: all its values at once
    float v[kFewCols];
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int j = 0; j < kFewCols; ++j) v[j] = (i == 0 || lane == i) ? acc[i][j] : v[j];
    forward_out<T, kFewCols>(v, lane, j0, (int)min((long long)kFewCols, p.cols - j0), p.n, p.act, static_cast<const T*>(p.bias),
                             static_cast<const T*>(p.residual), p.ldr, static_cast<T*>(p.out), static_cast<T*>(p.keep));
}

// dx: a block takes one piece of columns per lane (512 columns in the half types) and `split_len` rows of w, its
// waves every fourth of them; dz of those rows is worked out once, into LDS.
constexpr int kFewDepth = 256;   // longest split
template <typename T, int M>
__global__ __launch_bounds__(kThreads) void linear_few_rows_dx_kernel(TileArgs p) {
    constexpr int V = Vec16<T>::N;
    __shared__ float dz[M][kFewDepth];
    __shared__ float meet[kThreads / 64][64 * V];
    const int t = threadIdx.x, lane = t & 63, wave = wave_id();
    const long long c0 = ((long long)blockIdx.x * 64 + lane) * V;
    const long long lo = (long long)blockIdx.y * p.split_len;
    const int len = (int)(min(p.depth, lo + p.split_len) - lo);
    const T* __restrict__ w = static_cast<const T*>(p.b);
    const T* __restrict__ dy = static_cast<const T*>(p.dy);
    const T* __restrict__ z = static_cast<const T*>(p.z);
    for (int e = t; e < M * len; e += kThreads) {
        const int i = e / len, r = e - i * len;
        float g = 0.f;
        if (i < p.rows) {
            const long long at = i * p.n + lo + r;
            g = to_f32(dy[at]);
            if (p.act != kActNone) g *= act_slope<T>(p.act, to_f32(z[at]));
        }
        dz[i][r] = g;
    }
    __syncthreads();
    float acc[M][V] = {};
    const bool whole = c0 + V <= p.cols;
    const int rest = (int)max(0ll, min((long long)V, p.cols - c0));
#pragma unroll 4
    for (int r = wave; r < len; r += kThreads / 64) {
        const T* row = w + (lo + r) * p.ldb + c0;
        float f[V];
        if (whole) {
            const Vec16<T> v = load_vec(row);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = v.get(e);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = e < rest ? to_f32(row[e]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const float g = dz[i][r];
#pragma unroll
            for (int e = 0; e < V; ++e) acc[i][e] = fmaf(g, f[e], acc[i][e]);
        }
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) meet[wave][lane * V + e] = acc[i][e];
        __syncthreads();
        if (i >= p.rows) continue;
        for (int e = t; e < 64 * V; e += kThreads) {
            const long long c = (long long)blockIdx.x * 64 * V + e;
            if (c >= p.cols) continue;
            const float s = (meet[0][e] + meet[1][e]) + (meet[2][e] + meet[3][e]);
            if (p.splits > 1)
                p.part[((long long)blockIdx.y * p.rows + i) * p.cols + c] = s;
            else
                static_cast<T*>(p.out)[i * p.cols + c] = from_f32<T>(s);
        }
    }
}

constexpr long long kMaxFewCols = 1 << 22;   // splits of dx fit a grid's second dimension
// Against tiles, which read w no faster but multiply on the matrix cores.  Microseconds, this way / tiles, in bfloat16 and
// float32:  1 row 4096 -> 16384 24 / 35, 45 / 94, and 50 -> 128 3.2 / 4.4, 3.5 / 6.1;  2 rows 4.2 / 4.4, 4.7 / 6.1;
// 4 rows 4096 -> 16384 28 / 35, 52 / 94, 4096 -> 4096 14.6 / 14.8, 21 / 30, 500 -> 1000 9.1 / 7.2, 9.1 / 9.2;
// 8 rows 4096 -> 16384 52 / 35, 71 / 94, 500 -> 1000 16 / 7.3, 16 / 9.5.
// (Blocks are as many as outputs allow, 16 to 128 each: for one or two rows of very many inputs and few outputs that is too few.
// 1 row 100 000 -> 16 53 / 18, 146 / 25; 20 000 -> 200 14.8 / 11.3, 17.4 / 17.1; 4096 -> 16 5.5 / 7.3 in bfloat16.)
bool has_few_rows(long long m, long long n, long long k, bool float32) {
    if (m < 1 || m > kFewRows || n > kMaxFewCols) return false;
    const long long weights = n * k;
    if (m <= 2) return true;
    if (m <= 4) return weights >= (float32 ? 1 << 20 : 1 << 24);
    return float32 && weights >= (1 << 24);
}
// dx, its splits and their join in two launches of their own: 1 row with dw, 4096 -> 4096 42 / 45, 59 / 69, 1000 -> 8000
// 37 / 27, 45 / 37;  8 rows 4096 -> 16384 159 / 150, 239 / 273.
bool has_few_rows_dx(long long m, long long n, long long k, bool float32) {
    return m >= 1 && m <= (float32 ? kFewRows : 4) && n <= kMaxFewCols && n * k >= (1 << 24);
}

void plan_few_dx(long long n, long long k, int esize, int& splits, long long& len) {
    const long long groups = ceil_div(k, 64 * (16 / esize));
    long long s = ceil_div(1024, groups);                 // four blocks for every compute unit
    if (s > n / 32) s = n / 32;                           // none shorter than eight rows a wave
    if (s < 1) s = 1;
    len = ceil_div(n, s);
    if (len > kFewDepth) len = kFewDepth;
    splits = (int)ceil_div(n, len);
}
size_t few_dx_bytes(long long m, long long n, long long k, int esize) {
    int splits;
    long long len;
    plan_few_dx(n, k, esize, splits, len);
    return splits > 1 ? sizeof(float) * (size_t)splits * m * k : 0;
}

template <typename T>
hipError_t run_few_rows(TileArgs p, hipStream_t stream) {
    p.lanes = 8;
    while (p.lanes < 64 && p.lanes * Vec16<T>::N < p.depth) p.lanes *= 2;
    const dim3 grid((unsigned)ceil_div(p.cols, kFewCols * (kThreads / p.lanes)));
    if (p.rows == 1) linear_few_rows_kernel<T, 1><<<grid, kThreads, 0, stream>>>(p);
    else if (p.rows == 2) linear_few_rows_kernel<T, 2><<<grid, kThreads, 0, stream>>>(p);
    else if (p.rows <= 4) linear_few_rows_kernel<T, 4><<<grid, kThreads, 0, stream>>>(p);
    else if constexpr (sizeof(T) == 4) linear_few_rows_kernel<T, 8><<<grid, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T>
hipError_t run_few_rows_dx(TileArgs p, void* ws, hipStream_t stream) {
    plan_few_dx(p.depth, p.cols, sizeof(T), p.splits, p.split_len);
    p.part = static_cast<float*>(ws);
    const dim3 grid((unsigned)ceil_div(p.cols, 64 * Vec16<T>::N), (unsigned)p.splits);
    if (p.rows == 1) linear_few_rows_dx_kernel<T, 1><<<grid, kThreads, 0, stream>>>(p);
    else if (p.rows == 2) linear_few_rows_dx_kernel<T, 2><<<grid, kThreads, 0, stream>>>(p);
    else if (p.rows <= 4) linear_few_rows_dx_kernel<T, 4><<<grid, kThreads, 0, stream>>>(p);
    else if constexpr (sizeof(T) == 4) linear_few_rows_dx_kernel<T, 8><<<grid, kThreads, 0, stream>>>(p);
    if (p.splits > 1) {
        linear_join_kernel<T, kDx><<<dim3(join_blocks(p.rows * p.cols)), kThreads, 0, stream>>>(p);
    }
    return hipGetLastError();
}

// ------------------------------------------------------------------ large products
//
// C[i, j] = sum_c A[i, c] B[j, c] on 16-bit operands.  A block owns a BM x BN tile; its operands pass through LDS in steps of
// 64 along the contraction, two buffers deep, written by the memory pipe itself (16 bytes a lane, no registers).
//
// An operand lies along the contraction (x and w forward, dz for dx) or across it ("turned": w for dx, dz and x for dw), and
// is used as it lies: its 64-wide piece of the contraction is 64 columns of BM rows, or 64 rows of BM columns, in LDS
// as in memory.  A lane's eight values of one row are then 16 bytes, or come from the LDS through
// its transposing read, which hands a lane four rows of its column (within 16 lanes, lane 4 e + l / 4 names the row of
// value e of lane l, four columns each).  The memory pipe writes lane after lane, row after row, and reading one chunk
// of many rows would hit the same banks every time; so a lane fetches the chunk that belongs there once rows
// are turned against each other, and the reads look it up.
// Bound by the LDS (three operand reads to eight products, and the memory pipe's writes) and the clock, beside the matrix pipe:
// 8192 x 4096 -> 4096 in bf16 235 us = 1.17 PFLOP/s, its backward pass 471; with gelu and residual 783 to 809 together on several
// cards, 890 with turned copies of the operands and the compiler's order of the reads.  Without the loads from memory it takes 202 us
// (with operands of zeros, at a higher clock, 152 and with the loads 186).  Tiles of 128 x 128 a wave take
// 247 us, steps of 32 with three on their way 272, a fifth slot for an operand 243.
//
// float32 operands come as three bf16 planes whose sum is the value to 2^-25 or better (to 2^-134 below 2^-108, where the planes'
// numbers end; an infinity makes NaN of the other planes' zeros): the product is
// the six products of planes that matter (the other three are below 2^-24 of the result), run as one
// contraction six times as long.  Six passes at the bf16 rate are 2.6 times as fast as float32 MFMA.

constexpr int kBK = 64;
constexpr long long kMaxLd = 1 << 22;    // a tile's 256 rows are addressed by 32-bit byte offsets
constexpr int kPlanes = 3, kPairs = 6;

struct Operand {
    const void* p;
    long long ld, plane;             // elements between rows, and between planes
    long long width;                 // elements of a row that may be read: a multiple of 8
    long long valid;                 // length of the contraction that is there; zeros are taken for the rest of its last step
};
struct GemmArgs {
    Operand a, b;
    long long rows, cols, depth;
    int pairs;                       // 1, or kPairs
    int splits, split_len;           // in steps
    unsigned tiles_i, tiles_j;
    TileArgs t;                      // the epilogue's part
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ const u32x4 kZeros = {0u, 0u, 0u, 0u};

// 64 lanes x 16 bytes from global memory to LDS at `lds` + 16 lane
__device__ __forceinline__ void load_to_lds(const char* g, char* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// none of the wave's memory operations and LDS reads under way; then all waves
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
}

// One operand's share of a tile: W rows of C's (or columns), of which `count` are there from `first` on.
template <typename T16, int W, int kWavesAll, bool kTurned>
struct TileOperand {
    static constexpr int kLoads = W / 8 / kWavesAll;                   // of this wave in each step
    static constexpr int kChunks = kTurned ? W / 8 : 8, kRowsPer = 64 / kChunks;
    static constexpr int kBytes = W * kBK * 2;
    static constexpr bool kIsTurned = kTurned;
    const char* base;
    unsigned off[kLoads];
    int at_chunk, at_row;           // (of a lane in each load) its chunk's first element, its row
    long long step_bytes, plane_bytes, valid;

    // `wave`: which of the block's
    __device__ __forceinline__ void init(const Operand& o, long long first, long long count, int wave) {
        const int lane = threadIdx.x & 63;
        at_row = lane / kChunks;
        // chunk numbers of eight rows differ in their low bits, or of four rows in the next two: a read of one chunk of
        // 8 rows, or of 32 bytes of 4 rows, then goes round the banks once
        int chunk = (lane % kChunks) ^ (kTurned ? 2 * ((wave * kRowsPer + at_row) & 3) : at_row & 7);
        plane_bytes = o.plane * 2;
        valid = o.valid;
        if constexpr (kTurned) {
            base = reinterpret_cast<const char*>(o.p) + first * 2;
            step_bytes = kBK * o.ld * 2;
            chunk = min(chunk, (int)min((long long)W, o.width - first) / 8 - 1);      // (columns behind the last: not used)
        } else {
            base = reinterpret_cast<const char*>(o.p) + first * o.ld * 2;
            step_bytes = kBK * 2;
        }
        at_chunk = chunk * 8;
        const int last = (int)min((long long)W, count) - 1;                            // (rows behind the last: not used)
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
            const int r = (q * kWavesAll + wave) * kRowsPer + at_row;
            off[q] = (unsigned)(kTurned ? r : min(r, last)) * (unsigned)(o.ld * 2) + chunk * 16;
        }
    }
    // step kb of plane `plane`; `edge`: it may reach behind the end of the contraction
    __device__ __forceinline__ void fetch(int plane, int kb, bool edge, char* lds, int wave) const {
        const char* g = base + plane * plane_bytes + kb * step_bytes;
        char* to = lds + wave * 1024;
        if (!edge) {
#pragma unroll
            for (int q = 0; q < kLoads; ++q) load_to_lds(g + off[q], to + q * kWavesAll * 1024);
        } else {
            const char* zeros = reinterpret_cast<const char*>(&kZeros);
#pragma unroll
            for (int q = 0; q < kLoads; ++q) {
                const int c = kTurned ? (q * kWavesAll + wave) * kRowsPer + at_row : at_chunk;
                load_to_lds((long long)kb * kBK + c < valid ? g + off[q] : zeros, to + q * kWavesAll * 1024);
            }
        }
    }
    // Where this lane reads from, for rows of C (columns) from `from` on, and the eight steps of the contraction that are
    // this half wave's of the sixteen from 16 kk on: along the contraction 16 bytes of a row for every 32 rows, at(kk) +
    // 32 rows f; across it two times 8 bytes, four steps apart, at(kk, f & 1) + 128 (f / 2).
    uint32_t start[2];
    static constexpr int kStepBytes = 16 * (W * 2), kHalf = 4 * (W * 2), kRows32 = 32 * (kBK * 2);
    __device__ __forceinline__ void init_reads(int from, const char* lds) {
        const int lane = threadIdx.x & 63, half = lane >> 5;
        const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds;
        if constexpr (kTurned) {
            const int s = lane & 15, row = 8 * half + (s >> 2);
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
                const int chunk = (from / 8 + 4 * odd + 2 * ((lane >> 4) & 1) + ((s & 3) >> 1)) ^ (2 * (s >> 2));
                start[odd] = base + row * (W * 2) + chunk * 16 + (s & 1) * 8;
            }
        } else {
            start[0] = base + (from + (lane & 31)) * (kBK * 2) + ((half ^ (lane & 7)) * 16);
            start[1] = 0;
        }
    }
    __device__ __forceinline__ uint32_t at(int kk, int odd = 0) const {
        return kTurned ? start[odd] + kk * kStepBytes : start[0] ^ (kk * 32);
    }
};

// A wave's fragments of sixteen steps of the contraction: 32 rows of C each (columns), eight steps a lane.
template <int F, bool kTurned>
struct Fragments {
    u32x4 whole[F];
    __device__ __forceinline__ u32x4 get(int f) const { return whole[f]; }
};
template <int F>
struct Fragments<F, true> {
    u32x2 part[2 * F];
    __device__ __forceinline__ u32x4 get(int f) const { return __builtin_shufflevector(part[2 * f], part[2 * f + 1], 0, 1, 2, 3); }
};

// One step of sixteen: C += the products of the fragments x, y, while the next ones are on their way from LDS.  Written
// out in one block with its wait, since the compiler gathers a step's reads in front of its products.  The products of a
// block go to different accumulators, and the next use of one is the same product of the next block, three others
// and two wait states (s_nop 1, which also keeps a copied fragment's distance) later: accumulating needs no more.  What reads
// the sums otherwise comes after settle().
#define SCMIAC_MUL(t, i, j) "v_mfma_f32_32x32x16_" t " %[c" #i #j "], %[x" #i "], %[y" #j "], %[c" #i #j "]\n\t"
#define SCMIAC_ROW(v, f, off) "ds_read_b128 %[" #v #f "], %[" #v "at0] offset:" #off "\n\t"
#define SCMIAC_TURNED(v, f, odd, off)                                            \
    "ds_read_b64_tr_b16 %[" #v #f "l], %[" #v "at" #odd "] offset:" #off "\n\t" \
    "ds_read_b64_tr_b16 %[" #v #f "h], %[" #v "at" #odd "] offset:%c[" #v "h" #off "]\n\t"
#define SCMIAC_BLOCK_4_2(t, a0, a1, a2, a3, b0, b1)                                                               \
    "s_nop 1\n\t" SCMIAC_MUL(t, 0, 0) a0 SCMIAC_MUL(t, 0, 1) a1 SCMIAC_MUL(t, 1, 0) a2 SCMIAC_MUL(t, 1, 1) a3      \
        SCMIAC_MUL(t, 2, 0) b0 SCMIAC_MUL(t, 2, 1) b1 SCMIAC_MUL(t, 3, 0) SCMIAC_MUL(t, 3, 1) "s_waitcnt lgkmcnt(0)"
#define SCMIAC_BLOCK_2_2(t, a0, a1, b0, b1) \
    "s_nop 1\n\t" SCMIAC_MUL(t, 0, 0) a0 b0 SCMIAC_MUL(t, 0, 1) a1 b1 SCMIAC_MUL(t, 1, 0) SCMIAC_MUL(t, 1, 1) "s_waitcnt lgkmcnt(0)"
#define SCMIAC_ROWS_4(v) SCMIAC_ROW(v, 0, 0), SCMIAC_ROW(v, 1, 4096), SCMIAC_ROW(v, 2, 8192), SCMIAC_ROW(v, 3, 12288)
#define SCMIAC_ROWS_2(v) SCMIAC_ROW(v, 0, 0), SCMIAC_ROW(v, 1, 4096)
#define SCMIAC_TURNED_4(v) SCMIAC_TURNED(v, 0, 0, 0), SCMIAC_TURNED(v, 1, 1, 0), SCMIAC_TURNED(v, 2, 0, 128), SCMIAC_TURNED(v, 3, 1, 128)
#define SCMIAC_TURNED_2(v) SCMIAC_TURNED(v, 0, 0, 0), SCMIAC_TURNED(v, 1, 1, 0)
#define SCMIAC_SUM_2 [c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c10] "+v"(c[1][0]), [c11] "+v"(c[1][1])
#define SCMIAC_SUM_4 SCMIAC_SUM_2, [c20] "+v"(c[2][0]), [c21] "+v"(c[2][1]), [c30] "+v"(c[3][0]), [c31] "+v"(c[3][1])
#define SCMIAC_OUT_ROWS_2(v, n) [v##0] "=&v"(n.whole[0]), [v##1] "=&v"(n.whole[1])
#define SCMIAC_OUT_ROWS_4(v, n) SCMIAC_OUT_ROWS_2(v, n), [v##2] "=&v"(n.whole[2]), [v##3] "=&v"(n.whole[3])
#define SCMIAC_OUT_TURNED_2(v, n) \
    [v##0l] "=&v"(n.part[0]), [v##0h] "=&v"(n.part[1]), [v##1l] "=&v"(n.part[2]), [v##1h] "=&v"(n.part[3])
#define SCMIAC_OUT_TURNED_4(v, n) \
    SCMIAC_OUT_TURNED_2(v, n), [v##2l] "=&v"(n.part[4]), [v##2h] "=&v"(n.part[5]), [v##3l] "=&v"(n.part[6]), [v##3h] "=&v"(n.part[7])
#define SCMIAC_AT_ROWS(v, at) [v##at0] "v"(at[0])
#define SCMIAC_AT_TURNED(v, at, half) [v##at0] "v"(at[0]), [v##at1] "v"(at[1]), [v##h0] "n"(half), [v##h128] "n"(half + 128)
#define SCMIAC_IN_2 [x0] "v"(x.get(0)), [x1] "v"(x.get(1)), [y0] "v"(y.get(0)), [y1] "v"(y.get(1))
#define SCMIAC_IN_4 SCMIAC_IN_2, [x2] "v"(x.get(2)), [x3] "v"(x.get(3))
#define SCMIAC_MULTIPLY(t)                                                                                                        \
    if constexpr (FA == 4 && !kTurnedA && !kTurnedB)                                                                              \
        asm volatile(SCMIAC_EXPAND(SCMIAC_BLOCK_4_2, t, SCMIAC_ROWS_4(a), SCMIAC_ROWS_2(b))                                       \
                     : SCMIAC_SUM_4, SCMIAC_OUT_ROWS_4(a, xn), SCMIAC_OUT_ROWS_2(b, yn)                                           \
                     : SCMIAC_IN_4, SCMIAC_AT_ROWS(a, at_a), SCMIAC_AT_ROWS(b, at_b)                                              \
                     : "memory");                                                                                                 \
    else if constexpr (FA == 4 && !kTurnedA)                                                                                      \
        asm volatile(SCMIAC_EXPAND(SCMIAC_BLOCK_4_2, t, SCMIAC_ROWS_4(a), SCMIAC_TURNED_2(b))                                     \
                     : SCMIAC_SUM_4, SCMIAC_OUT_ROWS_4(a, xn), SCMIAC_OUT_TURNED_2(b, yn)                                         \
                     : SCMIAC_IN_4, SCMIAC_AT_ROWS(a, at_a), SCMIAC_AT_TURNED(b, at_b, kHalfB)                                    \
                     : "memory");                                                                                                 \
    else if constexpr (FA == 4)                                                                                                   \
        asm volatile(SCMIAC_EXPAND(SCMIAC_BLOCK_4_2, t, SCMIAC_TURNED_4(a), SCMIAC_TURNED_2(b))                                   \
                     : SCMIAC_SUM_4, SCMIAC_OUT_TURNED_4(a, xn), SCMIAC_OUT_TURNED_2(b, yn)                                       \
                     : SCMIAC_IN_4, SCMIAC_AT_TURNED(a, at_a, kHalfA), SCMIAC_AT_TURNED(b, at_b, kHalfB)                          \
                     : "memory");                                                                                                 \
    else if constexpr (!kTurnedA && !kTurnedB)                                                                                    \
        asm volatile(SCMIAC_EXPAND(SCMIAC_BLOCK_2_2, t, SCMIAC_ROWS_2(a), SCMIAC_ROWS_2(b))                                       \
                     : SCMIAC_SUM_2, SCMIAC_OUT_ROWS_2(a, xn), SCMIAC_OUT_ROWS_2(b, yn)                                           \
                     : SCMIAC_IN_2, SCMIAC_AT_ROWS(a, at_a), SCMIAC_AT_ROWS(b, at_b)                                              \
                     : "memory");                                                                                                 \
    else if constexpr (!kTurnedA)                                                                                                 \
        asm volatile(SCMIAC_EXPAND(SCMIAC_BLOCK_2_2, t, SCMIAC_ROWS_2(a), SCMIAC_TURNED_2(b))                                     \
                     : SCMIAC_SUM_2, SCMIAC_OUT_ROWS_2(a, xn), SCMIAC_OUT_TURNED_2(b, yn)                                         \
                     : SCMIAC_IN_2, SCMIAC_AT_ROWS(a, at_a), SCMIAC_AT_TURNED(b, at_b, kHalfB)                                    \
                     : "memory");                                                                                                 \
    else                                                                                                                          \
        asm volatile(SCMIAC_EXPAND(SCMIAC_BLOCK_2_2, t, SCMIAC_TURNED_2(a), SCMIAC_TURNED_2(b))                                   \
                     : SCMIAC_SUM_2, SCMIAC_OUT_TURNED_2(a, xn), SCMIAC_OUT_TURNED_2(b, yn)                                       \
                     : SCMIAC_IN_2, SCMIAC_AT_TURNED(a, at_a, kHalfA), SCMIAC_AT_TURNED(b, at_b, kHalfB)                          \
                     : "memory")
#define SCMIAC_EXPAND(block, ...) block(__VA_ARGS__)

template <typename T16, int FA, int FB, bool kTurnedA, bool kTurnedB, int kHalfA, int kHalfB>
__device__ __forceinline__ void multiply(f32x16 (&c)[FA][FB], const Fragments<FA, kTurnedA>& x, const Fragments<FB, kTurnedB>& y,
                                         Fragments<FA, kTurnedA>& xn, Fragments<FB, kTurnedB>& yn, const uint32_t (&at_a)[2],
                                         const uint32_t (&at_b)[2]) {
    static_assert((FA == 4 || FA == 2) && FB == 2 && (kTurnedB || !kTurnedA), "the blocks there are");
    if constexpr (__is_same(T16, bf16)) {
        SCMIAC_MULTIPLY("bf16");
    } else {
        SCMIAC_MULTIPLY("f16");
    }
}
// the last products are done: the compiler does not know of them
template <int FA, int FB>
__device__ __forceinline__ void settle(f32x16 (&c)[FA][FB]) {
    if constexpr (FA == 4)
        asm volatile("s_nop 15\n\ts_nop 15" : SCMIAC_SUM_4);
    else
        asm volatile("s_nop 15\n\ts_nop 15" : SCMIAC_SUM_2);
}
template <typename T16, typename OutT, int BM, int BN, int WM, int WN, int OP>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64) void linear_gemm_kernel(GemmArgs p) {
    constexpr int kWavesN = BN / WN, kWavesAll = (BM / WM) * kWavesN;
    constexpr int FA = WM / 32, FB = WN / 32;
    constexpr bool kInParts = BM == 256;
    typedef TileOperand<T16, BM, kWavesAll, OP == kDw> OperandA;
    typedef TileOperand<T16, BN, kWavesAll, OP != kForward> OperandB;
    constexpr int kBytesA = OperandA::kBytes, kBytes = kBytesA + OperandB::kBytes;
    __shared__ __align__(128) char lds[2 * kBytes];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int wm = (wave / kWavesN) * WM, wn = (wave % kWavesN) * WN;

    // Blocks go to the eight XCDs in turn: give each XCD a run of tiles of its own, and within it walk
    // eight rows of tiles at a time, so that the tiles at work share their operands in that XCD's L2.
    const unsigned tiles = p.tiles_i * p.tiles_j;
    const unsigned xcd = blockIdx.x & 7, per = tiles / 8, extra = tiles % 8;
    unsigned id = xcd * per + min(xcd, extra) + (blockIdx.x >> 3);
    const unsigned group = 8 * p.tiles_j, first = id / group * 8;
    const unsigned high = min(8u, p.tiles_i - first);
    id %= group;
    const unsigned ti = first + id % high, tj = id / high;
    const long long i0 = (long long)ti * BM, j0 = (long long)tj * BN;
    const int k_blocks = (int)((p.depth + kBK - 1) / kBK);
    const bool ragged = p.depth % kBK != 0;
    const int s_lo = blockIdx.y * p.split_len, s_hi = min(k_blocks * p.pairs, s_lo + p.split_len);

    OperandA a;
    OperandB b;
    a.init(p.a, i0, p.rows - i0, wave);
    b.init(p.b, j0, p.cols - j0, wave);
    a.init_reads(wm, lds);
    b.init_reads(wn, lds + kBytesA);
    // half 0, 1: one operand of a step
    auto stage = [&](int step, int buf, int half) {
        int kb = step, pa = 0, pb = 0;
        if (p.pairs > 1) {
            const int pair = step / k_blocks;
            kb -= pair * k_blocks;
            // the small products first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
            pa = (pair == 0) ? 2 : (pair == 2 || pair == 3) ? 1 : 0;
            pb = (pair == 1) ? 2 : (pair == 2 || pair == 4) ? 1 : 0;
        }
        const bool edge = ragged && kb == k_blocks - 1;
        char* to = lds + buf * kBytes;
        if (half == 0)
            a.fetch(pa, kb, edge, to, wave);
        else
            b.fetch(pb, kb, edge, to + kBytesA, wave);
    };

    f32x16 acc[FA][FB] = {};
    const int half = lane >> 5, l31 = lane & 31;
    Fragments<FA, OperandA::kIsTurned> x, xn;
    Fragments<FB, OperandB::kIsTurned> y, yn;
    auto step16 = [&](int kk, int buf) {      // the products of x, y, and the fragments of kk from buffer buf in their place
        const uint32_t at_a[2] = {a.at(kk) + buf * kBytes, a.at(kk, 1) + buf * kBytes};
        const uint32_t at_b[2] = {b.at(kk) + buf * kBytes, b.at(kk, 1) + buf * kBytes};
        multiply<T16, FA, FB, OperandA::kIsTurned, OperandB::kIsTurned, OperandA::kHalf, OperandB::kHalf>(acc, x, y, xn, yn, at_a, at_b);
        x = xn, y = yn;
    };
    x = {}, y = {};                           // (whose products are zeros)
    stage(s_lo, 0, 0), stage(s_lo, 0, 1);
    if (s_lo + 1 < s_hi) {
        stage(s_lo + 1, 1, 0);
        if (!kInParts) stage(s_lo + 1, 1, 1);
    }
    wait_and_meet();
    step16(0, 0);
    // While one buffer is read, the next step is on its way to the other.  In the large tiles an operand at a time, between the
    // products: all of it at once would hold up the products behind it (8192 x 4096 -> 4096 250 us, in two parts 235; in
    // four, of which the last has too little time to land, 255).  In the small ones, two blocks of which share a
    // compute unit, all at once (2048 x 2048 -> 2048 28 us, in two parts 31).  Before its last sixteen products a wave has the last of a
    // buffer in hand: when they meet, the buffer can be filled anew, and the other has landed, this wave's share of
    // it, then everybody's.  (Behind the last step there is no other: what is read then is not used.)
    int buf = 0;
    for (int step = s_lo; step < s_hi; ++step) {
        if (kInParts && step + 1 < s_hi) stage(step + 1, buf ^ 1, 1);
#pragma unroll
        for (int kk = 1; kk < kBK / 16; ++kk) step16(kk, buf);
        wait_and_meet();
        if (step + 2 < s_hi) {
            stage(step + 2, buf, 0);
            if (!kInParts) stage(step + 2, buf, 1);
        }
        buf ^= 1;
        step16(0, buf);
    }
    settle(acc);

    if (p.splits > 1) {
#pragma unroll
        for (int f = 0; f < FA; ++f)
#pragma unroll
            for (int g = 0; g < FB; ++g) {
                const long long j = j0 + wn + g * 32 + l31;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const long long i = i0 + wm + f * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
                    if (i < p.rows && j < p.cols) p.t.part[((long long)blockIdx.y * p.rows + i) * p.cols + j] = acc[f][g][r];
                }
            }
        return;
    }
    static_assert(WN % 64 == 0 && WM % 64 == 0 && kWavesAll * kTileSize * 4 <= 2 * kBytes, "a 64 x 64 tile of LDS for every wave");
    __syncthreads();                             // the operands are read: the room is each wave's own now
    float* c = reinterpret_cast<float*>(lds) + wave * kTileSize;
#pragma unroll
    for (int m = 0; m < WM / 64; ++m)
#pragma unroll
        for (int n = 0; n < WN / 64; ++n) {
            wave_lds_fence();
#pragma unroll
            for (int q = 0; q < 4; ++q) put_quadrant<64>(acc[2 * m + (q >> 1)][2 * n + (q & 1)], c, (q >> 1) * 32, (q & 1) * 32);
            wave_lds_fence();
            tile_out<OutT, OP, 64, 64>(p.t, c, i0 + wm + m * 64, j0 + wn + n * 64, lane);
        }
}

// An operand of the large products from a matrix src [rows, cols] (or from dz = dy act'(z), given as src = dy and z) that
// cannot be read as it stands: rows padded with zeros to pc elements, float32 as three bf16 planes.
// `sums` [ceil(rows / 64)][cols]: what each 64 rows add up to, before any rounding.
struct PackArgs {
    const void *src, *z;
    long long ld, rows, cols, pc;
    int act;
    void* out;
    float* sums;
};
template <typename T>
struct Plane {
    typedef T type;
    static constexpr int N = 1;
};
template <>
struct Plane<float> {
    typedef bf16 type;
    static constexpr int N = kPlanes;
};
template <typename T>
__device__ __forceinline__ void split_planes(float v, typename Plane<T>::type (&o)[Plane<T>::N]) {
    if constexpr (sizeof(T) == 4) {
        // each plane is what the ones before leave; a value that rounds up to infinity, or is not finite,
        // is cut short instead, or stands in the first plane alone
        bf16 h = static_cast<bf16>(v);
        if (!(fabsf(static_cast<float>(h)) < INFINITY) && fabsf(v) < INFINITY)
            h = __builtin_bit_cast(bf16, (uint16_t)(__float_as_uint(v) >> 16));
        const bool finite = fabsf(v) < INFINITY;
        const float r1 = finite ? v - static_cast<float>(h) : 0.f;
        const bf16 m = static_cast<bf16>(r1);
        o[0] = h;
        o[1] = m;
        o[2] = static_cast<bf16>(r1 - static_cast<float>(m));
    } else {
        o[0] = from_f32<T>(v);      // (of dz the one rounding more that the small tiles make, too)
    }
}
template <typename T, bool kSlope>
__global__ __launch_bounds__(kThreads) void linear_pack_kernel(PackArgs p) {
    typedef typename Plane<T>::type P;
    constexpr int NP = Plane<T>::N;
    typedef P Four __attribute__((ext_vector_type(4)));
    __shared__ float part[16][64];
    const int t = threadIdx.x, q = (t & 15) * 4, r0 = t >> 4;
    const unsigned tiles_c = (unsigned)(p.pc / 64), tile_r = blockIdx.x / tiles_c;
    const long long c0 = (long long)(blockIdx.x - tile_r * tiles_c) * 64, y0 = (long long)tile_r * 64;
    const T* __restrict__ src = static_cast<const T*>(p.src);
    const T* __restrict__ z = static_cast<const T*>(p.z);
    P* out = static_cast<P*>(p.out);
    const long long left = p.cols - c0 - q;      // of this thread's four columns
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long r = y0 + r0 + 16 * i;
        if (r >= p.rows) continue;
        T in[4];
        float v[4];
        take_run<T, 4>(in, src + r * p.ld + c0 + q, left);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to_f32(in[e]);
        if (kSlope) {
            take_run<T, 4>(in, z + r * p.ld + c0 + q, left);
            slope_values(p.act, v, in);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v[e];
        if (out) {
            Four w[NP];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                P o[NP];
                split_planes<T>(v[e], o);
#pragma unroll
                for (int s = 0; s < NP; ++s) w[s][e] = o[s];
            }
#pragma unroll
            for (int s = 0; s < NP; ++s) *reinterpret_cast<Four*>(out + (s * p.rows + r) * p.pc + c0 + q) = w[s];
        }
    }
    if (p.sums) {
#pragma unroll
        for (int e = 0; e < 4; ++e) part[r0][q + e] = sum[e];
        __syncthreads();
        if (t < 64 && c0 + t < p.cols) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += part[i][t];
            p.sums[(long long)tile_r * p.cols + c0 + t] = s;
        }
    }
}

// dbias from the sums of the pack: 64 columns a block, four runs of partial sums each, joined in order
template <typename T>
__global__ __launch_bounds__(kThreads) void linear_bias_kernel(const float* __restrict__ sums, long long parts, long long cols,
                                                               T* __restrict__ dbias) {
    __shared__ float run[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long c = (long long)blockIdx.x * 64 + lane;
    const long long len = (parts + 3) / 4, lo = w * len, hi = min(parts, lo + len);
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (long long i = lo; i < hi; ++i) s += sums[i * cols + c];
    }
    run[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < cols) dbias[c] = from_f32<T>((run[0][lane] + run[1][lane]) + (run[2][lane] + run[3][lane]));
}

// Whether a layer goes through the large tiles: with at least 64 inputs and outputs, from 2^30 multiply-adds on (in float32,
// of which the small tiles' instructions do a quarter of what six products of planes cost the large ones, with
// at least 128 and from three times as many on); below, packing the operands and filling a few tiles cost more than the
// 64 x 64 tiles' slower inner loop.  Forward and backward, large / small tiles, in microseconds: bfloat16
// 1024 x 512 -> 1024 45 / 40, 765 x 2937 -> 252 57 / 44, 2048 x 1024 -> 1024 57 / 64, 8192 x 64 -> 8192 153 / 164; float32
// 1024 x 1024 -> 1024 124 / 81, 10412 x 2000 -> 128 321 / 205, 912 x 3499 -> 1098 270 / 280 and with silu 270 / 364,
// 16384 x 4096 -> 120 760 / 571 and with gelu by the error function 766 / 774 (small now 681), 100 000 x 64 -> 512 664 / 261.
bool is_large(long long rows, long long cols, long long depth, int dtype) {
    const int least = dtype == 0 ? 128 : 64;
    if (rows <= kFewRows || cols < least || depth < least) return false;
    if (rows > kMaxLd || cols > kMaxLd || depth > kMaxLd) return false;
    return (double)rows * (double)cols * (double)depth >= (dtype == 0 ? 3221225472.0 : 1073741824.0);
}

struct GemmPlan {
    bool wide;               // 256 x 256 tiles (8 waves), or 128 x 128 (4 waves)
    unsigned tiles_i, tiles_j;
    int steps, splits, split_len;
    size_t part_bytes;
};
GemmPlan plan_gemm(long long rows, long long cols, long long depth, int pairs) {
    GemmPlan g;
    g.steps = (int)ceil_div(depth, kBK) * pairs;
    // By expected time.  A step of one small tile on a compute unit takes 0.68 us, of two at a time 1.13; of a large one,
    // which has the unit to itself, 1.85 with all units at work and less with fewer.  Where there are few small tiles the
    // contraction is cut into pieces; joining costs a launch and the partial sums' way to memory and back (4 bytes a value
    // each way, 4 TB/s).  bfloat16 with large / small tiles, 4096 inputs: 4096 x 4096 123 / 146 us, 3584 x 3584 107 / 130,
    // 2816 x 2560 92 / 79, 3840 x 4864 (29 large tiles over) 195 / 176; 2048 x 2048 x 2048 in two pieces 41, in one 28.
    const long long t256 = ceil_div(rows, 256) * ceil_div(cols, 256), t128 = ceil_div(rows, 128) * ceil_div(cols, 128);
    const long long over = t256 % 256;
    const double large = g.steps * ((t256 / 256) * 1.85 + (over ? 1.35 + over / 512.0 : 0.0));
    long long s = 1;
    double small = 1e30;
    for (long long c = 1; c <= 32 && (c == 1 || c * 4 <= g.steps); ++c) {
        const long long blocks = ceil_div(t128 * c, 256);       // on the busiest compute unit
        const double step = (blocks / 2) * 1.13 + (blocks % 2) * 0.68;
        const double t = (double)ceil_div(g.steps, c) * step + (c > 1 ? 6.0 + c * (double)rows * cols * 2e-6 : 0.0);
        if (t < small) small = t, s = c;
    }
    g.wide = large < small;
    if (g.wide) s = 1;
    const int b = g.wide ? 256 : 128;
    g.tiles_i = (unsigned)ceil_div(rows, b);
    g.tiles_j = (unsigned)ceil_div(cols, b);
    g.split_len = (int)ceil_div(g.steps, s);
    g.splits = (int)ceil_div(g.steps, g.split_len);
    g.part_bytes = g.splits > 1 ? sizeof(float) * (size_t)g.splits * rows * cols : 0;
    return g;
}

template <typename T, int OP>
hipError_t run_gemm(const Operand& a, const Operand& b, long long rows, long long cols, long long depth, TileArgs t, void* part,
                    hipStream_t stream) {
    typedef typename Plane<T>::type P;
    const int pairs = sizeof(T) == 4 ? kPairs : 1;
    const GemmPlan g = plan_gemm(rows, cols, depth, pairs);
    t.part = static_cast<float*>(part);
    t.rows = rows, t.cols = cols, t.splits = g.splits;
    const GemmArgs p = {a, b, rows, cols, depth, pairs, g.splits, g.split_len, g.tiles_i, g.tiles_j, t};
    const dim3 grid(g.tiles_i * g.tiles_j, g.splits);
    if (g.wide)
        linear_gemm_kernel<P, T, 256, 256, 128, 64, OP><<<grid, 512, 0, stream>>>(p);
    else
        linear_gemm_kernel<P, T, 128, 128, 64, 64, OP><<<grid, 256, 0, stream>>>(p);
    if (g.splits > 1) linear_join_kernel<T, OP><<<dim3(join_blocks(rows * cols)), kThreads, 0, stream>>>(t);
    return hipGetLastError();
}

template <typename T>
hipError_t run_pack(const PackArgs& p, hipStream_t stream) {
    const dim3 grid((unsigned)((p.pc / 64) * ceil_div(p.rows, 64)));
    if (p.act != kActNone)
        linear_pack_kernel<T, true><<<grid, kThreads, 0, stream>>>(p);
    else
        linear_pack_kernel<T, false><<<grid, kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

// A 16-bit matrix that the large products can read where it stands: 16-byte pieces on 16 bytes.
bool reads_in_place(const void* x, long long ld, long long cols, int dtype) {
    return dtype != 0 && cols % 8 == 0 && ld % 8 == 0 && ld <= kMaxLd && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

// Scratch of a forward / backward call through the large products (offsets from the workspace's start).
struct BigWs {
    long long pn, pk;        // n, k padded
    size_t x, w, dz, sums, part, total;
};
BigWs carve_big(long long m, long long n, long long k, int dtype, bool backward) {
    BigWs o = {};
    o.pn = round_up(n, kBK), o.pk = round_up(k, kBK);
    const size_t e = dtype == 0 ? 2 * kPlanes : 2;
    const int pairs = dtype == 0 ? kPairs : 1;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    o.x = take(e * m * o.pk);
    o.w = take(e * n * o.pk);
    if (!backward) {
        o.part = take(plan_gemm(m, n, k, pairs).part_bytes);
    } else {
        o.dz = take(e * m * o.pn);
        o.sums = take(sizeof(float) * ceil_div(m, 64) * n);
        const size_t dx = plan_gemm(m, k, n, pairs).part_bytes, dw = plan_gemm(n, k, m, pairs).part_bytes;
        o.part = take(dx > dw ? dx : dw);
    }
    o.total = at;
    return o;
}

// src [rows, cols] as an operand: where it stands, or packed into `room`.  Along the contraction `depth` of
// its columns are there (zeros from then on, if packed); turned, its rows.
template <typename T>
hipError_t make_operand(Operand& o, const void* src, long long ld, long long rows, long long cols, bool turned, int dtype, void* room,
                        hipStream_t stream) {
    if (reads_in_place(src, ld, cols, dtype)) {
        o = {src, ld, 0, cols, turned ? rows : cols};
        return hipSuccess;
    }
    const long long pc = round_up(cols, kBK);
    o = {room, pc, rows * pc, pc, turned ? rows : pc};
    return run_pack<T>({src, nullptr, ld, rows, cols, pc, kActNone, room, nullptr}, stream);
}

template <typename T>
hipError_t forward_large(const LinearArgs& a, const TileArgs& t, void* ws_, hipStream_t stream) {
    char* ws = static_cast<char*>(ws_);
    const BigWs o = carve_big(a.m, a.n, a.k, a.dtype, false);
    Operand x, w;
    if (hipError_t e = make_operand<T>(x, a.x, a.ldx, a.m, a.k, false, a.dtype, ws + o.x, stream)) return e;
    if (hipError_t e = make_operand<T>(w, a.w, a.ldw, a.n, a.k, false, a.dtype, ws + o.w, stream)) return e;
    return run_gemm<T, kForward>(x, w, a.m, a.n, a.k, t, ws + o.part, stream);
}

template <typename T>
hipError_t backward_large(const LinearArgs& a, const void* z, const void* dy, void* dx, void* dw, void* dbias, void* ws_,
                          hipStream_t stream) {
    char* ws = static_cast<char*>(ws_);
    const BigWs o = carve_big(a.m, a.n, a.k, a.dtype, true);
    const bool as_it_is = a.act == kActNone && reads_in_place(dy, a.n, a.n, a.dtype);
    const bool pack = (dx || dw) && !as_it_is;
    float* sums = dbias ? reinterpret_cast<float*>(ws + o.sums) : nullptr;
    if (pack || dbias)
        if (hipError_t e = run_pack<T>({dy, z, a.n, a.m, a.n, o.pn, a.act, pack ? ws + o.dz : nullptr, sums}, stream)) return e;
    Operand dz = {dy, a.n, 0, a.n, a.n};
    if (pack) dz = {ws + o.dz, o.pn, a.m * o.pn, o.pn, o.pn};
    TileArgs t = {};
    if (dx) {
        Operand w;
        if (hipError_t e = make_operand<T>(w, a.w, a.ldw, a.n, a.k, true, a.dtype, ws + o.w, stream)) return e;
        t.out = dx;
        if (hipError_t e = run_gemm<T, kDx>(dz, w, a.m, a.k, a.n, t, ws + o.part, stream)) return e;
    }
    if (dw) {
        Operand x;
        if (hipError_t e = make_operand<T>(x, a.x, a.ldx, a.m, a.k, true, a.dtype, ws + o.x, stream)) return e;
        t.out = dw;
        dz.valid = a.m;
        if (hipError_t e = run_gemm<T, kDw>(dz, x, a.n, a.k, a.m, t, ws + o.part, stream)) return e;
    }
    if (dbias)
        linear_bias_kernel<T><<<dim3((unsigned)ceil_div(a.n, 64)), kThreads, 0, stream>>>(sums, ceil_div(a.m, 64), a.n,
                                                                                          static_cast<T*>(dbias));
    return hipGetLastError();
}

// The small tiles' backward pass: the same cuts, groups of waves and scratch, dx's in front of dw's, whichever of its outputs
// are wanted, so that a gradient is the same number beside others and alone.
struct BackwardPlan {
    int tn;
    bool few_rows;           // of dx
    bool share;
    TilePlan dx, dw;
    size_t dx_bytes, total;
};
BackwardPlan plan_backward(long long m, long long n, long long k, int dtype, int act) {
    BackwardPlan o;
    const int esize = dtype == 0 ? 4 : 2;
    o.tn = tile_width(k, m * n);      // (A is dz in both products)
    o.few_rows = has_few_rows_dx(m, n, k, dtype == 0);
    const TileShape of[2] = {{o.few_rows ? 0 : m, k, n}, {n, k, m}};
    TilePlan plan[2];
    plan_tiles(of, o.tn, esize, act, true, plan);
    o.dx = plan[0], o.dw = plan[1];
    long long pieces = 0, longest = 0;
    for (int i = 0; i < 2; ++i) {
        if (of[i].rows == 0) continue;
        pieces += ceil_div(of[i].rows, kTileSize / o.tn) * ceil_div(of[i].cols, o.tn) * plan[i].splits;
        if (plan[i].len > longest) longest = plan[i].len;
    }
    o.share = share_pieces(pieces, longest);
    o.dx_bytes = ((o.few_rows ? few_dx_bytes(m, n, k, esize) : part_bytes(of[0], o.dx)) + 255) & ~(size_t)255;
    o.total = o.dx_bytes + part_bytes(of[1], o.dw);      // (dbias alone: one column in place of k)
    return o;
}

template <typename T, int TN>
void run_tiles(TileArgs& p, void* ws, hipStream_t stream) {
    TilePlan plan[1];
    plan_tiles({{p.rows, p.cols, p.depth}}, TN, sizeof(T), p.act, false, plan);
    const unsigned pieces = set_tiles(p, TN, plan[0], ws);
    if (share_pieces(pieces, p.split_len))
        linear_tile_forward_kernel<T, kGroups, TN><<<dim3(pieces), kThreads * kGroups, 0, stream>>>(p);
    else
        linear_tile_forward_kernel<T, 1, TN><<<dim3(pieces), kThreads, 0, stream>>>(p);
}
template <typename T, int TN>
void run_tiles_backward(const TileArgs& dx, unsigned pieces_dx, const TileArgs& dw, unsigned pieces_dw, bool share, hipStream_t stream) {
    const unsigned pieces = pieces_dx + pieces_dw;
    if (share)
        linear_tile_backward_kernel<T, kGroups, TN><<<dim3(pieces), kThreads * kGroups, 0, stream>>>(dx, pieces_dx, dw);
    else
        linear_tile_backward_kernel<T, 1, TN><<<dim3(pieces), kThreads, 0, stream>>>(dx, pieces_dx, dw);
}

template <typename T>
hipError_t forward_t(const LinearArgs& a, void* y, void* z, void* ws, hipStream_t stream) {
    TileArgs p = {};
    p.a = a.x, p.b = a.w, p.lda = a.ldx, p.ldb = a.ldw;
    p.bias = a.bias, p.residual = a.residual, p.ldr = a.ldr;
    p.rows = a.m, p.cols = a.n, p.depth = a.k, p.n = a.n, p.act = a.act;
    p.out = y, p.keep = z;
    if (has_few_rows(a.m, a.n, a.k, sizeof(T) == 4)) return run_few_rows<T>(p, stream);
    if (is_large(a.m, a.n, a.k, a.dtype)) return forward_large<T>(a, p, ws, stream);
    if (tile_width(a.n, a.m * a.k) == 32)
        run_tiles<T, 32>(p, ws, stream);
    else
        run_tiles<T, 64>(p, ws, stream);
    if (p.splits > 1) linear_join_kernel<T, kForward><<<dim3(join_blocks(p.rows * p.cols)), kThreads, 0, stream>>>(p);
    return hipGetLastError();
}

template <typename T>
hipError_t backward_t(const LinearArgs& a, const void* z, const void* dy, void* dx, void* dw, void* dbias, void* ws_,
                      hipStream_t stream) {
    if (is_large(a.m, a.n, a.k, a.dtype)) return backward_large<T>(a, z, dy, dx, dw, dbias, ws_, stream);
    char* ws = static_cast<char*>(ws_);
    TileArgs p = {};
    p.z = z, p.dy = dy, p.n = a.n, p.act = a.act, p.splits = 1;
    TileArgs q = p;
    unsigned pieces_dx = 0, pieces_dw = 0;
    const BackwardPlan plan = plan_backward(a.m, a.n, a.k, a.dtype, a.act);
    if (dx) {
        p.b = a.w, p.ldb = a.ldw, p.rows = a.m, p.cols = a.k, p.depth = a.n, p.out = dx;
        if (plan.few_rows) {
            if (hipError_t e = run_few_rows_dx<T>(p, ws, stream)) return e;
        } else {
            pieces_dx = set_tiles(p, plan.tn, plan.dx, ws);
        }
    }
    if (dw || dbias) {
        // (for dbias alone there is no product: one column of tiles, and x, which may be NULL, is not read)
        q.b = dw ? a.x : nullptr, q.ldb = a.ldx, q.rows = a.n, q.cols = dw ? a.k : 1, q.depth = a.m, q.out = dw, q.dbias = dbias;
        pieces_dw = set_tiles(q, plan.tn, plan.dw, ws + plan.dx_bytes);
    }
    if (pieces_dx + pieces_dw == 0) return hipGetLastError();
    if (plan.tn == 32)
        run_tiles_backward<T, 32>(p, pieces_dx, q, pieces_dw, plan.share, stream);
    else
        run_tiles_backward<T, 64>(p, pieces_dx, q, pieces_dw, plan.share, stream);
    if (pieces_dx == 0) p.splits = 1;      // (its own launches have joined it)
    if (p.splits > 1 || q.splits > 1) {
        const long long ex = p.splits > 1 ? p.rows * p.cols : 0, ew = q.splits > 1 ? q.rows * q.cols : 0;
        linear_join_backward_kernel<T><<<dim3(join_blocks(ex > ew ? ex : ew)), kThreads, 0, stream>>>(p, q);
    }
    return hipGetLastError();
}

}  // namespace

size_t linear_workspace_bytes(long long m, long long n, long long k, int dtype, int act, int backward) {
    if (is_large(m, n, k, dtype)) return carve_big(m, n, k, dtype, backward).total;
    if (backward) return plan_backward(m, n, k, dtype, act).total;
    if (has_few_rows(m, n, k, dtype == 0)) return 0;
    TilePlan plan[1];
    const TileShape of[1] = {{m, n, k}};
    plan_tiles(of, tile_width(n, m * k), dtype == 0 ? 4 : 2, act, false, plan);
    return part_bytes(of[0], plan[0]);
}

hipError_t launch_linear_forward(const LinearArgs& a, void* y, void* z, void* ws, hipStream_t stream) {
    switch (a.dtype) {
        case 0: return forward_t<float>(a, y, z, ws, stream);
        case 1: return forward_t<f16>(a, y, z, ws, stream);
        default: return forward_t<bf16>(a, y, z, ws, stream);
    }
}

hipError_t launch_linear_backward(const LinearArgs& a, const void* z, const void* dy, void* dx, void* dw, void* dbias,
                                  void* ws, hipStream_t stream) {
    switch (a.dtype) {
        case 0: return backward_t<float>(a, z, dy, dx, dw, dbias, ws, stream);
        case 1: return backward_t<f16>(a, z, dy, dx, dw, dbias, ws, stream);
        default: return backward_t<bf16>(a, z, dy, dx, dw, dbias, ws, stream);
    }
}

}  // namespace scmiac
