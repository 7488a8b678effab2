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

constexpr float kSqrtHalf = 0.70710678118654752440f;
constexpr float kInvSqrt2Pi = 0.39894228040143267794f;

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + fast_exp2(-kLog2e * z)); }

__device__ __forceinline__ float act_value(int act, float z) {
    switch (act) {
        case kActRelu: return z < 0.f ? 0.f : z;   // (a NaN stays one)
        case kActGelu: return 0.5f * z * (1.f + erff(z * kSqrtHalf));
        case kActSilu: return z * sigmoid(z);
        default: return z;
    }
}
__device__ __forceinline__ float act_slope(int act, float z) {
    switch (act) {
        case kActRelu: return z > 0.f ? 1.f : 0.f;
        case kActGelu: return 0.5f * (1.f + erff(z * kSqrtHalf)) + z * kInvSqrt2Pi * fast_exp2(-0.5f * kLog2e * z * z);
        case kActSilu: {
            const float s = sigmoid(z);
            return s * (1.f + z * (1.f - s));
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

// One value of the forward product through the epilogue.
template <typename T>
__device__ __forceinline__ void forward_out(float z, long long i, long long j, long long n, int act, const T* __restrict__ bias,
                                            const T* __restrict__ residual, long long ldr, T* __restrict__ y, T* __restrict__ zk) {
    if (bias) z += to_f32(bias[j]);
    if (zk) zk[i * n + j] = keep_z<T>(z);
    float v = act_value(act, z);
    if (residual) v += to_f32(residual[i * ldr + j]);
    y[i * n + j] = from_f32<T>(v);
}

// ------------------------------------------------------------------ 64 x 64 tiles, any shape

constexpr int kTile = 64, kDepth = 32, kThreads = 256;

template <typename T>
struct Lds {
    static constexpr int LD = sizeof(T) == 4 ? kDepth + 4 : kDepth + 8;   // rows start on 16 bytes, four banks apart
};

struct TileArgs {
    const void *a, *b;             // forward: x, w;  dx: -, w;  dw: -, x
    const void *z, *dy;
    const void *bias, *residual;
    long long lda, ldb, ldr;
    long long rows, cols, depth;   // of C and of the contraction
    long long n;                   // row length of z, dy, y
    int act, splits;
    unsigned tiles_i;              // 64-row tiles of C
    long long split_len;
    void *out, *keep, *dbias;
    float *part, *part_bias;       // [splits][rows][cols], [splits][rows]
};

template <typename T, int OP>
__global__ __launch_bounds__(kThreads) void linear_tile_kernel(TileArgs p) {
    constexpr int LD = Lds<T>::LD;
    constexpr int NV = kTile * kDepth / kThreads;   // elements of a tile per thread
    __shared__ __align__(16) T as[kTile * LD];
    __shared__ __align__(16) T bs[kTile * LD];
    __shared__ float bias_sum[kThreads];
    const int t = threadIdx.x, lane = t & 63, wave = wave_id();
    const unsigned tile_j = blockIdx.x / p.tiles_i;
    const long long i0 = (long long)(blockIdx.x - tile_j * p.tiles_i) * kTile, j0 = (long long)tile_j * kTile;
    const long long c_lo = (long long)blockIdx.y * p.split_len;
    const long long c_hi = min(p.depth, c_lo + p.split_len);
    const T* __restrict__ a = static_cast<const T*>(p.a);
    const T* __restrict__ b = static_cast<const T*>(p.b);
    const T* __restrict__ z = static_cast<const T*>(p.z);
    const T* __restrict__ dy = static_cast<const T*>(p.dy);

    // this thread's elements: along the contraction (32 threads a row) or across it (64 threads a column)
    constexpr bool kAlongA = OP != kDw, kAlongB = OP == kForward;
    const int ca = kAlongA ? (t & 31) : (t >> 6), ra = kAlongA ? (t >> 5) : (t & 63);
    const int cb = kAlongB ? (t & 31) : (t >> 6), rb = kAlongB ? (t >> 5) : (t & 63);
    constexpr int kStepRA = kAlongA ? 8 : 0, kStepCA = kAlongA ? 0 : 4;
    constexpr int kStepRB = kAlongB ? 8 : 0, kStepCB = kAlongB ? 0 : 4;

    T va[NV], vb[NV];
    float dsum = 0.f;
    auto load = [&](long long c0) {
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const long long r = i0 + ra + q * kStepRA, c = c0 + ca + q * kStepCA;
            T v = T(0);
            if (r < p.rows && c < c_hi) {
                if (OP == kForward) {
                    v = a[r * p.lda + c];
                } else {
                    const long long at = OP == kDx ? r * p.n + c : c * p.n + r;
                    float g = to_f32(dy[at]);
                    if (p.act != kActNone) g *= act_slope(p.act, to_f32(z[at]));
                    if (OP == kDw) dsum += g;
                    v = from_f32<T>(g);
                }
            }
            va[q] = v;
        }
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            const long long r = j0 + rb + q * kStepRB, c = c0 + cb + q * kStepCB;
            T v = T(0);
            if (r < p.cols && c < c_hi) v = kAlongB ? b[r * p.ldb + c] : b[c * p.ldb + r];
            vb[q] = v;
        }
    };

    f32x16 acc = {};
    const int wr = (wave & 1) * 32 + (lane & 31), wc = (wave >> 1) * 32 + (lane & 31), half = lane >> 5;
    load(c_lo);
    for (long long c0 = c_lo; c0 < c_hi; c0 += kDepth) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NV; ++q) {
            as[(ra + q * kStepRA) * LD + ca + q * kStepCA] = va[q];
            bs[(rb + q * kStepRB) * LD + cb + q * kStepCB] = vb[q];
        }
        __syncthreads();
        if (c0 + kDepth < c_hi) load(c0 + kDepth);
        if constexpr (sizeof(T) == 4) {
            // the two halves of the wave take four neighbouring steps of the contraction each: any order of them
            // gives the same sum of products, and this one reads 16 bytes a lane
#pragma unroll
            for (int s = 0; s < kDepth / 8; ++s) {
                const f32x4 fa = *reinterpret_cast<const f32x4*>(&as[wr * LD + s * 8 + half * 4]);
                const f32x4 fb = *reinterpret_cast<const f32x4*>(&bs[wc * LD + s * 8 + half * 4]);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[q], fb[q], acc, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < kDepth / 16; ++s) {
                if constexpr (__is_same(T, bf16)) {
                    const bf16x8 fa = *reinterpret_cast<const bf16x8*>(&as[wr * LD + s * 16 + half * 8]);
                    const bf16x8 fb = *reinterpret_cast<const bf16x8*>(&bs[wc * LD + s * 16 + half * 8]);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb, acc, 0, 0, 0);
                } else {
                    const f16x8 fa = *reinterpret_cast<const f16x8*>(&as[wr * LD + s * 16 + half * 8]);
                    const f16x8 fb = *reinterpret_cast<const f16x8*>(&bs[wc * LD + s * 16 + half * 8]);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa, fb, acc, 0, 0, 0);
                }
            }
        }
    }

    const long long j = j0 + wc;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const long long i = i0 + (wave & 1) * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
        if (i >= p.rows || j >= p.cols) continue;
        if (p.splits > 1)
            p.part[((long long)blockIdx.y * p.rows + i) * p.cols + j] = acc[r];
        else if (OP == kForward)
            forward_out<T>(acc[r], i, j, p.n, p.act, static_cast<const T*>(p.bias), static_cast<const T*>(p.residual), p.ldr,
                           static_cast<T*>(p.out), static_cast<T*>(p.keep));
        else if (p.out)
            static_cast<T*>(p.out)[i * p.cols + j] = from_f32<T>(acc[r]);
    }
    if (OP == kDw && p.dbias && tile_j == 0) {   // rows of C are the outputs: their sums of dz, four partial sums each
        bias_sum[t] = dsum;
        __syncthreads();
        if (t < kTile && i0 + t < p.rows) {
            const float s = (bias_sum[t] + bias_sum[t + 64]) + (bias_sum[t + 128] + bias_sum[t + 192]);
            if (p.splits > 1)
                p.part_bias[(long long)blockIdx.y * p.rows + i0 + t] = s;
            else
                static_cast<T*>(p.dbias)[i0 + t] = from_f32<T>(s);
        }
    }
}

// Joins the splits of the contraction, in their order.
template <typename T, int OP>
__global__ __launch_bounds__(kThreads) void linear_join_kernel(TileArgs p) {
    const long long total = p.rows * p.cols;
    for (long long e = (long long)blockIdx.x * kThreads + threadIdx.x; e < total; e += (long long)gridDim.x * kThreads) {
        float s = 0.f;
        for (int q = 0; q < p.splits; ++q) s += p.part[q * total + e];
        if (OP == kForward)
            forward_out<T>(s, e / p.cols, e % p.cols, p.n, p.act, static_cast<const T*>(p.bias),
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

// Pieces of the contraction: enough blocks to give every compute unit two, none of them shorter than 256.
void plan_tiles(long long rows, long long cols, long long depth, int& splits, long long& len) {
    splits = 1, len = depth;
    const long long tiles = ceil_div(rows, kTile) * ceil_div(cols, kTile);
    if (tiles == 0 || depth == 0) return;
    long long s = 512 / tiles;
    if (s > depth / 256) s = depth / 256;
    if (s < 1) s = 1;
    len = round_up(ceil_div(depth, s), kDepth);
    splits = (int)ceil_div(depth, len);
}
size_t tile_bytes(long long rows, long long cols, long long depth) {
    int splits;
    long long len;
    plan_tiles(rows, cols, depth, splits, len);
    return splits > 1 ? sizeof(float) * (size_t)splits * ((size_t)rows * cols + rows) : 0;
}

template <typename T, int OP>
hipError_t run_tiles(TileArgs p, void* ws, hipStream_t stream) {
    plan_tiles(p.rows, p.cols, p.depth, p.splits, p.split_len);
    p.part = static_cast<float*>(ws);
    p.part_bias = p.part + (size_t)p.splits * p.rows * p.cols;
    p.tiles_i = (unsigned)ceil_div(p.rows, kTile);
    const dim3 grid((unsigned)(p.tiles_i * ceil_div(p.cols, kTile)), p.splits);
    linear_tile_kernel<T, OP><<<grid, kThreads, 0, stream>>>(p);
    if (p.splits > 1) {
        const long long blocks = ceil_div(p.rows * p.cols, kThreads);
        linear_join_kernel<T, OP><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)), kThreads, 0, stream>>>(p);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t forward_t(const LinearArgs& a, void* y, void* z, void* ws, hipStream_t stream) {
    TileArgs p = {};
    p.a = a.x, p.b = a.w, p.lda = a.ldx, p.ldb = a.ldw;
    p.bias = a.bias, p.residual = a.residual, p.ldr = a.ldr;
    p.rows = a.m, p.cols = a.n, p.depth = a.k, p.n = a.n, p.act = a.act;
    p.out = y, p.keep = z;
    return run_tiles<T, kForward>(p, ws, stream);
}

template <typename T>
hipError_t backward_t(const LinearArgs& a, const void* z, const void* dy, void* dx, void* dw, void* dbias, void* ws,
                      hipStream_t stream) {
    TileArgs p = {};
    p.z = z, p.dy = dy, p.n = a.n, p.act = a.act;
    if (dx) {
        p.b = a.w, p.ldb = a.ldw, p.rows = a.m, p.cols = a.k, p.depth = a.n, p.out = dx;
        if (hipError_t e = run_tiles<T, kDx>(p, ws, stream)) return e;
    }
    if (dw || dbias) {
        p.b = a.x, p.ldb = a.ldx, p.rows = a.n, p.cols = a.k, p.depth = a.m, p.out = dw, p.dbias = dbias;
        if (hipError_t e = run_tiles<T, kDw>(p, ws, stream)) return e;
    }
    return hipSuccess;
}

}  // namespace

size_t linear_workspace_bytes(long long m, long long n, long long k, int dtype, int act, int backward) {
    (void)dtype, (void)act;
    if (!backward) return tile_bytes(m, n, k);
    const size_t a = tile_bytes(m, k, n), b = tile_bytes(n, k, m);
    return a > b ? a : b;
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
