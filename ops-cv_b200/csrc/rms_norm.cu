// Root-mean-square norm of a residual sum, with its gradient and with 8-bit outputs.
//
// z = T(x + residual) is rounded to the storage type first and everything else is a function of that stored value, so that the
// backward, which reads z and not its two terms, is the gradient of exactly what the forward computed. Squares, their mean, the
// dot product of the backward and the sums of the weight's gradient are fp32.
//
// Bound by HBM: the forward moves two rows in and two out, the backward three in and one out. A row stays in registers between
// the reduction and the output (each thread owns the same columns in every pass over the row), so each value moves once.
// 8192 x 4096 bf16: forward 46 us (5.85 TB/s), backward 48 us and 5 more for the weight's sums (5.0 TB/s over both); to e4m3 in groups of
// 128, 8192 x 5120: 64 us (4.6 TB/s), no unit full (issue slots 59 % busy). 16 rows of 4096: 2.6 us.
#include <cuda_fp8.h>

#include "cp_async.cuh"
#include "launch_util.cuh"
#include "sequence_kernels.h"

namespace opscv {

namespace {

constexpr int kMaxThreads = 1024;

__device__ __forceinline__ int64_t RowAt(int64_t row, int64_t inner, RowStride s)
{
    return row < inner ? row * s.s1 : row / inner * s.s0 + row % inner * s.s1;
}

// V values of T as fp32; loads of up to 16 bytes.
template <typename T, int V>
__device__ __forceinline__ void LoadF(const T* p, float (&v)[V])
{
    if constexpr (V == 1) {
        v[0] = DType<T>::ToF(*p);
    } else {
        LoadPack<T, V>(p, v);
    }
}
template <typename T, int V>
__device__ __forceinline__ void StoreF(T* p, const float (&v)[V])
{
    if constexpr (V == 1) {
        *p = DType<T>::FromF(v[0]);
    } else {
        StorePack<T, V>(p, v);
    }
}
template <typename T, int V>
__device__ __forceinline__ void LoadWeight(const void* w, bool w32, int32_t col, float (&v)[V])
{
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = 1.0f;
        }
    } else if (w32) {
        const float* p = static_cast<const float*>(w) + col;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = __ldg(p + i);
        }
    } else {
        LoadF<T, V>(static_cast<const T*>(w) + col, v);
    }
}

// The sum of v over the blockDim.x threads of a row, for all of them. Rows of one warp need no shared memory. The order of the
// additions is fixed, so equal inputs give equal bits.
__device__ __forceinline__ float RowSum(float v, float* part)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    if (blockDim.x == 32) {
        return v;
    }
    // one row a block: rows of several warps have blockDim.y == 1
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    v = static_cast<int>(threadIdx.x & 31) < warps ? part[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

__device__ __forceinline__ float WarpSum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

struct FwdArgs {
    const void *x, *residual, *weight;
    void *y, *sum;
    float* rstd;
    RowStride xs, rs, ys, ss;
    int64_t rows, inner;
    int32_t width;
    float eps;
    bool weight32;
    // 8-bit outputs
    float* scales;
    int32_t group, groups;
};

// Rows are held as they are stored (two 16-bit values a register) and taken apart where they are used: the registers of a row halve, and
// the sum of two 16-bit values costs one instruction a pair. Its rounding is that of the fp32 sum: two values whose exponents are near
// enough for a tie have an exact fp32 sum.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> AddPacks(const Pack<T, V>& a, const Pack<T, V>& b)
{
    Pack<T, V> s;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        using T2 = std::conditional_t<DType<T>::kIsHalf, __half2, __nv_bfloat162>;
        const T2 *x = reinterpret_cast<const T2*>(&a), *y = reinterpret_cast<const T2*>(&b);
        T2* z = reinterpret_cast<T2*>(&s);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            z[i] = __hadd2_rn(x[i], y[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s.v[i] = DType<T>::FromF(DType<T>::ToF(a.v[i]) + DType<T>::ToF(b.v[i]));
        }
    }
    return s;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> LoadSum(const T* x, const T* r, int32_t col)
{
    const Pack<T, V> z = *reinterpret_cast<const Pack<T, V>*>(x + col);
    return r != nullptr ? AddPacks(z, *reinterpret_cast<const Pack<T, V>*>(r + col)) : z;
}
template <typename T, int V>
__device__ __forceinline__ void StorePacked(T* p, const Pack<T, V>& z)
{
    *reinterpret_cast<Pack<T, V>*>(p) = z;
}
// v[i] = a[i] * b[i], two at a time
template <int V>
__device__ __forceinline__ void Times(float (&v)[V], const float (&b)[V])
{
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            SplitF2(Mul2(MakeF2(v[i], v[i + 1]), MakeF2(b[i], b[i + 1])), v[i], v[i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] *= b[i];
        }
    }
}
template <int V>
__device__ __forceinline__ void Times(float (&v)[V], float f)
{
    float b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        b[i] = f;
    }
    Times(v, b);
}
// sum of a[i] * b[i], even and odd ones apart until the end
template <int V>
__device__ __forceinline__ void AddDot(const float (&a)[V], const float (&b)[V], F2& s)
{
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            s = Fma2(MakeF2(a[i], a[i + 1]), MakeF2(b[i], b[i + 1]), s);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s = Fma2(MakeF2(a[i], 0.0f), MakeF2(b[i], 0.0f), s);
        }
    }
}
// s[i] += a[i] * b[i]
template <int V>
__device__ __forceinline__ void AddProducts(const float (&a)[V], const float (&b)[V], float (&s)[V])
{
    if constexpr (V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            SplitF2(Fma2(MakeF2(a[i], a[i + 1]), MakeF2(b[i], b[i + 1]), MakeF2(s[i], s[i + 1])), s[i], s[i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s[i] = fmaf(a[i], b[i], s[i]);
        }
    }
}
__device__ __forceinline__ float Both(F2 s)
{
    float a, b;
    SplitF2(s, a, b);
    return a + b;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> ZeroPack()
{
    Pack<T, V> z;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        z.v[i] = DType<T>::FromF(0.0f);
    }
    return z;
}

// The weight of a row's chunks. One of the tensors' type is read before the reduction's wait, whose time covers the load's; an fp32
// one takes twice the registers and is read after it.
template <typename T, int V, int N>
struct WeightOf {
    Pack<T, V> held[N];
    __device__ __forceinline__ void Early(const FwdArgs& a, int k, int32_t col)
    {
        if (a.weight != nullptr && !a.weight32) {
            held[k] = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.weight) + col);
        }
    }
    // v[i] *= rstd * weight[i]
    __device__ __forceinline__ void Apply(const FwdArgs& a, int k, int32_t col, float rstd, float (&v)[V]) const
    {
        Times(v, rstd);
        if (a.weight != nullptr) {
            float w[V];
            if (a.weight32) {
                LoadWeight<T, V>(a.weight, true, col, w);
            } else {
                UnpackToF<T, V>(held[k], w);
            }
            Times(v, w);
        }
    }
};

// NV > 0: the row is held in NV * V values a thread. NV == 0: rows too wide for that are read again for the second pass (from L2
// mostly), from `sum` where there is one, since it may lie over one of the terms.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(kMaxThreads) RmsNormFwdKernel(FwdArgs a)
{
    __shared__ float part[32];
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= a.rows) { // rows of several warps have one row a block, so that no barrier is left out
        return;
    }
    const T* x = static_cast<const T*>(a.x) + RowAt(row, a.inner, a.xs);
    const T* r = a.residual != nullptr ? static_cast<const T*>(a.residual) + RowAt(row, a.inner, a.rs) : nullptr;
    T* y = static_cast<T*>(a.y) + RowAt(row, a.inner, a.ys);
    T* sum = a.sum != nullptr ? static_cast<T*>(a.sum) + RowAt(row, a.inner, a.ss) : nullptr;
    const int32_t step = blockDim.x * V;
    const int32_t first = threadIdx.x * V;
    constexpr int N = NV > 0 ? NV : 1;
    Pack<T, V> z[N];
    WeightOf<T, V, N> w;
    F2 sq = MakeF2(0.0f, 0.0f);
    float f[V];
    if constexpr (NV > 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            z[k] = ZeroPack<T, V>();
            if (col < a.width) {
                z[k] = LoadSum<T, V>(x, r, col);
                w.Early(a, k, col);
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            if (sum != nullptr && col < a.width) {
                StorePacked<T, V>(sum + col, z[k]);
            }
            UnpackToF<T, V>(z[k], f);
            AddDot(f, f, sq);
        }
    } else {
        for (int32_t col = first; col < a.width; col += step) {
            z[0] = LoadSum<T, V>(x, r, col);
            if (sum != nullptr) {
                StorePacked<T, V>(sum + col, z[0]);
            }
            UnpackToF<T, V>(z[0], f);
            AddDot(f, f, sq);
        }
    }
    const float mean = RowSum(Both(sq), part) / static_cast<float>(a.width);
    const float rstd = 1.0f / sqrtf(mean + a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) {
        a.rstd[row] = rstd;
    }
    if constexpr (NV > 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            if (col < a.width) {
                UnpackToF<T, V>(z[k], f);
                w.Apply(a, k, col, rstd, f);
                StoreF<T, V>(y + col, f);
            }
        }
    } else {
        for (int32_t col = first; col < a.width; col += step) {
            z[0] = sum != nullptr ? *reinterpret_cast<const Pack<T, V>*>(sum + col) : LoadSum<T, V>(x, r, col);
            w.Early(a, 0, col);
            UnpackToF<T, V>(z[0], f);
            w.Apply(a, 0, col, rstd, f);
            StoreF<T, V>(y + col, f);
        }
    }
}

// ---- 8-bit outputs ---------------------------------------------------------------------------------------------------------
// A NaN is above all other magnitudes, so a row or group with one gets a NaN as its scale. As unsigned integers, non-negative floats
// (and NaNs) order alike, which is what the maximum in shared memory uses.
__device__ __forceinline__ float MaxOrNaN(float a, float b)
{
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
template <int V>
__device__ __forceinline__ float Most(const float (&v)[V], float m)
{
#pragma unroll
    for (int i = 0; i < V; ++i) {
        m = MaxOrNaN(m, fabsf(v[i]));
    }
    return m;
}

template <Q8 Q>
struct Q8Type;
template <>
struct Q8Type<Q8::E4M3> {
    static constexpr float kMost = 448.0f;
    template <int V>
    static __device__ __forceinline__ void Store(uint8_t* p, const float (&v)[V])
    {
        if constexpr (V == 1) {
            *p = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
        } else {
            Pack<uint16_t, V / 2> b;
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                b.v[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
            }
            *reinterpret_cast<Pack<uint16_t, V / 2>*>(p) = b;
        }
    }
};
template <>
struct Q8Type<Q8::INT8> {
    static constexpr float kMost = 127.0f;
    template <int V>
    static __device__ __forceinline__ void Store(uint8_t* p, const float (&v)[V])
    {
        Pack<uint8_t, V> b;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            b.v[i] = static_cast<uint8_t>(__float2int_rn(v[i])); // no quotient rounds to more than 127, the largest magnitude's own
        }
        *reinterpret_cast<Pack<uint8_t, V>*>(p) = b;
    }
};

// A group of zeros, or of magnitudes below kLeast, has scale 0 and zeros.
constexpr float kLeast = 1e-35f;
__device__ __forceinline__ float ScaleOf(float most, float range) { return most < kLeast ? 0.0f : most / range; }
// v[i] / scale, two at a time: the product with the inverse, within 1.5 steps of the quotient, and what its remainder adds to it. The
// remainder fma(-q, scale, v) loses no more than its last bit, so the result is the rounded quotient unless that lies within 2^-22 of a
// step of the middle between two floats (the correction of a quotient by its remainder: Markstein, IBM J. Res. Dev. 34, 1990). Without
// the correction a value next to the middle of two 8-bit ones goes to the wrong one now and then; the operator / takes 84 us where this
// takes 63.8 and the product alone 63.5 (8192 x 5120 bf16, groups of 128).
struct Divisor {
    float scale, inverse;
    __device__ __forceinline__ explicit Divisor(float s) : scale(s), inverse(s == 0.0f ? 0.0f : 1.0f / s) {}
    template <int V>
    __device__ __forceinline__ void Divide(float (&v)[V]) const
    {
        if constexpr (V % 2 == 0) {
            const F2 by = MakeF2(inverse, inverse), minus = MakeF2(-scale, -scale);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const F2 x = MakeF2(v[i], v[i + 1]), q = Mul2(x, by);
                SplitF2(Fma2(Fma2(q, minus, x), by, q), v[i], v[i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float q = v[i] * inverse;
                v[i] = fmaf(fmaf(q, -scale, v[i]), inverse, q);
            }
        }
    }
};

// Where the largest magnitudes of a row's groups come together. LG > 0: within warps, LG lanes to a group (groups of a power of two of
// columns); kShared: in one word of shared memory each; kRowScale: in the row's block, one scale for all. (With the lanes as an argument
// of the kernel, groups of 128 of 8192 x 5120 take 65.6 us, not 63.8.)
constexpr int kShared = 0, kRowScale = -1;

// 48 registers where 16 values a thread allow it: blocks of 320 threads come four to an SM, not three (8192 x 5120 to int8 in groups of
// 128, bf16: 69.6 us against 80.5; fp32 to either type 123 against 139).
template <typename T, int V, int NV, Q8 Q, int LG>
__global__ void __launch_bounds__(kMaxThreads) __maxnreg__(NV * V == 16 && LG != kShared ? 48 : 64) RmsNormQuantKernel(FwdArgs a)
{
    extern __shared__ uint32_t most[]; // [groups] (kShared)
    __shared__ float part[32];
    using QT = Q8Type<Q>;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= a.rows) {
        return;
    }
    const T* x = static_cast<const T*>(a.x) + RowAt(row, a.inner, a.xs);
    const T* r = a.residual != nullptr ? static_cast<const T*>(a.residual) + RowAt(row, a.inner, a.rs) : nullptr;
    uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.width;
    T* sum = a.sum != nullptr ? static_cast<T*>(a.sum) + RowAt(row, a.inner, a.ss) : nullptr;
    float* scales = a.scales + row * a.groups;
    const int32_t step = blockDim.x * V;
    const int32_t first = threadIdx.x * V;
    constexpr int N = NV > 0 ? NV : 1;
    Pack<T, V> z[N];
    WeightOf<T, V, N> w;
    F2 sq = MakeF2(0.0f, 0.0f);
    float f[V];
    if constexpr (LG == kShared) { // one row a block (the launcher sees to it)
        for (int32_t g = threadIdx.x; g < a.groups; g += blockDim.x) {
            most[g] = 0;
        }
        __syncthreads();
    }
    if constexpr (NV > 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            z[k] = ZeroPack<T, V>();
            w.held[k] = ZeroPack<T, V>();
            if (col < a.width) {
                z[k] = LoadSum<T, V>(x, r, col);
                w.Early(a, k, col);
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            if (sum != nullptr && col < a.width) {
                StorePacked<T, V>(sum + col, z[k]);
            }
            UnpackToF<T, V>(z[k], f);
            AddDot(f, f, sq);
        }
    } else {
        for (int32_t col = first; col < a.width; col += step) {
            z[0] = LoadSum<T, V>(x, r, col);
            if (sum != nullptr) {
                StorePacked<T, V>(sum + col, z[0]);
            }
            UnpackToF<T, V>(z[0], f);
            AddDot(f, f, sq);
        }
    }
    const float rstd = 1.0f / sqrtf(RowSum(Both(sq), part) / static_cast<float>(a.width) + a.eps);
    if constexpr (NV > 0 && LG == kRowScale) {
        __shared__ float tops[32];
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            UnpackToF<T, V>(z[k], f);
            w.Apply(a, k, col < a.width ? col : 0, rstd, f);
            top = col < a.width ? Most(f, top) : top; // behind the row: 0 times a weight that may be infinite
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top = MaxOrNaN(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (blockDim.x > 32) {
            if ((threadIdx.x & 31) == 0) {
                tops[threadIdx.x >> 5] = top;
            }
            __syncthreads();
            top = static_cast<int>(threadIdx.x & 31) < static_cast<int>(blockDim.x >> 5) ? tops[threadIdx.x & 31] : 0.0f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                top = MaxOrNaN(top, __shfl_xor_sync(0xffffffffu, top, o));
            }
        }
        const float scale = ScaleOf(top, QT::kMost);
        if (threadIdx.x == 0) {
            scales[0] = scale;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            if (col < a.width) {
                UnpackToF<T, V>(z[k], f);
                w.Apply(a, k, col, rstd, f);
                Divisor(scale).Divide(f);
                QT::template Store<V>(q + col, f);
            }
        }
        return;
    }
    if constexpr (NV > 0 && LG > 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            const bool inside = col < a.width;
            // A lane behind the row forms 0 times a weight that may be infinite, and puts 0 into the exchange: one select, where a branch
            // around the arithmetic would keep the chunks' from overlapping (8192 x 5120: 74 us against 63).
            UnpackToF<T, V>(z[k], f);
            w.Apply(a, k, inside ? col : 0, rstd, f);
            float top = inside ? Most(f, 0.0f) : 0.0f;
#pragma unroll
            for (int o = LG / 2; o > 0; o >>= 1) {
                top = MaxOrNaN(top, __shfl_xor_sync(0xffffffffu, top, o));
            }
            if (inside) {
                const float scale = ScaleOf(top, QT::kMost);
                if ((threadIdx.x & (LG - 1)) == 0) {
                    scales[col / (LG * V)] = scale;
                }
                Divisor(scale).Divide(f);
                QT::template Store<V>(q + col, f);
            }
        }
        return;
    }
    if constexpr (LG == kShared) {
        // two passes over the row's values: largest magnitudes, then the quantised values
        for (int pass = 0; pass < 2; ++pass) {
            float top = 0.0f; // of all of this thread's values
            auto chunk = [&](int k, int32_t col) {
                UnpackToF<T, V>(z[k], f);
                w.Apply(a, k, col, rstd, f);
                const int32_t g = a.groups > 1 ? col / a.group : 0;
                if (pass == 0) {
                    if (a.groups > 1) {
                        atomicMax(&most[g], __float_as_uint(Most(f, 0.0f)));
                    } else {
                        top = Most(f, top);
                    }
                } else {
                    Divisor(ScaleOf(__uint_as_float(most[g]), QT::kMost)).Divide(f);
                    QT::template Store<V>(q + col, f);
                }
            };
            if constexpr (NV > 0) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int32_t col = first + k * step;
                    if (col < a.width) {
                        chunk(k, col);
                    }
                }
            } else {
                for (int32_t col = first; col < a.width; col += step) {
                    z[0] = sum != nullptr ? *reinterpret_cast<const Pack<T, V>*>(sum + col) : LoadSum<T, V>(x, r, col);
                    w.Early(a, 0, col);
                    chunk(0, col);
                }
            }
            if (pass == 0 && a.groups == 1) {
                const uint32_t t = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);
                if ((threadIdx.x & 31) == 0) {
                    atomicMax(&most[0], t);
                }
            }
            __syncthreads();
        }
        for (int32_t g = threadIdx.x; g < a.groups; g += blockDim.x) {
            scales[g] = ScaleOf(__uint_as_float(most[g]), QT::kMost);
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------
struct BwdArgs {
    const void *gradY, *sum, *weight, *gradSum;
    const float* rstd;
    void* gradX;
    float* scratch; // [gridDim.x][width] sums of the weight's gradient, null without a weight
    RowStride gs, ss, as, xs;
    int64_t rows, inner;
    int32_t width;
    bool weight32;
};

// A block walks rows blockIdx.x, + gridDim.x, ...; each thread keeps its columns' weight and the sum of the weight's gradient in
// registers over all of them, so the weight's gradient costs no second pass over gradY and z. The rows' loads of one step are
// issued before the reduction of the step before is waited for.
//
// RING (16-byte chunks): the next rows come by asynchronous copies into slots of shared memory, each thread its own chunks, up to three
// rows ahead; else the next row is loaded into registers, which hold one.
constexpr int Ahead(int nv) { return nv <= 2 ? 3 : 2; } // 4 chunks a thread leave room for two rows
constexpr int RingBytes(int nv, int threads) { return Ahead(nv) * 3 * nv * threads * 16; }
// 16 values a thread are the most whose weight, sums and rows fit its registers, and only with 512 threads a block.
constexpr int kBwdValues = 16;
constexpr int BwdThreads(int nv, int v) { return nv * v == kBwdValues ? 512 : kMaxThreads; }

template <typename T, int V, int NV, bool RING>
__global__ void __launch_bounds__(BwdThreads(NV, V)) RmsNormBwdKernel(BwdArgs a)
{
    constexpr int kAhead = Ahead(NV);
    extern __shared__ uint4 slots[]; // [kAhead][3][NV][threads] (RING)
    __shared__ float part[2][32];
    const int32_t step = blockDim.x * V;
    const int32_t first = threadIdx.x * V;
    const float inverse = 1.0f / static_cast<float>(a.width);
    float w[NV][V], gw[NV][V];
    Pack<T, V> nextG[NV], nextZ[NV], nextA[NV];
    float nextRstd = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int32_t col = first + k * step;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[k][i] = gw[k][i] = 0.0f;
            nextG[k].v[i] = nextZ[k].v[i] = nextA[k].v[i] = DType<T>::FromF(0.0f);
        }
        if (col < a.width) {
            LoadWeight<T, V>(a.weight, a.weight32, col, w[k]);
        }
    }
    auto fetch = [&](int64_t row, int stage) {
        const T* g = static_cast<const T*>(a.gradY) + RowAt(row, a.inner, a.gs);
        const T* z = static_cast<const T*>(a.sum) + RowAt(row, a.inner, a.ss);
        const T* s = a.gradSum != nullptr ? static_cast<const T*>(a.gradSum) + RowAt(row, a.inner, a.as) : nullptr;
        if constexpr (!RING) {
            nextRstd = a.rstd[row];
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            if (col < a.width) {
                if constexpr (RING) {
                    uint4* at = slots + ((stage * 3) * NV + k) * blockDim.x + threadIdx.x;
                    CpAsync16(at, g + col);
                    CpAsync16(at + NV * blockDim.x, z + col);
                    if (s != nullptr) {
                        CpAsync16(at + 2 * NV * blockDim.x, s + col);
                    }
                } else {
                    nextG[k] = *reinterpret_cast<const Pack<T, V>*>(g + col);
                    nextZ[k] = *reinterpret_cast<const Pack<T, V>*>(z + col);
                    if (s != nullptr) {
                        nextA[k] = *reinterpret_cast<const Pack<T, V>*>(s + col);
                    }
                }
            }
        }
    };
    int64_t row = blockIdx.x;
    int stage = 0;
    if constexpr (RING) {
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            if (row + x * static_cast<int64_t>(gridDim.x) < a.rows) {
                fetch(row + x * static_cast<int64_t>(gridDim.x), x);
            }
            CpAsyncCommit();
        }
    } else if (row < a.rows) {
        fetch(row, 0);
    }
    int turn = 0;
    for (; row < a.rows; row += gridDim.x, turn ^= 1) {
        Pack<T, V> gp[NV], zp[NV], ap[NV];
        float rstd;
        if constexpr (RING) {
            rstd = a.rstd[row];
            CpAsyncWait<kAhead - 1>();
        } else {
            rstd = nextRstd;
        }
        F2 dots = MakeF2(0.0f, 0.0f);
        float g[V], u[V];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if constexpr (RING) {
                const uint4* at = slots + ((stage * 3) * NV + k) * blockDim.x + threadIdx.x;
                const uint4 zero = make_uint4(0, 0, 0, 0);
                const bool inside = first + k * step < a.width;
                const uint4 raw[3] = {inside ? at[0] : zero, inside ? at[NV * blockDim.x] : zero,
                                      inside && a.gradSum != nullptr ? at[2 * NV * blockDim.x] : zero};
                gp[k] = reinterpret_cast<const Pack<T, V>&>(raw[0]);
                zp[k] = reinterpret_cast<const Pack<T, V>&>(raw[1]);
                ap[k] = reinterpret_cast<const Pack<T, V>&>(raw[2]);
            } else {
                gp[k] = nextG[k];
                zp[k] = nextZ[k];
                ap[k] = nextA[k];
            }
            UnpackToF<T, V>(gp[k], g);
            UnpackToF<T, V>(zp[k], u);
            Times(u, rstd);
            AddProducts(g, u, gw[k]);
            Times(g, w[k]);
            AddDot(g, u, dots);
        }
        if constexpr (RING) {
            const int64_t later = row + kAhead * static_cast<int64_t>(gridDim.x);
            if (later < a.rows) {
                fetch(later, stage);
            }
            CpAsyncCommit();
            stage = stage == kAhead - 1 ? 0 : stage + 1;
        } else if (row + gridDim.x < a.rows) {
            fetch(row + gridDim.x, 0);
        }
        // two sets of partial sums in turn: the next row's are written while a slow warp still reads this row's
        const float c = RowSum(Both(dots), part[turn]) * inverse * rstd;
        T* out = static_cast<T*>(a.gradX) + RowAt(row, a.inner, a.xs);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            if (col < a.width) {
                float v[V];
                UnpackToF<T, V>(gp[k], g);
                UnpackToF<T, V>(zp[k], u);
                UnpackToF<T, V>(ap[k], v);
                Times(g, w[k]);
                Times(u, -c);
                // gradSum + rstd (g - u c)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    v[i] = fmaf(rstd, g[i] + u[i], v[i]);
                }
                StoreF<T, V>(out + col, v);
            }
        }
    }
    if (a.scratch != nullptr) {
        float* s = a.scratch + static_cast<int64_t>(blockIdx.x) * a.width;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int32_t col = first + k * step;
            if (col < a.width) {
                StoreF<float, V>(s + col, gw[k]);
            }
        }
    }
}

// Rows too wide for the registers of a block: gradX with two passes over the row.
template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) RmsNormBwdWideKernel(BwdArgs a)
{
    __shared__ float part[32];
    const int64_t row = blockIdx.x;
    const T* gy = static_cast<const T*>(a.gradY) + RowAt(row, a.inner, a.gs);
    const T* z = static_cast<const T*>(a.sum) + RowAt(row, a.inner, a.ss);
    const T* s = a.gradSum != nullptr ? static_cast<const T*>(a.gradSum) + RowAt(row, a.inner, a.as) : nullptr;
    T* out = static_cast<T*>(a.gradX) + RowAt(row, a.inner, a.xs);
    const float rstd = a.rstd[row];
    float dot = 0.0f;
    const int32_t step = blockDim.x * V;
    for (int32_t col = threadIdx.x * V; col < a.width; col += step) {
        float g[V], u[V], w[V];
        LoadF<T, V>(gy + col, g);
        LoadF<T, V>(z + col, u);
        LoadWeight<T, V>(a.weight, a.weight32, col, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            dot = fmaf(g[i] * w[i], u[i] * rstd, dot);
        }
    }
    const float c = RowSum(dot, part) / static_cast<float>(a.width);
    for (int32_t col = threadIdx.x * V; col < a.width; col += step) {
        float g[V], u[V], w[V], v[V];
        LoadF<T, V>(gy + col, g);
        LoadF<T, V>(z + col, u);
        LoadWeight<T, V>(a.weight, a.weight32, col, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = 0.0f;
        }
        if (s != nullptr) {
            LoadF<T, V>(s + col, v);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[i] = fmaf(rstd, g[i] * w[i] - u[i] * rstd * c, v[i]);
        }
        StoreF<T, V>(out + col, v);
    }
}
// and the sums of the weight's gradient: a thread per column, a block per (columns, share of the rows); the shares, 64 at most, along y.
template <typename T>
__global__ void RmsNormWeightSumsKernel(BwdArgs a)
{
    const int32_t col = blockIdx.x * blockDim.x + threadIdx.x;
    if (col >= a.width) {
        return;
    }
    float acc = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = DType<T>::ToF(static_cast<const T*>(a.gradY)[RowAt(row, a.inner, a.gs) + col]);
        const float z = DType<T>::ToF(static_cast<const T*>(a.sum)[RowAt(row, a.inner, a.ss) + col]);
        acc = fmaf(g, z * a.rstd[row], acc);
    }
    a.scratch[static_cast<int64_t>(blockIdx.y) * a.width + col] = acc;
}

// The blocks' sums of one column, added in a fixed order: 32 warps take every 32nd block, then add up.
template <typename W>
__global__ void __launch_bounds__(1024) RmsNormWeightGradKernel(const float* scratch, int32_t blocks, int32_t width, W* out)
{
    __shared__ float part[32][33];
    const int32_t col = blockIdx.x * 32 + threadIdx.x;
    float acc = 0.0f;
    if (col < width) {
#pragma unroll 8
        for (int32_t b = threadIdx.y; b < blocks; b += 32) {
            acc += scratch[static_cast<int64_t>(b) * width + col];
        }
    }
    part[threadIdx.y][threadIdx.x] = acc;
    __syncthreads();
    const float sum = WarpSum(part[threadIdx.x][threadIdx.y]); // of column threadIdx.y
    const int32_t mine = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && mine < width) {
        out[mine] = DType<W>::FromF(sum);
    }
}

// ---- launch shapes ---------------------------------------------------------------------------------------------------------
// The widest vector that the row length, the row strides and the pointers allow.
struct RowUse {
    const void* p;
    RowStride s;
};
int VecOfRows(int elem, const NormShape& n, std::initializer_list<RowUse> uses)
{
    int v = 16 / elem;
    for (; v > 1; v >>= 1) {
        bool ok = n.width % v == 0;
        for (const RowUse& u : uses) {
            ok = ok && (u.p == nullptr || (Aligned(u.p, static_cast<size_t>(v) * elem) && u.s.s0 % v == 0 && u.s.s1 % v == 0));
        }
        if (ok) {
            break;
        }
    }
    return v;
}

// Threads of a row and chunks of V values per thread. Where rows are many, 256 threads with more chunks each: what a thread spends once a
// row is shared by more values (8192 x 4096 bf16 forward: 46 us against 49 with 512). Rows of up to 4 chunks a lane take one warp each, 4
// rows a block; wider ones a block of their own with as few chunks per thread as 512 threads allow, and up to 1024 threads with the most
// chunks that `values` a thread allow. nv 0: too wide for that.
struct RowShape {
    int nv, threads, rows;
};
RowShape ShapeOfRow(int32_t width, int v, int values, int mostThreads, int64_t rows)
{
    const int32_t wide = rows >= 4 * NumSMs() ? 256 : 512;
    const int32_t chunks = (width + v - 1) / v;
    if (chunks <= 32 * 4) {
        const int nv = chunks <= 32 ? 1 : (chunks <= 64 ? 2 : 4);
        if (nv * v <= values) {
            return {nv, 32, 4};
        }
    }
    for (int nv = 1; nv <= 8 && nv * v <= values; nv *= 2) {
        const bool last = nv == 8 || 2 * nv * v > values;
        const int32_t threads = ((chunks + nv - 1) / nv + 31) / 32 * 32;
        if (threads <= (last ? mostThreads : wide)) {
            return {nv, threads, 1};
        }
    }
    return {0, kMaxThreads, 1};
}

#define OPSCV_DISPATCH_NV(nv, NV, ...)                                 \
    {                                                                  \
        auto opscvNv_ = [&](auto opscvNvTag_) {                        \
            constexpr int NV = decltype(opscvNvTag_)::value;           \
            __VA_ARGS__;                                               \
        };                                                             \
        switch (nv) {                                                  \
            case 8: opscvNv_(std::integral_constant<int, 8>{}); break; \
            case 4: opscvNv_(std::integral_constant<int, 4>{}); break; \
            case 2: opscvNv_(std::integral_constant<int, 2>{}); break; \
            case 1: opscvNv_(std::integral_constant<int, 1>{}); break; \
            default: opscvNv_(std::integral_constant<int, 0>{}); break; \
        }                                                              \
    }

FwdArgs MakeFwd(const NormShape& n, const void* x, RowStride xs, const void* residual, RowStride rs, const void* weight,
                void* sum, RowStride ss)
{
    FwdArgs a{};
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.sum = sum;
    a.xs = xs;
    a.rs = rs;
    a.ss = ss;
    a.rows = n.rows;
    a.inner = n.inner;
    a.width = n.width;
    a.eps = static_cast<float>(n.eps);
    a.weight32 = n.weight32;
    return a;
}

bool GridFits(int64_t blocks) { return blocks <= INT32_MAX; }

} // namespace

cudaError_t RmsNormFwd(Dt dt, const NormShape& n, const void* x, RowStride xs, const void* residual, RowStride rs,
                       const void* weight, void* y, RowStride ys, void* sum, RowStride ss, float* rstd, cudaStream_t s)
{
    FwdArgs a = MakeFwd(n, x, xs, residual, rs, weight, sum, ss);
    a.y = y;
    a.ys = ys;
    a.rstd = rstd;
    const int v = VecOfRows(DtSize(dt), n,
                            {{x, xs}, {residual, rs}, {y, ys}, {sum, ss}, {n.weight32 ? nullptr : weight, {}}});
    const RowShape shape = ShapeOfRow(n.width, v, 32, kMaxThreads, n.rows);
    const int64_t blocks = CeilDiv(n.rows, shape.rows);
    if (!GridFits(blocks)) {
        return cudaErrorInvalidConfiguration;
    }
    const dim3 block(shape.threads, shape.rows);
    OPSCV_DISPATCH_DT(dt, T, OPSCV_DISPATCH_VEC(v, V, if constexpr (V * sizeof(T) <= 16) {
        OPSCV_DISPATCH_NV(shape.nv, NV, if constexpr (NV * V <= 32) {
            RmsNormFwdKernel<T, V, NV><<<static_cast<unsigned>(blocks), block, 0, s>>>(a);
        });
    }));
    CountLaunch();
    return cudaGetLastError();
}

cudaError_t RmsNormQuant(Dt dt, const NormShape& n, const void* x, RowStride xs, const void* residual, RowStride rs,
                         const void* weight, Q8 type, int32_t group, void* q, float* scales, void* sum, RowStride ss,
                         cudaStream_t s)
{
    FwdArgs a = MakeFwd(n, x, xs, residual, rs, weight, sum, ss);
    a.y = q;
    a.scales = scales;
    a.group = group > 0 ? group : n.width;
    a.groups = (n.width + a.group - 1) / a.group;
    int v = VecOfRows(DtSize(dt), n, {{x, xs}, {residual, rs}, {sum, ss}, {n.weight32 ? nullptr : weight, {}}});
    while (v > 1 && !(n.width % v == 0 && Aligned(q, v))) {
        v >>= 1;
    }
    // Groups of a power of two of columns that one to 32 lanes hold lie within a warp: lanes hold consecutive chunks of a row, and a
    // warp's first chunk starts a group. Others go through shared memory, with one row a block. 8192 x 5120 bf16 to e4m3: groups of 32, 64,
    // 128 and 256 68 us a call, through shared memory 106 to 112.
    const bool small = a.groups > 1 && (a.group & (a.group - 1)) == 0 && a.group <= 32 * v;
    // with groups in a warp, 512 threads a row are a little faster (8192 x 5120 bf16: 64 us against 68 with 256)
    RowShape shape = ShapeOfRow(n.width, v, 32, kMaxThreads, small ? 0 : n.rows);
    const bool inWarp = small && shape.nv > 0, ofRow = a.groups == 1 && shape.nv > 0;
    if (!inWarp && !ofRow) {
        shape.rows = 1;
    }
    const int64_t blocks = CeilDiv(n.rows, shape.rows);
    const size_t shared = inWarp || ofRow ? 0 : static_cast<size_t>(a.groups) * 4;
    if (!GridFits(blocks) || shared > 40 * 1024) {
        return cudaErrorInvalidConfiguration;
    }
    const dim3 block(shape.threads, shape.rows);
    const unsigned grid = static_cast<unsigned>(blocks);
    OPSCV_DISPATCH_DT(dt, T, OPSCV_DISPATCH_VEC(v, V, if constexpr (V * sizeof(T) <= 16) {
        OPSCV_DISPATCH_NV(shape.nv, NV, if constexpr (NV * V <= 32) {
            constexpr int Least = 32 / V; // lanes of a group of 32 columns
            auto launch = [&](auto tag) {
                constexpr Q8 Q = decltype(tag)::value;
                auto with = [&](auto lanes) {
                    constexpr int LG = decltype(lanes)::value;
                    if constexpr (LG <= 32 && (NV > 0 || LG == kShared)) {
                        RmsNormQuantKernel<T, V, NV, Q, LG><<<grid, block, shared, s>>>(a);
                    }
                };
                const int lanes = inWarp ? a.group / V : ofRow ? kRowScale : kShared;
                switch (lanes) {
                    case kShared: with(std::integral_constant<int, kShared>{}); break;
                    case kRowScale: with(std::integral_constant<int, kRowScale>{}); break;
                    case Least: with(std::integral_constant<int, Least>{}); break;
                    case 2 * Least: with(std::integral_constant<int, 2 * Least>{}); break;
                    case 4 * Least: with(std::integral_constant<int, 4 * Least>{}); break;
                    default: with(std::integral_constant<int, 8 * Least>{}); break;
                }
            };
            if (type == Q8::E4M3) {
                launch(std::integral_constant<Q8, Q8::E4M3>{});
            } else {
                launch(std::integral_constant<Q8, Q8::INT8>{});
            }
        });
    }));
    CountLaunch();
    return cudaGetLastError();
}

namespace {

// The backward's grid: the weight's gradient takes a row of fp32 sums per block, so the blocks walk the rows, as many of them as
// the device holds at once (about 1024 threads an SM: two blocks of 512 or more of fewer threads).
struct BwdPlan {
    int v;
    RowShape shape;
    int64_t blocks;
};
BwdPlan PlanBwd(int v, const NormShape& n)
{
    BwdPlan p{};
    p.v = v;
    const int mostNv = v >= kBwdValues / 8 ? kBwdValues / v : 8;
    p.shape = ShapeOfRow(n.width, v, kBwdValues, BwdThreads(mostNv, v), 0);
    if (p.shape.nv > 0 && p.shape.threads == 32 && p.shape.rows > 1) {
        // one row a block here too, of as many warps as give each lane one chunk
        const int32_t chunks = (n.width + v - 1) / v;
        p.shape.nv = 1;
        p.shape.threads = (chunks + 31) / 32 * 32;
        p.shape.rows = 1;
    }
    if (p.shape.nv > 0) {
        const int perSm = p.shape.threads >= 512 ? (p.shape.threads > 512 ? 1 : 2) : 1024 / p.shape.threads;
        p.blocks = static_cast<int64_t>(NumSMs()) * (perSm < 16 ? perSm : 16);
    } else {
        p.blocks = 64;
    }
    p.blocks = p.blocks < n.rows ? p.blocks : n.rows;
    return p;
}

} // namespace

int64_t RmsNormBwdScratch(Dt dt, const NormShape& n, bool weight)
{
    if (!weight) {
        return 0;
    }
    int64_t most = 0; // the vector width is known only with the pointers
    for (int v = 16 / DtSize(dt); v >= 1; v >>= 1) {
        const int64_t b = PlanBwd(v, n).blocks;
        most = b > most ? b : most;
    }
    return most * n.width;
}

cudaError_t RmsNormBwd(Dt dt, const NormShape& n, const void* gradY, RowStride gs, const void* sum, RowStride ss,
                       const float* rstd, const void* weight, const void* gradSum, RowStride as, void* gradX,
                       RowStride xs, void* gradWeight, float* scratch, int64_t scratchFloats, cudaStream_t s)
{
    if (n.rows == 0) { // no rows: the weight's gradient is zero
        return gradWeight == nullptr ? cudaSuccess :
                                       cudaMemsetAsync(gradWeight, 0, static_cast<size_t>(n.width) * (n.weight32 ? 4 : DtSize(dt)), s);
    }
    BwdArgs a{};
    a.gradY = gradY;
    a.sum = sum;
    a.weight = weight;
    a.gradSum = gradSum;
    a.rstd = rstd;
    a.gradX = gradX;
    a.scratch = gradWeight != nullptr ? scratch : nullptr;
    a.gs = gs;
    a.ss = ss;
    a.as = as;
    a.xs = xs;
    a.rows = n.rows;
    a.inner = n.inner;
    a.width = n.width;
    a.weight32 = n.weight32;
    const int v = VecOfRows(DtSize(dt), n,
                            {{gradY, gs}, {sum, ss}, {gradSum, as}, {gradX, xs}, {n.weight32 ? nullptr : weight, {}}});
    BwdPlan p = PlanBwd(v, n);
    if (gradWeight != nullptr) { // the scratch was sized in the first phase
        const int64_t room = scratchFloats / n.width;
        p.blocks = p.blocks < room ? p.blocks : room;
    }
    if (p.shape.nv == 0) {
        if (!GridFits(n.rows)) {
            return cudaErrorInvalidConfiguration;
        }
        if (a.scratch != nullptr) { // before gradX, which may lie over gradY
            const dim3 grid(static_cast<unsigned>(CeilDiv(n.width, 256)), static_cast<unsigned>(p.blocks));
            OPSCV_DISPATCH_DT(dt, T, RmsNormWeightSumsKernel<T><<<grid, 256, 0, s>>>(a));
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess) {
                return e;
            }
            CountLaunch();
        }
        OPSCV_DISPATCH_DT(dt, T, OPSCV_DISPATCH_VEC(v, V, if constexpr (V * sizeof(T) <= 16) {
            RmsNormBwdWideKernel<T, V><<<static_cast<unsigned>(n.rows), kMaxThreads, 0, s>>>(a);
        }));
    } else {
        cudaError_t failed = cudaSuccess;
        OPSCV_DISPATCH_DT(dt, T, OPSCV_DISPATCH_VEC(v, V, if constexpr (V * sizeof(T) <= 16) {
            OPSCV_DISPATCH_NV(p.shape.nv, NV, if constexpr (NV > 0 && NV * V <= kBwdValues) {
                if constexpr (V * sizeof(T) == 16) {
                    static std::atomic<uint64_t> asked;
                    const int shared = RingBytes(NV, p.shape.threads);
                    const cudaError_t e = AskOnce(RmsNormBwdKernel<T, V, NV, true>, asked, RingBytes(NV, 512));
                    if (e != cudaSuccess) {
                        failed = e;
                    } else {
                        RmsNormBwdKernel<T, V, NV, true><<<static_cast<unsigned>(p.blocks), p.shape.threads, shared, s>>>(a);
                    }
                } else {
                    RmsNormBwdKernel<T, V, NV, false><<<static_cast<unsigned>(p.blocks), p.shape.threads, 0, s>>>(a);
                }
            });
        }));
        if (failed != cudaSuccess) {
            return failed;
        }
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) { // no sums to make gradWeight of
        return e;
    }
    CountLaunch();
    if (gradWeight != nullptr) {
        const unsigned grid = static_cast<unsigned>(CeilDiv(n.width, 32));
        const dim3 block(32, 32);
        if (n.weight32) {
            RmsNormWeightGradKernel<float><<<grid, block, 0, s>>>(scratch, static_cast<int32_t>(p.blocks), n.width,
                                                                  static_cast<float*>(gradWeight));
        } else {
            OPSCV_DISPATCH_DT(dt, T, RmsNormWeightGradKernel<T><<<grid, block, 0, s>>>(scratch, static_cast<int32_t>(p.blocks),
                                                                                      n.width, static_cast<T*>(gradWeight)));
        }
        CountLaunch();
    }
    return cudaGetLastError();
}

} // namespace opscv
