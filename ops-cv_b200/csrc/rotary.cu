// Rotary positions: the pairs (a, b) of a head's first 2 * half values are turned by the angle position * frequency,
//   a' = (a cos - b sin) * scale, b' = (b cos + a sin) * scale,
// pair i being values (i, i + half) or, interleaved, (2i, 2i + 1). The backward turns by the negative angle.
//
// Bound by HBM: q and k move once each way. The angle is formed and reduced to a turn of [-1/2, 1/2] in 64 bits and more (in 32 bits
// the angle of a position of 10^6 is off by up to 1/16); after that fp32 is enough for its sine and cosine. They depend on the token
// and the frequency alone, so a block forms them once for its tokens, in shared memory, and all heads of q and k use them.
#include "launch_util.cuh"
#include "sequence_kernels.h"

namespace opscv {

namespace {

constexpr int kThreads = 256;
constexpr int kTable = 2048; // (token, frequency) pairs of a block at most: 16 KiB of sines and cosines

struct Args {
    RotaryShape r;
    RotaryTensor q, k;
    const void* positions;
    const void* frequencies;
    int32_t tokensPerBlock;
};

__device__ __forceinline__ int64_t TokenAt(int64_t token, int64_t inner, RowStride s)
{
    return token < inner ? token * s.s1 : token / inner * s.s0 + token % inner * s.s1;
}

// One item of V values of a pair's first half and V of its second (half layout), of V / 2 pairs (interleaved), or V values that
// are copied. A thread reads all it needs of an item before it writes, so out may be in.
template <typename T, int V>
__device__ __forceinline__ void TurnItem(const Args& a, const T* in, T* out, int32_t item, int32_t turned, const float2* table)
{
    const int32_t half = a.r.half;
    if (item >= turned) {
        const int32_t c = 2 * half + (item - turned) * V;
        *reinterpret_cast<Pack<T, V>*>(out + c) = *reinterpret_cast<const Pack<T, V>*>(in + c);
        return;
    }
    if (a.r.interleaved) {
        if constexpr (V >= 2) {
            float v[V];
            LoadPack<T, V>(in + item * V, v);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 cs = table[item * (V / 2) + i];
                const float x = v[2 * i], y = v[2 * i + 1];
                v[2 * i] = x * cs.x - y * cs.y;
                v[2 * i + 1] = y * cs.x + x * cs.y;
            }
            StorePack<T, V>(out + item * V, v);
        } else {
            const float2 cs = table[item];
            const float x = DType<T>::ToF(in[2 * item]), y = DType<T>::ToF(in[2 * item + 1]);
            out[2 * item] = DType<T>::FromF(x * cs.x - y * cs.y);
            out[2 * item + 1] = DType<T>::FromF(y * cs.x + x * cs.y);
        }
        return;
    }
    float x[V], y[V];
    const int32_t c = item * V;
    LoadPack<T, V>(in + c, x);
    LoadPack<T, V>(in + half + c, y);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 cs = table[c + i];
        const float u = x[i] * cs.x - y[i] * cs.y;
        y[i] = y[i] * cs.x + x[i] * cs.y;
        x[i] = u;
    }
    StorePack<T, V>(out + c, x);
    StorePack<T, V>(out + half + c, y);
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) RotaryKernel(Args a)
{
    __shared__ float2 table[kTable];
    const int32_t half = a.r.half;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.tokensPerBlock;
    const int32_t tokens = static_cast<int32_t>(min(static_cast<int64_t>(a.tokensPerBlock), a.r.tokens - first));
    for (int32_t e = threadIdx.x; e < tokens * half; e += kThreads) {
        const int32_t t = e / half, i = e - t * half;
        int axis = 0;
        while (axis < a.r.axes - 1 && i >= a.r.ends[axis]) {
            ++axis;
        }
        const int64_t at = TokenAt(first + t, a.r.inner, a.r.posTok) + axis * a.r.posAxis;
        const double p = a.r.pos64 ? static_cast<double>(static_cast<const long long*>(a.positions)[at]) :
                                     static_cast<double>(static_cast<const int*>(a.positions)[at]);
        const double f = a.r.freq64 ? static_cast<const double*>(a.frequencies)[i] :
                                      static_cast<double>(static_cast<const float*>(a.frequencies)[i]);
        // In turns, p * f / (2 pi): the whole ones fall away, the rest keeps its leading bits in fp32. 1 / (2 pi) and the products
        // are sums of two doubles, so that positions of 10^12 and more, whose angle in one double is off by 10^-4, keep theirs.
        constexpr double kHigh = 0.15915494309189535, kLow = -9.839338337591243e-18; // 1 / (2 pi)
        const double fHigh = f * kHigh, fLow = fma(f, kHigh, -fHigh) + f * kLow;
        const double high = p * fHigh, low = fma(p, fHigh, -high) + p * fLow;
        float sn, cs;
        sincospif(2.0f * static_cast<float>((high - rint(high)) + low), &sn, &cs);
        table[e] = make_float2(cs * a.r.scale, (a.r.inverse ? -sn : sn) * a.r.scale);
    }
    __syncthreads();
    const int32_t turned = a.r.interleaved && V > 1 ? 2 * half / V : half / V;
    const int32_t items = turned + (a.r.dim - 2 * half) / V; // of a head
    const int32_t heads = a.q.heads + a.k.heads;
    const int32_t perToken = heads * items;
    for (int32_t e = threadIdx.x; e < tokens * perToken; e += kThreads) {
        const int32_t t = e / perToken;
        const int32_t rest = e - t * perToken;
        int32_t head = rest / items;
        const int32_t item = rest - head * items;
        const bool ofK = head >= a.q.heads;
        head -= ofK ? a.q.heads : 0;
        const RotaryTensor& x = ofK ? a.k : a.q;
        const T* in = static_cast<const T*>(x.in) + TokenAt(first + t, a.r.inner, x.inTok) + head * x.inHead;
        T* out = static_cast<T*>(x.out) + TokenAt(first + t, a.r.inner, x.outTok) + head * x.outHead;
        if (in == out && item >= turned) {
            continue; // the copied part of a head that is turned in place
        }
        TurnItem<T, V>(a, in, out, item, turned, table + t * half);
    }
}

// f_i = base^(-i / half), scaled for contexts longer than the trained ones.
__global__ void RotaryFrequenciesKernel(void* out, bool is64, int32_t half, double base, RotaryScaling kind, double factor,
                                        double originalLength, double low, double high)
{
    const int32_t i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= half) {
        return;
    }
    const double pi = 3.14159265358979323846;
    if (kind == RotaryScaling::BASE && half > 1) {
        base *= pow(factor, static_cast<double>(half) / (half - 1));
    }
    double f = pow(base, -static_cast<double>(i) / half);
    if (kind == RotaryScaling::LINEAR) {
        f /= factor;
    } else if (kind == RotaryScaling::WAVELENGTH) {
        // periods that the trained length holds at least `high` times stay, those that it holds at most `low` times are
        // stretched, the ones between are blended
        const double times = originalLength * f / (2.0 * pi);
        double keep = (times - low) / (high - low);
        keep = keep < 0.0 ? 0.0 : (keep > 1.0 ? 1.0 : keep);
        f = f * keep + f / factor * (1.0 - keep);
    } else if (kind == RotaryScaling::RAMP) {
        // the same, blended linearly over the frequencies' indices between those that turn `high` and `low` times
        const double first = floor(half * log(originalLength / (high * 2.0 * pi)) / log(base));
        const double last = ceil(half * log(originalLength / (low * 2.0 * pi)) / log(base));
        const double a = first < 0.0 ? 0.0 : first;
        double b = last > 2.0 * half - 1.0 ? 2.0 * half - 1.0 : last;
        b = b <= a ? a + 0.001 : b;
        double stretch = (i - a) / (b - a);
        stretch = stretch < 0.0 ? 0.0 : (stretch > 1.0 ? 1.0 : stretch);
        f = f * (1.0 - stretch) + f / factor * stretch;
    }
    if (is64) {
        static_cast<double*>(out)[i] = f;
    } else {
        static_cast<float*>(out)[i] = static_cast<float>(f);
    }
}

} // namespace

cudaError_t RotaryFrequencies(void* out, bool is64, int32_t half, double base, RotaryScaling kind, double factor,
                              double originalLength, double low, double high, cudaStream_t s)
{
    RotaryFrequenciesKernel<<<static_cast<unsigned>(CeilDiv(half, 64)), 64, 0, s>>>(out, is64, half, base, kind, factor,
                                                                                    originalLength, low, high);
    CountLaunch();
    return cudaGetLastError();
}

cudaError_t RotaryTurn(Dt dt, const RotaryShape& r, const RotaryTensor& q, const RotaryTensor& k, const void* positions,
                       const void* frequencies, cudaStream_t s)
{
    if (r.half > kTable) {
        return cudaErrorInvalidValue;
    }
    const int elem = DtSize(dt);
    int v = 16 / elem;
    for (; v > 1; v >>= 1) {
        bool ok = r.dim % v == 0 && (r.interleaved ? 2 * r.half : r.half) % v == 0;
        for (const RotaryTensor* x : {&q, &k}) {
            if (x->heads > 0) {
                ok = ok && Aligned(x->in, static_cast<size_t>(v) * elem) && Aligned(x->out, static_cast<size_t>(v) * elem) &&
                     x->inHead % v == 0 && x->outHead % v == 0 && x->inTok.s0 % v == 0 && x->inTok.s1 % v == 0 &&
                     x->outTok.s0 % v == 0 && x->outTok.s1 % v == 0;
            }
        }
        if (ok) {
            break;
        }
    }
    Args a{};
    a.r = r;
    a.q = q;
    a.k = k;
    a.positions = positions;
    a.frequencies = frequencies;
    // Tokens per block: about four items a thread, so that the sines' time hides behind other blocks' copies, but at least a
    // block per SM slot, and no more than the table holds.
    const int64_t perToken = static_cast<int64_t>(q.heads + k.heads) * CeilDiv(r.dim, r.interleaved ? v : 2 * v);
    int64_t t = CeilDiv(4 * kThreads, perToken < 1 ? 1 : perToken);
    const int64_t spread = CeilDiv(r.tokens, static_cast<int64_t>(NumSMs()) * 8);
    t = t < spread ? t : spread;
    const int64_t room = kTable / (r.half < 1 ? 1 : r.half);
    t = t < room ? t : room;
    t = t < 1 ? 1 : t;
    a.tokensPerBlock = static_cast<int32_t>(t);
    const int64_t blocks = CeilDiv(r.tokens, t);
    if (blocks > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    OPSCV_DISPATCH_DT(dt, T, OPSCV_DISPATCH_VEC(v, V, if constexpr (V * sizeof(T) <= 16) {
        RotaryKernel<T, V><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(a);
    }));
    CountLaunch();
    return cudaGetLastError();
}

} // namespace opscv
