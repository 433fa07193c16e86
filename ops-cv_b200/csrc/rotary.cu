// Rotary positions: the pairs (a, b) of a head's first 2 * half values are turned by the angle position * frequency,
//   a' = (a cos - b sin) * scale, b' = (b cos + a sin) * scale,
// pair i being values (i, i + half) or, interleaved, (2i, 2i + 1). The backward turns by the negative angle.
//
// Bound by HBM: q and k move once each way. The angle is formed and reduced to a turn of [-1/2, 1/2] in 64 bits and more (in 32 bits
// the angle of a position of 10^6 is off by up to 1/16); after that fp32 is enough for its sine and cosine. They depend on the token
// and the frequency alone, so a block forms them once for its tokens, in shared memory, and all heads of q and k use them.
// 16384 tokens of 40 heads of 128, bf16: 65 us (5.2 TB/s); 2 x 4099 tokens of 32 heads of 80, three axes, fp16: 24 us; 32 tokens: 2.7 us.
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

// An item is V values of the pairs' first half and V of their second (half layout), V / 2 pairs (interleaved), or values that are
// copied: V, in the half layout twice V, so that all threads of a block have the same to move (8192 tokens, 40 heads of 128, 64 of which
// turn, bf16: 47 us with V, 38 us so). A thread reads all it needs of an item before it writes, so out may be in.
template <typename T, int V>
struct Item {
    Pack<T, V> a, b;
    __device__ __forceinline__ void Load(const T* p, int32_t second, bool both)
    {
        a = *reinterpret_cast<const Pack<T, V>*>(p);
        if (both) {
            b = *reinterpret_cast<const Pack<T, V>*>(p + second);
        }
    }
};

// Which product is rounded is written out, so that all widths and layouts give the same bits.
__device__ __forceinline__ void TurnPair(float& x, float& y, float cs, float sn)
{
    const float u = fmaf(x, cs, -Mul(y, sn));
    y = fmaf(y, cs, Mul(x, sn));
    x = u;
}

// A block has a few tokens. Threads are (item of a head) x (heads) x (tokens); each has kHeads heads of one or two tokens at a time: its
// addresses serve all the tokens, and all its loads are on their way while the block forms the sines and cosines. Heads of a thread, a
// call of 2, 3 and 4: 16384 tokens, 40 heads of 128, bf16, halves 78, 71 and 74 us; 64 values of them, neighbours 82, 67 and 69; 2 x 4099
// tokens, 32 heads of 80, three axes, fp16 29, 27 and 31.
constexpr int kHeads = 3;
// two tokens at a time, one where a pair's values lie apart and take twice the registers
constexpr int TokensAtATime(bool interleaved) { return interleaved ? 2 : 1; }

__host__ __device__ constexpr int32_t CopiedItems(int32_t values, int32_t v, bool interleaved)
{
    return interleaved ? values / v : (values / v + 1) / 2;
}

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kThreads, INTER ? 4 : 3) RotaryKernel(const __grid_constant__ Args a)
{
    __shared__ __align__(16) float cosines[kTable], sines[kTable]; // [token][frequency]
    constexpr int kTokens = TokensAtATime(INTER);
    const int32_t half = a.r.half;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.tokensPerBlock;
    const int32_t tokens = static_cast<int32_t>(min(static_cast<int64_t>(a.tokensPerBlock), a.r.tokens - first));
    const int32_t threads = blockDim.x * blockDim.y * blockDim.z;
    constexpr bool kNeighbours = INTER && V > 1; // pairs within an item
    const int32_t turned = kNeighbours ? 2 * half / V : half / V; // items of a head that are turned
    const int32_t items = turned + CopiedItems(a.r.dim - 2 * half, V, INTER);
    const int32_t heads = a.q.heads + a.k.heads;
    bool ready = false; // the table
    // all threads of the block make the same turns of these loops
    for (int32_t item0 = 0; item0 < items; item0 += blockDim.x) {
        const int32_t item = item0 + threadIdx.x;
        const bool turn = item < turned;
        // the item's values, and those of the second half (interleaved single values: the pair's second)
        const int32_t at = !turn ? 2 * half + (item - turned) * (INTER ? V : 2 * V) : INTER && V == 1 ? 2 * item : item * V;
        const int32_t second = kNeighbours ? -1 : !turn ? (!INTER && at + V < a.r.dim ? at + V : -1) : INTER ? at + 1 : half + at;
        for (int32_t h0 = 0; h0 < heads; h0 += kHeads * blockDim.y) {
            int64_t in[kHeads], out[kHeads];
            bool ofQ[kHeads], inside[kHeads];
#pragma unroll
            for (int i = 0; i < kHeads; ++i) {
                const int32_t h = h0 + threadIdx.y + i * blockDim.y;
                inside[i] = item < items && h < heads;
                ofQ[i] = h < a.q.heads;
                in[i] = (ofQ[i] ? h * a.q.inHead : (h - a.q.heads) * a.k.inHead) + at;
                out[i] = (ofQ[i] ? h * a.q.outHead : (h - a.q.heads) * a.k.outHead) + at;
            }
            for (int32_t t0 = 0; t0 < tokens; t0 += kTokens * blockDim.z) {
                Item<T, V> x[kTokens][kHeads];
#pragma unroll
                for (int y = 0; y < kTokens; ++y) {
                    const int32_t t = t0 + threadIdx.z + y * blockDim.z;
                    if (t < tokens) {
                        const T* q = static_cast<const T*>(a.q.in) + TokenAt(first + t, a.r.inner, a.q.inTok);
                        const T* k = static_cast<const T*>(a.k.in) + TokenAt(first + t, a.r.inner, a.k.inTok);
#pragma unroll
                        for (int i = 0; i < kHeads; ++i) {
                            if (inside[i]) {
                                x[y][i].Load((ofQ[i] ? q : k) + in[i], second - at, second >= 0);
                            }
                        }
                    }
                }
                if (!ready) {
                    ready = true;
                    const int32_t me = (threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + threadIdx.x;
                    for (int32_t e = me; e < tokens * half; e += threads) {
                        const int32_t t = e / half, i = e - t * half;
                        int axis = 0;
                        while (axis < a.r.axes - 1 && i >= a.r.ends[axis]) {
                            ++axis;
                        }
                        const int64_t from = TokenAt(first + t, a.r.inner, a.r.posTok) + axis * a.r.posAxis;
                        const double p = a.r.pos64 ? static_cast<double>(static_cast<const long long*>(a.positions)[from]) :
                                                     static_cast<double>(static_cast<const int*>(a.positions)[from]);
                        const double f = a.r.freq64 ? static_cast<const double*>(a.frequencies)[i] :
                                                      static_cast<double>(static_cast<const float*>(a.frequencies)[i]);
                        // In turns, p * f / (2 pi): the whole ones fall away, the rest keeps its leading bits in fp32. 1 / (2 pi) and
                        // the products are sums of two doubles, so that positions of 10^12 and more, whose angle in one double is off
                        // by 10^-4, keep theirs.
                        constexpr double kHigh = 0.15915494309189535, kLow = -9.839338337591243e-18; // 1 / (2 pi)
                        const double fHigh = f * kHigh, fLow = fma(f, kHigh, -fHigh) + f * kLow;
                        const double high = p * fHigh, low = fma(p, fHigh, -high) + p * fLow;
                        float sn, cs;
                        sincospif(2.0f * static_cast<float>((high - rint(high)) + low), &sn, &cs);
                        cosines[e] = cs * a.r.scale;
                        sines[e] = (a.r.inverse ? -sn : sn) * a.r.scale;
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int y = 0; y < kTokens; ++y) {
                    const int32_t t = t0 + threadIdx.z + y * blockDim.z;
                    if (t >= tokens) {
                        break;
                    }
                    T* q = static_cast<T*>(a.q.out) + TokenAt(first + t, a.r.inner, a.q.outTok);
                    T* k = static_cast<T*>(a.k.out) + TokenAt(first + t, a.r.inner, a.k.outTok);
                    constexpr int kOwn = kNeighbours ? V / 2 : V;
                    float cs[kOwn], sn[kOwn];
                    if (turn) {
                        const int32_t from = t * half + item * kOwn;
                        if (half % kOwn == 0) { // aligned to the item's frequencies
                            *reinterpret_cast<Pack<float, kOwn>*>(cs) = *reinterpret_cast<const Pack<float, kOwn>*>(cosines + from);
                            *reinterpret_cast<Pack<float, kOwn>*>(sn) = *reinterpret_cast<const Pack<float, kOwn>*>(sines + from);
                        } else {
#pragma unroll
                            for (int e = 0; e < kOwn; ++e) {
                                cs[e] = cosines[from + e];
                                sn[e] = sines[from + e];
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kHeads; ++i) {
                        if (!inside[i]) {
                            break;
                        }
                        T* to = (ofQ[i] ? q : k) + out[i];
                        if (!turn) {
                            *reinterpret_cast<Pack<T, V>*>(to) = x[y][i].a;
                            if (second >= 0) {
                                *reinterpret_cast<Pack<T, V>*>(to + (second - at)) = x[y][i].b;
                            }
                            continue;
                        }
                        float u[V];
                        UnpackToF<T, V>(x[y][i].a, u);
                        if constexpr (kNeighbours) {
#pragma unroll
                            for (int e = 0; e < V / 2; ++e) {
                                TurnPair(u[2 * e], u[2 * e + 1], cs[e], sn[e]);
                            }
                        } else {
                            float v[V];
                            UnpackToF<T, V>(x[y][i].b, v);
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                TurnPair(u[e], v[e], cs[e], sn[e]);
                            }
                            StorePack<T, V>(to + (second - at), v);
                        }
                        StorePack<T, V>(to, u);
                    }
                }
            }
        }
    }
}

// f_i = base^(-i / half), scaled for contexts longer than the trained ones. The rules of "base", "wavelength" and "ramp" (which frequencies
// stay, which are divided, the blend between) follow B. Peng et al., "YaRN: Efficient Context Window Extension of Large Language
// Models", 2023.
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
        // the same, blended linearly over the frequencies' indices between those that turn `high` and `low` times, as far as there are
        // such indices
        const double first = floor(half * log(originalLength / (high * 2.0 * pi)) / log(base));
        const double last = ceil(half * log(originalLength / (low * 2.0 * pi)) / log(base));
        const double a = first < 0.0 ? 0.0 : first;
        const double b = last > 2.0 * half - 1.0 ? 2.0 * half - 1.0 : last;
        double stretch = b > a ? (i - a) / (b - a) : i > b ? 1.0 : 0.0; // b < a: all turn less than `low` times, or all more than `high`
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
    // Threads: the items of a head by the heads, kHeads to each, by as many tokens as make up to 256. Tokens: as many as the threads take
    // at a time, but at least some blocks for each SM, and no more than the table holds.
    const int32_t turned = r.interleaved && v > 1 ? 2 * r.half / v : r.half / v, items = turned + CopiedItems(r.dim - 2 * r.half, v, r.interleaved);
    const int32_t heads = q.heads + k.heads;
    const int32_t across = items < kThreads ? items : kThreads;
    int32_t down = static_cast<int32_t>(CeilDiv(heads, kHeads));
    down = down < kThreads / across ? down : kThreads / across;
    int32_t deep = kThreads / (across * down);
    int64_t t = static_cast<int64_t>(TokensAtATime(r.interleaved)) * deep;
    const int64_t spread = CeilDiv(r.tokens, static_cast<int64_t>(NumSMs()) * 4);
    t = t < spread ? t : spread;
    const int64_t room = kTable / (r.half < 1 ? 1 : r.half);
    t = t < room ? t : room;
    t = t < 1 ? 1 : t;
    a.tokensPerBlock = static_cast<int32_t>(t);
    deep = deep < t ? deep : static_cast<int32_t>(t);
    deep = deep < 64 ? deep : 64; // a block's limit
    const dim3 block(across, down, deep);
    const int64_t blocks = CeilDiv(r.tokens, t);
    if (blocks > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    OPSCV_DISPATCH_DT(dt, T, OPSCV_DISPATCH_VEC(v, V, if constexpr (V * sizeof(T) <= 16) {
        if (r.interleaved) {
            RotaryKernel<T, V, true><<<static_cast<unsigned>(blocks), block, 0, s>>>(a);
        } else {
            RotaryKernel<T, V, false><<<static_cast<unsigned>(blocks), block, 0, s>>>(a);
        }
    }));
    CountLaunch();
    return cudaGetLastError();
}

} // namespace opscv
