// Attention over a sliding window with sinks in fp32 arithmetic, tile by tile: fp32 tensors, heads of more than 128 values, and 16-bit
// tensors that boxes cannot be loaded from.
//
// Bound by the fp32 pipes and the reads of shared memory that feed them: 4 (forward) and 14 (backward) operations for each pair and value,
// packed in twos, of which a 2 x 8 (4 x 4) block of a tile's products in a thread's registers takes 64 for 10 (8) reads of 16 bytes.
// 2 x 777 tokens, window 200, 6 heads of 72 on 2: 43 us forward, 180 us backward; 2 x 1500, window 512, 16 heads of 128 on 4: 477 us and
// 1548 us. Tensor cores would need three products of tf32 parts for
// each of fp32 and still lose bits that fp32 callers have. Blocks own their sums (gradQ in one kernel, gradK and gradV in another), so
// nothing is added up in memory and the order of all sums is fixed.
#include <algorithm>

#include "cp_async.cuh"
#include "window_attention.cuh"

namespace opscv {

namespace {

// DP: values of a head, padded to a multiple of 32. Rows of a tile as `a` (whose sums a block owns, A of them) and as `b` (that it walks, B
// of them): a thread has rows ty + kRows r of a and tx + kCols c of b. Reads of shared memory are the limit, so a thread has as many rows of
// both as registers and the number of warps allow: 4 x 4 of 64 rows; 2 x 8 of 32 (16 x 16 threads with 2 x 4 each: 56 us against 43 at 2 x 777
// tokens, 6 heads of 72 on 2; 2 x 8 of 64 rows: 564 us against 463 of 4 x 4 at 2 x 1500 tokens, 16 heads of 128 on 4, window 512).
template <int DP, int A, int B>
struct Tile {
    static constexpr int kCols = A == 32 && DP <= 128 ? 8 : 16; // threads along b's rows
    static constexpr int kA = A == 64 ? 4 : 2, kB = B / kCols;
    static constexpr int kRows = A / kA; // threads along a's rows
    static constexpr int kThreads = kCols * kRows;
    static constexpr int kChunks = DP / 32, kPairs = 16 / kCols; // a thread's pairs of values of a row
    static constexpr int kStride = DP + 4; // floats of a row: 4 more shift neighbouring rows to other banks
    static constexpr int kWeights = B + 4; // the same for the rows of weights
    static constexpr int kFloatsA = A * kStride, kFloatsB = B * kStride;
    static constexpr int kWeightFloats = A * kWeights;
};

// Rows of one head as fp32, zeros for rows behind `end` and values behind dim: `from` and the next, those from `split` on `jump` rows
// further down (a walk's sinks and its window). fp32 rows that can be read 16 bytes at a
// time are copied asynchronously: the caller commits and waits, and the copies of the next step run under the products of this one.
template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void LoadTile(float* dst, const AttnTensor& t, int32_t b, int32_t h, int32_t from, int32_t end, int32_t dim,
                                         bool vec, int32_t split = 0, int32_t jump = 0)
{
    constexpr int kStride = DP + 4;
    const T* base = RowOf<T>(t, b, 0, h);
    auto rowAt = [&](int r) { return from + r < split ? from + r : from + r + jump; };
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
            for (int e = threadIdx.x; e < ROWS * (DP / 4); e += THREADS) {
                const int r = e / (DP / 4), d = e % (DP / 4) * 4;
                const int32_t row = rowAt(r);
                const bool live = row < end && d < dim;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (r * kStride + d) * 4),
                             "l"(live ? base + row * t.l + d : base), "r"(live ? 16 : 0)
                             : "memory");
            }
            return;
        }
    }
    if (vec) {
#pragma unroll 4
        for (int e = threadIdx.x; e < ROWS * (DP / 4); e += THREADS) {
            const int r = e / (DP / 4), d = e % (DP / 4) * 4;
            const int32_t row = rowAt(r);
            float v[4] = {};
            if (row < end && d < dim) {
                LoadPack<T, 4>(base + row * t.l + d, v);
            }
            *reinterpret_cast<float4*>(dst + r * kStride + d) = make_float4(v[0], v[1], v[2], v[3]);
        }
    } else {
        for (int e = threadIdx.x; e < ROWS * DP; e += THREADS) {
            const int r = e / DP, d = e % DP;
            const int32_t row = rowAt(r);
            dst[r * kStride + d] = row < end && d < dim ? DType<T>::ToF(base[row * t.l + d]) : 0.0f;
        }
    }
}

__device__ __forceinline__ void ReadQuad(const float* p, F2 (&v)[2])
{
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(p);
    v[0].r = x.x;
    v[1].r = x.y;
}

// s[r][c] = row (ty + kRows r) of a . row (tx + kCols c) of b, over the dim values (the rows hold zeros behind them); even and odd values
// are summed apart
template <typename L>
__device__ __forceinline__ void Inner(const float* a, const float* b, int32_t dim, float (&s)[L::kA][L::kB])
{
    const int tx = threadIdx.x % L::kCols, ty = threadIdx.x / L::kCols;
    F2 sum[L::kA][L::kB];
#pragma unroll
    for (int r = 0; r < L::kA; ++r) {
#pragma unroll
        for (int c = 0; c < L::kB; ++c) {
            sum[r][c] = MakeF2(0.0f, 0.0f);
        }
    }
    const float* pa = a + ty * L::kStride;
    const float* pb = b + tx * L::kStride;
#pragma unroll 2
    for (int d = 0; d < dim; d += 4) {
        F2 x[L::kA][2], y[L::kB][2];
#pragma unroll
        for (int r = 0; r < L::kA; ++r) {
            ReadQuad(pa + L::kRows * r * L::kStride + d, x[r]);
        }
#pragma unroll
        for (int c = 0; c < L::kB; ++c) {
            ReadQuad(pb + L::kCols * c * L::kStride + d, y[c]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int r = 0; r < L::kA; ++r) {
#pragma unroll
                for (int c = 0; c < L::kB; ++c) {
                    sum[r][c] = Fma2(x[r][k], y[c][k], sum[r][c]);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < L::kA; ++r) {
#pragma unroll
        for (int c = 0; c < L::kB; ++c) {
            float even, odd;
            SplitF2(sum[r][c], even, odd);
            s[r][c] = even + odd;
        }
    }
}

// A thread's sums of a row: kPairs pairs of values from 2 kPairs tx + 32 c on.
template <typename L>
struct Sums {
    F2 v[L::kA][L::kChunks][L::kPairs];
    __device__ __forceinline__ Sums()
    {
#pragma unroll
        for (int r = 0; r < L::kA; ++r) {
#pragma unroll
            for (int c = 0; c < L::kChunks; ++c) {
                for (int e = 0; e < L::kPairs; ++e) {
                    v[r][c][e] = MakeF2(0.0f, 0.0f);
                }
            }
        }
    }
};

// o[r] += sum over j of w[ty + kRows r][j] row j of v (B rows)
template <typename L, int B>
__device__ __forceinline__ void Outer(const float* w, const float* v, Sums<L>& o)
{
    const int tx = threadIdx.x % L::kCols, ty = threadIdx.x / L::kCols;
    const float* pw = w + ty * L::kWeights;
    const float* pv = v + 2 * L::kPairs * tx;
#pragma unroll 2
    for (int j = 0; j < B; j += 4) {
        float4 x[L::kA];
#pragma unroll
        for (int r = 0; r < L::kA; ++r) {
            x[r] = *reinterpret_cast<const float4*>(pw + L::kRows * r * L::kWeights + j);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            F2 z[L::kA];
#pragma unroll
            for (int r = 0; r < L::kA; ++r) {
                const float one = k == 0 ? x[r].x : k == 1 ? x[r].y : k == 2 ? x[r].z : x[r].w;
                z[r] = MakeF2(one, one);
            }
#pragma unroll
            for (int c = 0; c < L::kChunks; ++c) {
                F2 y[L::kPairs];
                const float* at = pv + (j + k) * L::kStride + 32 * c;
                if constexpr (L::kPairs == 2) {
                    ReadQuad(at, y);
                } else {
                    y[0].r = *reinterpret_cast<const unsigned long long*>(at);
                }
#pragma unroll
                for (int r = 0; r < L::kA; ++r) {
#pragma unroll
                    for (int e = 0; e < L::kPairs; ++e) {
                        o.v[r][c][e] = Fma2(z[r], y[e], o.v[r][c][e]);
                    }
                }
            }
        }
    }
}

// A thread's sums of its row r, times a factor; true: not all finite.
template <typename T, typename L>
__device__ __forceinline__ bool StoreSums(T* row, const Sums<L>& o, int r, float factor, int32_t dim, bool some = true)
{
    const int tx = threadIdx.x % L::kCols;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < L::kChunks; ++c) {
        float v[2 * L::kPairs];
#pragma unroll
        for (int e = 0; e < L::kPairs; ++e) {
            SplitF2(o.v[r][c][e], v[2 * e], v[2 * e + 1]);
        }
#pragma unroll
        for (int e = 0; e < 2 * L::kPairs; ++e) {
            const int32_t d = 2 * L::kPairs * tx + 32 * c + e;
            if (d < dim) {
                v[e] = some ? v[e] * factor : 0.0f; // a masked NaN times a weight of 0 is one
                row[d] = DType<T>::FromF(v[e]);
                bad = bad || !(fabsf(v[e]) <= 3.4e38f);
            }
        }
    }
    return bad;
}

// over the N threads of a row
template <int N>
__device__ __forceinline__ float RowMax(float v)
{
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}
template <int N>
__device__ __forceinline__ float RowSum(float v)
{
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// Steps over the keys of queries at [low, high], the sinks in front of the window and then the window, without a gap: a few sinks take
// places of the window's first step, not a step.
template <int ROWS>
struct Walk {
    int32_t sinkEnd = 0, jump = 0, steps = 0;
    __device__ __forceinline__ Walk(const AttnShape& s, int32_t low, int32_t high)
    {
        if (high >= 0) {
            low = low > 0 ? low : 0;
            const int32_t first = low >= s.window ? low - s.window + 1 : 0;
            sinkEnd = s.sinks < first ? s.sinks : first;
            jump = first - sinkEnd;
            steps = (sinkEnd + (high - first) + ROWS) / ROWS;
        }
    }
    // the key at a place of the walk
    __device__ __forceinline__ int32_t Key(int32_t at) const { return at < sinkEnd ? at : at + jump; }
    __device__ __forceinline__ bool Sees(const AttnShape& s, int32_t p, int32_t at) const
    {
        const int32_t j = Key(at);
        return j <= p && (j > p - s.window || j < s.sinks);
    }
};

struct TileArgs {
    AttnArgs a;
    int32_t tiles;
    bool vec; // rows can be read 4 values at a time
    // gradK and gradV, see there
    bool perHead;
    int32_t sinkTiles, chunks;
    float* partial;
};
// Tiles whose blocks leave sums: all with a block a query head, otherwise those with sinks.
__host__ __device__ __forceinline__ int32_t PartialTiles(bool perHead, int32_t tiles, int32_t sinkTiles) { return perHead ? tiles : sinkTiles; }
// Where a block's sums start: the tiles of a unit (a head or key head), each with its chunks behind it where it has sinks.
__device__ __forceinline__ int64_t PartialSlot(const TileArgs& m, int32_t unit, int32_t tile, int32_t slot, int32_t rows)
{
    const int64_t perUnit = PartialTiles(m.perHead, m.tiles, m.sinkTiles) + static_cast<int64_t>(m.sinkTiles) * m.chunks;
    const int64_t at = tile + static_cast<int64_t>(min(tile, m.sinkTiles)) * m.chunks + slot;
    return (unit * perUnit + at) * 2 * rows * m.a.s.dim;
}

// ---- forward ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int A, int B>
__global__ void __launch_bounds__(Tile<DP, A, B>::kThreads) AttnForwardTilesKernel(const __grid_constant__ TileArgs m)
{
    using L = Tile<DP, A, B>;
    constexpr int R = L::kA, C = L::kB;
    extern __shared__ float shared[];
    __shared__ uint32_t again[2];
    float *sq = shared, *sk = sq + L::kFloatsA, *sv = sk + L::kFloatsB, *sw = sv + L::kFloatsB;
    const AttnShape& s = m.a.s;
    const int32_t tile = blockIdx.x % m.tiles, bh = blockIdx.x / m.tiles;
    const int32_t b = bh / s.heads, h = bh % s.heads, u = h / m.a.group;
    const Lengths n = LengthsOf(s, b);
    const int32_t i0 = tile * A, iLast = min(i0 + A, n.q) - 1;
    const Walk<B> walk(s, n.shift + i0, iLast >= i0 ? n.shift + iLast : -1);
    const int tx = threadIdx.x % L::kCols, ty = threadIdx.x / L::kCols;
    if (threadIdx.x < 2) {
        again[threadIdx.x] = 0;
    }
    auto fetch = [&](float* to, const AttnTensor& x, int32_t step) {
        if (step < walk.steps) {
            LoadTile<T, DP, B, L::kThreads>(to, x, b, u, step * B, n.kv, s.dim, m.vec, walk.sinkEnd, walk.jump);
        }
        CpAsyncCommit();
    };
    LoadTile<T, DP, A, L::kThreads>(sq, m.a.q, b, h, i0, iLast + 1, s.dim, m.vec);
    fetch(sk, m.a.k, 0);
    fetch(sv, m.a.v, 0);
    Sums<L> o;
    float top[R], total[R];
    int32_t p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        top[r] = -INFINITY;
        total[r] = 0.0f;
        const int32_t i = i0 + ty + L::kRows * r;
        p[r] = i <= iLast ? n.shift + i : -1;
    }
    for (int32_t step = 0; step < walk.steps; ++step) {
        CpAsyncWait<1>(); // the keys; the values may still be on their way
        __syncthreads();
        float x[R][C];
        Inner<L>(sq, sk, s.dim, x);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float most = top[r];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                x[r][c] = walk.Sees(s, p[r], step * B + tx + L::kCols * c) ? x[r][c] * s.scale : -INFINITY;
                most = fmaxf(most, x[r][c]);
            }
            most = RowMax<L::kCols>(most);
            const float base = most == -INFINITY ? 0.0f : most;
            const float fade = expf(top[r] - base);
            top[r] = most;
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                x[r][c] = expf(x[r][c] - base);
                sum += x[r][c];
                sw[(ty + L::kRows * r) * L::kWeights + tx + L::kCols * c] = x[r][c];
            }
            total[r] = total[r] * fade + sum;
            const F2 fade2 = MakeF2(fade, fade);
#pragma unroll
            for (int c = 0; c < L::kChunks; ++c) {
#pragma unroll
                for (int e = 0; e < L::kPairs; ++e) {
                    o.v[r][c][e] = Mul2(o.v[r][c][e], fade2);
                }
            }
        }
        __syncthreads(); // the keys have been read, the weights written
        fetch(sk, m.a.k, step + 1);
        CpAsyncWait<1>();
        __syncthreads();
        Outer<L, B>(sw, sv, o);
        __syncthreads();
        fetch(sv, m.a.v, step + 1);
    }
    CpAsyncWait<0>(); // a block without a step has its first copies under way
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int32_t i = i0 + ty + L::kRows * r;
        const float sum = RowSum<L::kCols>(total[r]);
        const bool some = p[r] >= 0;
        const float inverse = some ? 1.0f / sum : 0.0f; // a sum of 0 gives a NaN, and the row is formed again
        bool bad = false;
        if (i < s.lq) {
            T* out = OutRowOf<T>(m.a.out, b, i, h);
            bad = StoreSums<T>(out, o, r, inverse, s.dim, some);
            if (tx == 0 && m.a.lse != nullptr) {
                m.a.lse[static_cast<int64_t>(bh) * s.lq + i] = some ? top[r] + logf(sum) : -INFINITY;
            }
        }
        if (bad || (some && !(sum > 0.0f))) {
            atomicOr(&again[(ty + L::kRows * r) >> 5], 1u << ((ty + L::kRows * r) & 31));
        }
    }
    __syncthreads();
    // rows that are not finite again, without the masked keys' part
    for (int r = threadIdx.x >> 5; r < A; r += L::kThreads / 32) {
        if ((again[r >> 5] >> (r & 31) & 1) != 0 && i0 + r < s.lq) {
            AttnForwardRow<T>(m.a, b, h, i0 + r);
        }
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, int A, int B>
__global__ void __launch_bounds__(Tile<DP, A, B>::kThreads) AttnGradQTilesKernel(const __grid_constant__ TileArgs m)
{
    using L = Tile<DP, A, B>;
    constexpr int R = L::kA, C = L::kB;
    extern __shared__ float shared[];
    __shared__ uint32_t again[2];
    float *sq = shared, *sg = sq + L::kFloatsA, *sk = sg + L::kFloatsA, *sv = sk + L::kFloatsB, *sw = sv + L::kFloatsB;
    const AttnShape& s = m.a.s;
    const int32_t tile = blockIdx.x % m.tiles, bh = blockIdx.x / m.tiles;
    const int32_t b = bh / s.heads, h = bh % s.heads, u = h / m.a.group;
    const Lengths n = LengthsOf(s, b);
    const int32_t i0 = tile * A, iLast = min(i0 + A, n.q) - 1;
    const Walk<B> walk(s, n.shift + i0, iLast >= i0 ? n.shift + iLast : -1);
    const int tx = threadIdx.x % L::kCols, ty = threadIdx.x / L::kCols;
    if (threadIdx.x < 2) {
        again[threadIdx.x] = 0;
    }
    LoadTile<T, DP, A, L::kThreads>(sq, m.a.q, b, h, i0, iLast + 1, s.dim, m.vec);
    LoadTile<T, DP, A, L::kThreads>(sg, m.a.gradOut, b, h, i0, iLast + 1, s.dim, m.vec);
    auto fetch = [&](float* to, const AttnTensor& x, int32_t step) {
        if (step < walk.steps) {
            LoadTile<T, DP, B, L::kThreads>(to, x, b, u, step * B, n.kv, s.dim, m.vec, walk.sinkEnd, walk.jump);
        }
        CpAsyncCommit();
    };
    fetch(sv, m.a.v, 0);
    fetch(sk, m.a.k, 0);
    Sums<L> o;
    float lse[R], delta[R];
    int32_t p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int32_t i = i0 + ty + L::kRows * r;
        p[r] = i <= iLast ? n.shift + i : -1;
        lse[r] = p[r] >= 0 ? m.a.lse[static_cast<int64_t>(bh) * s.lq + i] : 0.0f;
        delta[r] = p[r] >= 0 ? m.a.delta[static_cast<int64_t>(bh) * m.a.deltaStride + i] : 0.0f;
    }
    for (int32_t step = 0; step < walk.steps; ++step) {
        CpAsyncWait<1>();
        __syncthreads();
        float x[R][C], y[R][C];
        Inner<L>(sg, sv, s.dim, y);
        __syncthreads();
        fetch(sv, m.a.v, step + 1); // under the products with the keys
        CpAsyncWait<1>();
        __syncthreads();
        Inner<L>(sq, sk, s.dim, x);
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const bool live = walk.Sees(s, p[r], step * B + tx + L::kCols * c);
                sw[(ty + L::kRows * r) * L::kWeights + tx + L::kCols * c] =
                    live ? expf(x[r][c] * s.scale - lse[r]) * (y[r][c] - delta[r]) * s.scale : 0.0f;
            }
        }
        __syncthreads();
        Outer<L, B>(sw, sk, o);
        __syncthreads();
        fetch(sk, m.a.k, step + 1); // under the next products with the values
    }
    CpAsyncWait<0>();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int32_t i = i0 + ty + L::kRows * r;
        bool bad = false;
        if (i < s.lq) {
            T* out = OutRowOf<T>(m.a.gradQ, b, i, h);
            bad = StoreSums<T>(out, o, r, 1.0f, s.dim, p[r] >= 0);
        }
        if (bad) {
            atomicOr(&again[(ty + L::kRows * r) >> 5], 1u << ((ty + L::kRows * r) & 31));
        }
    }
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < A; r += L::kThreads / 32) {
        if ((again[r >> 5] >> (r & 31) & 1) != 0 && i0 + r < s.lq) {
            AttnGradQRow<T>(m.a, b, h, i0 + r);
        }
    }
}

// A block has a tile of keys and the query heads of its key head. Where those blocks are too few for the SMs (`perHead`), a block has one
// query head instead; and where sinks are seen by many more queries than a window's, these are shared out among `chunks` further blocks
// of their tile. The sums of such blocks go to `partial` in fp32 ([batch, heads or key heads, tiles, 1 + chunks of one with sinks,
// gradK and gradV, rows of the tile, dim]), and AttnGradKvSumKernel adds them up in order.
template <typename T, int DP, int A, int B>
__global__ void __launch_bounds__(Tile<DP, A, B>::kThreads) AttnGradKvTilesKernel(const __grid_constant__ TileArgs m)
{
    using L = Tile<DP, A, B>;
    constexpr int R = L::kA, C = L::kB;
    extern __shared__ float shared[];
    __shared__ uint32_t again[2];
    __shared__ float sLse[B], sDelta[B];
    float *sk = shared, *sv = sk + L::kFloatsA, *sq = sv + L::kFloatsA, *sg = sq + L::kFloatsB, *sw = sg + L::kFloatsB,
          *sd = sw + L::kWeightFloats;
    const AttnShape& s = m.a.s;
    const int32_t perUnit = m.tiles + m.sinkTiles * m.chunks;
    int32_t tile = blockIdx.x % perUnit, chunk = -1;
    const int32_t unit = blockIdx.x / perUnit, units = m.perHead ? s.heads : s.kvHeads;
    if (tile >= m.tiles) {
        chunk = (tile - m.tiles) % m.chunks;
        tile = (tile - m.tiles) / m.chunks;
    }
    const int32_t b = unit / units, u = m.perHead ? unit % units / m.a.group : unit % units;
    const int32_t hFirst = m.perHead ? unit % units : u * m.a.group, hEnd = m.perHead ? hFirst + 1 : hFirst + m.a.group;
    const bool far = m.chunks > 0 && tile < m.sinkTiles; // its far queries are others'
    const Lengths n = LengthsOf(s, b);
    const int32_t j0 = tile * A, jLast = min(j0 + A, n.kv) - 1, end = n.kv - 1;
    // positions of the queries that this block walks
    int32_t low = max(j0, max(n.shift, 0)), high = jLast < j0 ? -1 : j0 < s.sinks && !far ? end : min(end, jLast + s.window - 1);
    if (chunk >= 0) {
        low = max(low, jLast + s.window);
        const int32_t steps = end >= low ? (end - low + B) / B : 0, share = (steps + m.chunks - 1) / m.chunks;
        high = jLast < j0 ? -1 : static_cast<int32_t>(min(static_cast<int64_t>(end), low + static_cast<int64_t>(chunk + 1) * share * B - 1));
        low += chunk * share * B;
    }
    const int32_t stop = high; // queries behind it are another block's
    const int tx = threadIdx.x % L::kCols, ty = threadIdx.x / L::kCols;
    if (threadIdx.x < 2) {
        again[threadIdx.x] = 0;
    }
    LoadTile<T, DP, A, L::kThreads>(sk, m.a.k, b, u, j0, n.kv, s.dim, m.vec);
    LoadTile<T, DP, A, L::kThreads>(sv, m.a.v, b, u, j0, n.kv, s.dim, m.vec);
    Sums<L> ok, ov;
    // steps over the heads and their queries
    const int32_t perHead = high >= low ? (high - low + B) / B : 0, steps = perHead * (hEnd - hFirst);
    auto fetch = [&](float* to, const AttnTensor& x, int32_t step) {
        if (step < steps) {
            LoadTile<T, DP, B, L::kThreads>(to, x, b, hFirst + step / perHead, low + step % perHead * B - n.shift, n.q, s.dim, m.vec);
        }
        CpAsyncCommit();
    };
    fetch(sg, m.a.gradOut, 0);
    fetch(sq, m.a.q, 0);
    for (int32_t step = 0; step < steps; ++step) {
        const int64_t head = static_cast<int64_t>(b) * s.heads + hFirst + step / perHead;
        const int32_t p0 = low + step % perHead * B, i0 = p0 - n.shift;
        if (threadIdx.x < B) {
            const int32_t i = i0 + threadIdx.x;
            sLse[threadIdx.x] = i < n.q ? m.a.lse[head * s.lq + i] : 0.0f;
            sDelta[threadIdx.x] = i < n.q ? m.a.delta[head * m.a.deltaStride + i] : 0.0f;
        }
        CpAsyncWait<1>();
        __syncthreads();
        float x[R][C], y[R][C];
        Inner<L>(sv, sg, s.dim, y);
        CpAsyncWait<0>();
        __syncthreads();
        Inner<L>(sk, sq, s.dim, x);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int32_t j = j0 + ty + L::kRows * r;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int32_t e = tx + L::kCols * c, p = p0 + e;
                const bool live = j < n.kv && p <= stop && j <= p && (j > p - s.window || j < s.sinks);
                const float w = live ? expf(x[r][c] * s.scale - sLse[e]) : 0.0f;
                sw[(ty + L::kRows * r) * L::kWeights + e] = w;
                sd[(ty + L::kRows * r) * L::kWeights + e] = live ? w * (y[r][c] - sDelta[e]) * s.scale : 0.0f;
            }
        }
        __syncthreads();
        Outer<L, B>(sw, sg, ov);
        __syncthreads();
        fetch(sg, m.a.gradOut, step + 1); // under the other outer products
        Outer<L, B>(sd, sq, ok);
        __syncthreads();
        fetch(sq, m.a.q, step + 1); // under the next products with the values
    }
    CpAsyncWait<0>();
    if (tile < PartialTiles(m.perHead, m.tiles, m.sinkTiles)) {
        float* part = m.partial + PartialSlot(m, unit, tile, 1 + chunk, A);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int32_t at = (ty + L::kRows * r) * s.dim;
            StoreSums<float>(part + at, ok, r, 1.0f, s.dim);
            StoreSums<float>(part + A * s.dim + at, ov, r, 1.0f, s.dim);
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int32_t j = j0 + ty + L::kRows * r;
        bool bad = false;
        if (j < s.lk) {
            T *gk = OutRowOf<T>(m.a.gradK, b, j, u), *gv = OutRowOf<T>(m.a.gradV, b, j, u);
            bad = StoreSums<T>(gk, ok, r, 1.0f, s.dim);
            bad = StoreSums<T>(gv, ov, r, 1.0f, s.dim) || bad;
        }
        if (bad) {
            atomicOr(&again[(ty + L::kRows * r) >> 5], 1u << ((ty + L::kRows * r) & 31));
        }
    }
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < A; r += L::kThreads / 32) {
        if ((again[r >> 5] >> (r & 31) & 1) != 0 && j0 + r < s.lk) {
            AttnGradKvRow<T>(m.a, b, u, j0 + r);
        }
    }
}

// A warp per key of the tiles with sums.
template <typename T>
__global__ void __launch_bounds__(128) AttnGradKvSumKernel(const __grid_constant__ TileArgs m, int32_t rows)
{
    const AttnShape& s = m.a.s;
    const int lane = threadIdx.x & 31;
    const int64_t key = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5); // (batch, key head, key)
    const int32_t perUnit = m.perHead ? s.lk : min(s.lk, m.sinkTiles * rows);
    if (key >= static_cast<int64_t>(s.batch) * s.kvHeads * perUnit) {
        return;
    }
    const int32_t j = static_cast<int32_t>(key % perUnit), bu = static_cast<int32_t>(key / perUnit), b = bu / s.kvHeads, u = bu % s.kvHeads;
    const int32_t tile = j / rows, slots = tile < m.sinkTiles ? 1 + m.chunks : 1;
    const int32_t first = m.perHead ? b * s.heads + u * m.a.group : bu, units = m.perHead ? m.a.group : 1;
    bool bad = false;
    for (int which = 0; which < 2; ++which) {
        T* out = OutRowOf<T>(which == 0 ? m.a.gradK : m.a.gradV, b, j, u);
        for (int32_t d = lane; d < s.dim; d += 32) {
            float sum = 0.0f;
            const int64_t within = (which * rows + j % rows) * static_cast<int64_t>(s.dim) + d;
#pragma unroll 4
            for (int32_t x = 0; x < units * slots; ++x) { // by head, then by block
                sum += m.partial[PartialSlot(m, first + x / slots, tile, x % slots, rows) + within];
            }
            bad = bad || !(fabsf(sum) <= 3.4e38f);
            out[d] = DType<T>::FromF(sum);
        }
    }
    if (__any_sync(0xffffffffu, bad)) {
        __syncwarp();
        AttnGradKvRow<T>(m.a, b, u, j);
    }
}

bool ReadsByFour(Dt dt, const AttnTensor& t)
{
    return Aligned(t.p, 4 * DtSize(dt)) && t.b % 4 == 0 && t.l % 4 == 0 && t.h % 4 == 0;
}

// Rows of the tiles that blocks own: 64 (32 of more than 128 values), or 32 where that leaves SMs with one block: a block's loads and waits
// then hide behind another's products (2 x 777 tokens, 6 heads of 72: forward 94 us with 64 rows, 64 us with 32,
// both before copies ran ahead; 56 us since). The SMs are a constant here and in PlanKv because both phases of a call have to come to one plan.
int OwnRows(const AttnShape& s, int64_t units, int64_t tokens)
{
    return s.dim > 128 || units * CeilDiv(tokens, 64) < 2 * kNumSMsFallback ? 32 : 64;
}

template <typename T, int DP, int A, int B>
cudaError_t Forward(Dt dt, const AttnArgs& a, cudaStream_t stream)
{
    using L = Tile<DP, A, B>;
    const AttnShape& s = a.s;
    TileArgs m{};
    m.a = a;
    m.tiles = static_cast<int32_t>(CeilDiv(s.lq, A));
    m.vec = s.dim % 4 == 0 && ReadsByFour(dt, a.q) && ReadsByFour(dt, a.k) && ReadsByFour(dt, a.v);
    constexpr int shared = (L::kFloatsA + 2 * L::kFloatsB + L::kWeightFloats) * 4;
    static std::atomic<uint64_t> asked;
    const int64_t blocks = static_cast<int64_t>(s.batch) * s.heads * m.tiles;
    if (blocks > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    const cudaError_t e = AskOnce(AttnForwardTilesKernel<T, DP, A, B>, asked, shared);
    if (e != cudaSuccess) {
        return e;
    }
    AttnForwardTilesKernel<T, DP, A, B><<<static_cast<unsigned>(blocks), L::kThreads, shared, stream>>>(m);
    CountLaunch();
    return cudaGetLastError();
}

// The blocks of gradK and gradV (see the kernel), from the sizes alone: the workspace holds their sums.
struct KvPlan {
    int32_t rows = 64, tiles = 0, sinkTiles = 0, chunks = 0;
    bool perHead = false;
    int64_t units = 0;
    int64_t Blocks() const { return units * (tiles + static_cast<int64_t>(sinkTiles) * chunks); }
    int64_t Partials() const { return units * (PartialTiles(perHead, tiles, sinkTiles) + static_cast<int64_t>(sinkTiles) * chunks); }
};
KvPlan PlanKv(const AttnShape& s)
{
    KvPlan p;
    const int64_t group = s.heads / s.kvHeads;
    p.perHead = group > 1 && static_cast<int64_t>(s.batch) * s.kvHeads * CeilDiv(s.lk, 64) < 2 * kNumSMsFallback;
    p.units = static_cast<int64_t>(s.batch) * (p.perHead ? s.heads : s.kvHeads);
    p.rows = OwnRows(s, p.units, s.lk);
    p.tiles = static_cast<int32_t>(CeilDiv(s.lk, p.rows));
    const int64_t step = s.dim <= 128 ? 64 : 32;
    const int64_t near = CeilDiv(static_cast<int64_t>(s.window) + p.rows, step), far = CeilDiv(s.lq > s.window ? s.lq - s.window : 0, step);
    const int64_t sinks = s.sinks < s.lk ? s.sinks : s.lk;
    if (sinks > 0 && s.heads > 0 && 2 * far > near) {
        p.sinkTiles = static_cast<int32_t>(CeilDiv(sinks, p.rows));
        const int64_t chunks = CeilDiv(far, near > 1 ? near : 1);
        p.chunks = AttnFarChunks(p.units, p.sinkTiles, chunks);
        p.sinkTiles = p.chunks > 0 ? p.sinkTiles : 0;
    }
    return p;
}
uint64_t DeltaBytes(const AttnShape& s) { return (static_cast<uint64_t>(s.batch) * s.heads * s.lq * 4 + 255) & ~255ull; }

template <typename T, int DP, int A, int B>
cudaError_t GradQ(const TileArgs& args, cudaStream_t stream)
{
    using L = Tile<DP, A, B>;
    TileArgs m = args;
    const AttnShape& s = m.a.s;
    constexpr int shared = (2 * L::kFloatsA + 2 * L::kFloatsB + L::kWeightFloats) * 4;
    static std::atomic<uint64_t> asked;
    m.tiles = static_cast<int32_t>(CeilDiv(s.lq, A));
    const int64_t blocks = static_cast<int64_t>(s.batch) * s.heads * m.tiles;
    if (blocks > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    const cudaError_t e = AskOnce(AttnGradQTilesKernel<T, DP, A, B>, asked, shared);
    if (e != cudaSuccess || blocks == 0) {
        return e;
    }
    AttnGradQTilesKernel<T, DP, A, B><<<static_cast<unsigned>(blocks), L::kThreads, shared, stream>>>(m);
    CountLaunch();
    return cudaGetLastError();
}

template <typename T, int DP, int A, int B>
cudaError_t GradKv(const TileArgs& args, const KvPlan& plan, float* partial, cudaStream_t stream)
{
    using L = Tile<DP, A, B>;
    TileArgs m = args;
    const AttnShape& s = m.a.s;
    constexpr int shared = (2 * L::kFloatsA + 2 * L::kFloatsB + 2 * L::kWeightFloats) * 4;
    static std::atomic<uint64_t> asked;
    const int64_t blocks = plan.Blocks();
    const int64_t summed = plan.perHead ? s.lk : std::min<int64_t>(s.lk, static_cast<int64_t>(plan.sinkTiles) * A);
    const int64_t keys = static_cast<int64_t>(s.batch) * s.kvHeads * summed; // whose gradients are put together from blocks' sums
    if (blocks > INT32_MAX || CeilDiv(keys, 4) > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    cudaError_t e = AskOnce(AttnGradKvTilesKernel<T, DP, A, B>, asked, shared);
    if (e != cudaSuccess) {
        return e;
    }
    m.tiles = plan.tiles;
    m.perHead = plan.perHead;
    m.sinkTiles = plan.sinkTiles;
    m.chunks = plan.chunks;
    m.partial = partial;
    if (blocks > 0) {
        AttnGradKvTilesKernel<T, DP, A, B><<<static_cast<unsigned>(blocks), L::kThreads, shared, stream>>>(m);
        CountLaunch();
    }
    if (keys > 0) {
        AttnGradKvSumKernel<T><<<static_cast<unsigned>(CeilDiv(keys, 4)), 128, 0, stream>>>(m, A);
        CountLaunch();
    }
    return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t Backward(Dt dt, const AttnArgs& a, void* workspace, cudaStream_t stream)
{
    const AttnShape& s = a.s;
    TileArgs m{};
    m.a = a;
    m.vec = s.dim % 4 == 0 && ReadsByFour(dt, a.q) && ReadsByFour(dt, a.k) && ReadsByFour(dt, a.v) && ReadsByFour(dt, a.gradOut);
    const KvPlan plan = PlanKv(s);
    float* partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + DeltaBytes(s));
    const bool few = OwnRows(s, static_cast<int64_t>(s.batch) * s.heads, s.lq) == 32;
    cudaError_t e;
    if constexpr (DP <= 128) {
        e = few ? GradQ<T, DP, 32, 64>(m, stream) : GradQ<T, DP, 64, 64>(m, stream);
        return e != cudaSuccess ? e :
               plan.rows == 32  ? GradKv<T, DP, 32, 64>(m, plan, partial, stream) :
                                  GradKv<T, DP, 64, 64>(m, plan, partial, stream);
    } else {
        e = GradQ<T, DP, 32, 32>(m, stream);
        return e != cudaSuccess ? e : GradKv<T, DP, 32, 32>(m, plan, partial, stream);
    }
}

template <typename T, int DP>
cudaError_t ForwardBySize(Dt dt, const AttnArgs& a, cudaStream_t stream)
{
    if constexpr (DP <= 128) {
        return OwnRows(a.s, static_cast<int64_t>(a.s.batch) * a.s.heads, a.s.lq) == 32 ? Forward<T, DP, 32, 64>(dt, a, stream) :
                                                                                       Forward<T, DP, 64, 64>(dt, a, stream);
    } else {
        return Forward<T, DP, 32, 32>(dt, a, stream);
    }
}

} // namespace

cudaError_t AttnForwardTiles(Dt dt, const AttnArgs& a, cudaStream_t stream)
{
    const int32_t d = a.s.dim;
    OPSCV_DISPATCH_DT(dt, T, {
        return d <= 64 ? ForwardBySize<T, 64>(dt, a, stream) :
               d <= 96 ? ForwardBySize<T, 96>(dt, a, stream) :
               d <= 128 ? ForwardBySize<T, 128>(dt, a, stream) :
                          ForwardBySize<T, 256>(dt, a, stream);
    });
    return cudaErrorInvalidValue;
}

uint64_t AttnBackwardTilesWorkspace(const AttnShape& s)
{
    const KvPlan p = PlanKv(s);
    return DeltaBytes(s) + static_cast<uint64_t>(p.Partials()) * 2 * p.rows * s.dim * 4;
}

cudaError_t AttnBackwardTiles(Dt dt, const AttnArgs& a, void* workspace, cudaStream_t stream)
{
    const int32_t d = a.s.dim;
    OPSCV_DISPATCH_DT(dt, T, {
        return d <= 64 ? Backward<T, 64>(dt, a, workspace, stream) :
               d <= 96 ? Backward<T, 96>(dt, a, workspace, stream) :
               d <= 128 ? Backward<T, 128>(dt, a, workspace, stream) :
                          Backward<T, 256>(dt, a, workspace, stream);
    });
    return cudaErrorInvalidValue;
}

} // namespace opscv
