// Attention of few queries (a decoding step, a short chunk or draft) over long keys.
//
// Bound by reading the visible keys and values once: with one query a sequence there are only heads / kvHeads rows to share a key, too
// few for the 128 of tcgen05. A block has rows of one key head and a share of the keys, and each warp keeps a softmax of its own keys
// (maximum, sum and weighted values in fp32 registers). These join in shared memory, then across the blocks of a cluster through
// distributed shared memory: one launch, no workspace, sums in a fixed order.
//
// 16-bit rows: up to 16 a block, on the 16 x 8 x 16 products of a warp. Each warp has a ring of its own in shared memory, which TMA fills
// 16 keys at a time, so that no warp waits for another and loading costs one thread a few instructions.
// 32 sequences, window 1024, 32 heads of 128 on 8: 30 us (4.5 TB/s: a warp has 16 steps, whose chain the few warps of an SM do not hide);
// 8 sequences of 16384 keys: 85 us (6.3 TB/s).
// fp32 rows (and 16-bit ones that are not aligned, or of more than 128 values): up to 4 a block in fp32 arithmetic, 8 lanes a key.
#include <algorithm>

#include <cooperative_groups.h>

#include "tcgen05.cuh"
#include "window_attention.cuh"

namespace opscv {

namespace {

constexpr int kWarps = 4; // of a block; twice that where blocks are few (AttnStep)
constexpr int kThreads = 32 * kWarps;

struct StepArgs {
    AttnArgs a;
    int32_t splits, rowGroups;
};

// the chunks of 8 * V values of a row that a lane of 8 has its V of
template <typename T, int V, int N, bool VEC>
__device__ __forceinline__ void LoadRow(const T* p, int32_t lane, int32_t dim, bool live, Pack<T, V> (&r)[N])
{
#pragma unroll
    for (int c = 0; c < N; ++c) {
        const int32_t d = (c * 8 + lane) * V;
        if constexpr (VEC) {
            if (live && d < dim) {
                const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p + d));
                r[c] = reinterpret_cast<const Pack<T, V>&>(raw);
            } else {
                const uint4 zero = make_uint4(0, 0, 0, 0);
                r[c] = reinterpret_cast<const Pack<T, V>&>(zero);
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                r[c].v[e] = live && d + e < dim ? p[d + e] : DType<T>::FromF(0.0f);
            }
        }
    }
}

// Maxima (of scores in powers of two) and sums of the block's rows: of its warps, and of all of them.
constexpr int kMostRows = 16;
template <int W>
struct RowParts {
    float warpTop[W][kMostRows], warpSum[W][kMostRows], blockTop[kMostRows], blockSum[kMostRows];
};

// The warps' parts of `count` rows (weighted values [W][count][dim] in `shared`, which has room for [count][dim] more) to the
// results, by all threads of all blocks of the cluster.
template <typename T, int W>
__device__ __forceinline__ void JoinRows(const StepArgs& m, int32_t b, int32_t u, int32_t r0, int32_t count, const Lengths& n,
                                         float* shared, RowParts<W>& part)
{
    const AttnShape& s = m.a.s;
    const int32_t rows = s.lq * m.a.group, split = blockIdx.x % m.splits;
    const int warp = threadIdx.x >> 5;
    __syncthreads();
    // the block's warps: a thread has every 32 W-th column of the rows
    float* block = shared + W * count * s.dim;
    for (int32_t e = threadIdx.x; e < count * s.dim; e += 32 * W) {
        const int32_t r = e / s.dim;
        float most = -INFINITY, sum = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            most = fmaxf(most, part.warpTop[w][r]);
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float fade = most == -INFINITY ? 1.0f : Exp2(part.warpTop[w][r] - most);
            sum = fmaf(part.warpSum[w][r], fade, sum);
            x = fmaf(shared[w * count * s.dim + e], fade, x);
        }
        block[e] = x;
        if (e - r * s.dim == 0) {
            part.blockTop[r] = most;
            part.blockSum[r] = sum;
        }
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (m.splits > 1) {
        cluster.sync();
    } else {
        __syncthreads();
    }
    // the cluster's blocks: a warp has a row, a lane the maximum and the sum of a block; then the blocks' values, their loads together
    for (int32_t r = split + m.splits * warp; r < count; r += m.splits * W) {
        const int32_t row = r0 + r;
        if (row < rows) {
            const int32_t i = row / m.a.group, h = u * m.a.group + row % m.a.group;
            const int l = threadIdx.x & 31;
            const bool has = l < m.splits;
            const float mine = has ? *cluster.map_shared_rank(&part.blockTop[r], l) : -INFINITY;
            float sum = has ? *cluster.map_shared_rank(&part.blockSum[r], l) : 0.0f;
            const float most = WarpMax(mine);
            const float fade = most == -INFINITY ? 1.0f : Exp2(mine - most);
            sum = WarpSum(sum * fade);
            float x[kLaneDims] = {};
#pragma unroll 8
            for (int32_t c = 0; c < m.splits; ++c) {
                const float f = __shfl_sync(0xffffffffu, fade, c);
                const float* other = cluster.map_shared_rank(block + r * s.dim, c);
#pragma unroll
                for (int e = 0; e < kLaneDims; ++e) {
                    if (l + 32 * e < s.dim) {
                        x[e] = fmaf(other[l + 32 * e], f, x[e]);
                    }
                }
            }
            T* out = OutRowOf<T>(m.a.out, b, i, h);
            const bool some = i < n.q && n.shift + i >= 0;
            bool bad = some && !(sum > 0.0f);
#pragma unroll
            for (int e = 0; e < kLaneDims; ++e) {
                if (l + 32 * e < s.dim) {
                    const float y = some ? x[e] / sum : 0.0f;
                    bad = bad || !(fabsf(y) <= 3.4e38f);
                    out[l + 32 * e] = DType<T>::FromF(y);
                }
            }
            if (l == 0 && m.a.lse != nullptr) {
                m.a.lse[(static_cast<int64_t>(b) * s.heads + h) * s.lq + i] = some ? (most + log2f(sum)) * 0.6931471805599453f : -INFINITY;
            }
            if (__any_sync(0xffffffffu, bad)) { // again without the masked keys' part
                __syncwarp();
                AttnForwardRow<T>(m.a, b, h, i);
            }
        }
    }
    if (m.splits > 1) {
        cluster.sync(); // nobody's shared memory goes while others read it
    }
}

// R rows a block, N chunks a lane, U keys of a lane group in flight
template <typename T, int R, int N, int U, bool VEC>
__global__ void __launch_bounds__(kThreads) AttnStepKernel(const __grid_constant__ StepArgs m)
{
    constexpr int V = 16 / sizeof(T);
    extern __shared__ float shared[]; // [kWarps][R][dim] weighted values, then [R][dim] of the block
    __shared__ RowParts<kWarps> part;
    const AttnShape& s = m.a.s;
    const int32_t split = blockIdx.x % m.splits;
    int32_t unit = blockIdx.x / m.splits;
    const int32_t rows = s.lq * m.a.group;
    const int32_t r0 = unit % m.rowGroups * R;
    unit /= m.rowGroups;
    const int32_t b = unit / s.kvHeads, u = unit % s.kvHeads;
    const Lengths n = LengthsOf(s, b);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 7, slot = threadIdx.x >> 3; // 16 lane groups
    const float factor = s.scale * 1.4426950408889634f;

    // rows of the block: (query, head of the group), each with the position of its query
    Seen seen[R];
    float q[R][N][V];
    int32_t low = INT32_MAX, high = -1;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int32_t row = r0 + r, i = row / m.a.group;
        const bool live = row < rows && i < n.q;
        const int32_t p = live ? n.shift + i : -1;
        seen[r] = SeenOf(s, p);
        if (p >= 0) {
            low = min(low, p);
            high = max(high, p);
        }
        Pack<T, V> raw[N];
        LoadRow<T, V, N, VEC>(live ? RowOf<T>(m.a.q, b, i, u * m.a.group + row % m.a.group) : static_cast<const T*>(nullptr), lane, s.dim,
                              live, raw);
#pragma unroll
        for (int c = 0; c < N; ++c) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                q[r][c][e] = DType<T>::ToF(raw[c].v[e]) * factor;
            }
        }
    }
    // keys that some row sees, the sinks first; this block's share of them
    Seen all{0, 0, 0};
    if (high >= 0) {
        all = SeenOf(s, low);
        all.count = all.sinkEnd + (high - all.first + 1);
    }
    const int32_t share = ((all.count + m.splits - 1) / m.splits + 15) / 16 * 16;
    const int32_t begin = min(all.count, split * share), end = min(all.count, begin + share);

    float acc[R][N][V], top[R], total[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        top[r] = -INFINITY;
        total[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                acc[r][c][e] = 0.0f;
            }
        }
    }
    const bool alike = s.lq == 1; // all rows see the same keys
    for (int32_t at = begin; at < end; at += 16 * U) {
        Pack<T, V> k[U][N], v[U][N];
        int32_t j[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const int32_t key = at + x * 16 + slot;
            j[x] = key < end ? SeenKey(all, key) : -1;
            LoadRow<T, V, N, VEC>(RowOf<T>(m.a.k, b, max(j[x], 0), u), lane, s.dim, j[x] >= 0, k[x]);
        }
#pragma unroll
        for (int x = 0; x < U; ++x) {
            LoadRow<T, V, N, VEC>(RowOf<T>(m.a.v, b, max(j[x], 0), u), lane, s.dim, j[x] >= 0, v[x]);
        }
        float score[R][U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                score[r][x] = 0.0f;
            }
#pragma unroll
            for (int c = 0; c < N; ++c) {
                float f[V];
                UnpackToF<T, V>(k[x][c], f);
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        score[r][x] = fmaf(q[r][c][e], f[e], score[r][x]);
                    }
                }
            }
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int x = 0; x < U; ++x) {
                    score[r][x] += __shfl_xor_sync(0xffffffffu, score[r][x], o);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float most = top[r];
#pragma unroll
            for (int x = 0; x < U; ++x) {
                const bool live = j[x] >= 0 && (alike || (j[x] < seen[r].first + seen[r].count - seen[r].sinkEnd &&
                                                          (j[x] >= seen[r].first || j[x] < seen[r].sinkEnd)));
                score[r][x] = live ? score[r][x] : -INFINITY;
                most = fmaxf(most, score[r][x]);
            }
            const float base = most == -INFINITY ? 0.0f : most;
            const float fade = Exp2(top[r] - base);
            top[r] = most;
            total[r] *= fade;
#pragma unroll
            for (int x = 0; x < U; ++x) {
                score[r][x] = Exp2(score[r][x] - base);
                total[r] += score[r][x];
            }
#pragma unroll
            for (int c = 0; c < N; ++c) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    acc[r][c][e] *= fade;
                }
            }
        }
#pragma unroll
        for (int x = 0; x < U; ++x) {
#pragma unroll
            for (int c = 0; c < N; ++c) {
                float f[V];
                UnpackToF<T, V>(v[x][c], f);
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        acc[r][c][e] = fmaf(score[r][x], f[e], acc[r][c][e]);
                    }
                }
            }
        }
    }
    // the warp's four lane groups
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float most = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 8));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
        const float fade = most == -INFINITY ? 1.0f : Exp2(top[r] - most);
        float sum = total[r] * fade;
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
#pragma unroll
        for (int c = 0; c < N; ++c) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float x = acc[r][c][e] * fade;
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int32_t d = (c * 8 + lane) * V + e;
                if ((threadIdx.x & 31) < 8 && d < s.dim) {
                    shared[(warp * R + r) * s.dim + d] = x;
                }
            }
        }
        if ((threadIdx.x & 31) == 0) {
            part.warpTop[warp][r] = most;
            part.warpSum[warp][r] = sum;
        }
    }
    JoinRows<T, kWarps>(m, b, u, r0, R, n, shared, part);
}

// ---- 16-bit rows on the warp's products ------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void WarpMma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (DType<T>::kIsHalf) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
template <bool TRANSPOSED>
__device__ __forceinline__ void LoadMatrices(uint32_t addr, uint32_t (&r)[4])
{
    if constexpr (TRANSPOSED) {
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr));
    } else {
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr));
    }
}

__device__ unsigned int g_stepTimeouts = 0;

constexpr int kStages = 2;
constexpr int kStepKeys = 16;
constexpr uint32_t kBox = kStepKeys * 128; // 64 values of 16 keys

// B64: blocks of 64 dims (1 or 2). In a lane, g = lane / 4 and c = lane % 4 stand for the row and the pair of columns that the products'
// layout gives it.
template <typename T, int B64, int W>
__global__ void __launch_bounds__(32 * W, W == kWarps ? 3 : 1)
    AttnStepMmaKernel(const __grid_constant__ StepArgs m, int32_t mostRows, const __grid_constant__ CUtensorMap mapK,
                      const __grid_constant__ CUtensorMap mapV)
{
    extern __shared__ __align__(1024) float shared[];
    __shared__ RowParts<W> part;
    __shared__ uint64_t full[W][kStages];
    __shared__ uint32_t failure;
    const AttnShape& s = m.a.s;
    const int32_t split = blockIdx.x % m.splits;
    int32_t unit = blockIdx.x / m.splits;
    const int32_t rows = s.lq * m.a.group;
    const int32_t r0 = unit % m.rowGroups * kMostRows;
    unit /= m.rowGroups;
    const int32_t b = unit / s.kvHeads, u = unit % s.kvHeads;
    const Lengths n = LengthsOf(s, b);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const float factor = s.scale * 1.4426950408889634f;

    const int32_t iLow = r0 / m.a.group, iHigh = min(n.q, (min(r0 + kMostRows, rows) - 1) / m.a.group + 1) - 1;
    const int32_t low = max(n.shift + iLow, 0), high = iHigh >= iLow ? n.shift + iHigh : -1;
    // steps over the keys that some row sees: the sinks in front of the window, then the window
    Seen all{0, 0, 0};
    int32_t sinkSteps = 0, steps = 0;
    if (high >= 0) {
        all = SeenOf(s, low);
        sinkSteps = (all.sinkEnd + kStepKeys - 1) / kStepKeys;
        steps = sinkSteps + (high - all.first + kStepKeys) / kStepKeys;
    }
    const uint32_t ringBase = (SharedAddr(shared) + 1023) & ~1023u;
    const uint32_t ring = ringBase + warp * kStages * 2 * B64 * kBox;
    if (lane == 0) {
        for (int x = 0; x < kStages; ++x) {
            BarInit(&full[warp][x], 1);
        }
        BarInitDone();
        if (warp == 0) {
            failure = 0;
        }
    }
    __syncthreads();
    volatile uint32_t* failed = &failure;
    auto keyOf = [&](int32_t step) { return step < sinkSteps ? step * kStepKeys : all.first + (step - sinkSteps) * kStepKeys; };
    auto fetch = [&](int32_t step, int stage) { // by one lane
        const int32_t j = keyOf(step);
        const uint32_t at = ring + stage * 2 * B64 * kBox;
        BarExpect(&full[warp][stage], 2 * B64 * kBox);
#pragma unroll
        for (int e = 0; e < B64; ++e) {
            TmaLoad4At(at + e * kBox, &mapK, &full[warp][stage], 64 * e, j, u, b);
            TmaLoad4At(at + (B64 + e) * kBox, &mapV, &full[warp][stage], 64 * e, j, u, b);
        }
    };
    const int32_t first = split * W + warp, stride = m.splits * W;
    if (lane == 0) {
        for (int x = 0; x < kStages; ++x) {
            if (first + x * stride < steps) {
                fetch(first + x * stride, x);
            }
        }
    }

    // rows g and g + 8 as the first operand: values 16 k + 2 c, + 1 and 16 k + 2 c + 8, + 9 of each
    uint32_t q[4 * B64][4];
    Seen seen[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int32_t row = r0 + g + 8 * x, i = row / m.a.group;
        const bool live = row < rows && i < n.q;
        seen[x] = SeenOf(s, live ? n.shift + i : -1);
        const T* p = live ? RowOf<T>(m.a.q, b, i, u * m.a.group + row % m.a.group) : static_cast<const T*>(nullptr);
#pragma unroll
        for (int k = 0; k < 4 * B64; ++k) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int32_t d = 16 * k + 8 * y + 2 * c;
                q[k][x + 2 * y] = live && d < s.dim ? __ldg(reinterpret_cast<const uint32_t*>(p + d)) : 0u;
            }
        }
    }

    float acc[8 * B64][4] = {};
    float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.0f, 0.0f};
    const bool alike = s.lq == 1;
    // Where a lane reads the matrices of a step. Keys: keys 0 to 7 and 8 to 15, values 16 k to + 7 and + 8 to + 15 (two 16-byte pieces of
    // the 128 bytes of a key, whose place in them TMA's swizzle xors with the key's number). Values: keys 0 to 7 and 8 to 15, dims 16 k
    // to + 7 and + 8 to + 15.
    const int32_t keyRow = (lane & 7) + ((lane >> 4) << 3), keyPiece = (lane >> 3) & 1;
    const int32_t valueRow = lane & 15, valuePiece = lane >> 4;
    const uint32_t keyAt = keyRow * 128 + ((keyPiece ^ (keyRow & 7)) << 4), valueAt = valueRow * 128 + ((valuePiece ^ (valueRow & 7)) << 4);
    int stage = 0;
    uint32_t phase = 0;
    for (int32_t step = first; step < steps; step += stride) {
        const uint32_t at = ring + stage * 2 * B64 * kBox;
        BarWait(&full[warp][stage], phase, failed);
        if (__any_sync(0xffffffffu, *failed != 0)) {
            break;
        }
        float sc[2][4] = {}; // of keys 0 to 7 and 8 to 15: [0], [1] of row g, [2], [3] of row g + 8
#pragma unroll
        for (int k = 0; k < 4 * B64; ++k) {
            uint32_t f[4];
            LoadMatrices<false>(at + (k >> 2) * kBox + (keyAt ^ ((k & 3) << 5)), f);
            WarpMma<T>(sc[0], q[k], f[0], f[1]);
            WarpMma<T>(sc[1], q[k], f[2], f[3]);
        }
        const int32_t j0 = keyOf(step);
        const int32_t behind = step < sinkSteps ? all.sinkEnd - j0 : high + 1 - j0; // keys of the step that some row sees
        const bool whole = behind >= kStepKeys;
        bool grow = false;
        float fade[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float most = -INFINITY;
            if (!alike || !whole) {
                // of the row's own keys: the first `to` and not those between the sinks and the window
                const int32_t to = min(behind, seen[r].first + seen[r].count - seen[r].sinkEnd - j0);
                const int32_t from = seen[r].first - j0, sinkTo = seen[r].sinkEnd - j0;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int32_t e = 2 * c + (x & 1) + 8 * (x >> 1);
                    float& z = sc[x >> 1][2 * r + (x & 1)];
                    z = e < to && (e >= from || e < sinkTo) ? z * factor : -INFINITY;
                }
            } else {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    sc[x >> 1][2 * r + (x & 1)] *= factor;
                }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                most = fmaxf(most, sc[x >> 1][2 * r + (x & 1)]);
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            grow = grow || most > top[r];
            most = fmaxf(most, top[r]);
            const float base = most == -INFINITY ? 0.0f : most;
            fade[r] = Exp2(top[r] - base);
            top[r] = most;
            total[r] *= fade[r];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float& z = sc[x >> 1][2 * r + (x & 1)];
                z = Exp2(z - base);
                total[r] += z;
            }
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int e = 0; e < 8 * B64; ++e) {
                acc[e][0] *= fade[0];
                acc[e][1] *= fade[0];
                acc[e][2] *= fade[1];
                acc[e][3] *= fade[1];
            }
        }
        // The weights in two 16-bit parts: their rounding to one would be the largest error of the result, and the products wait for
        // memory anyway.
        uint32_t p0[4], p1[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float z0 = sc[e >> 1][2 * (e & 1)], z1 = sc[e >> 1][2 * (e & 1) + 1];
            p0[e] = PackPair(z0, z1, static_cast<const T*>(nullptr));
            const Pack<T, 2> back = reinterpret_cast<const Pack<T, 2>&>(p0[e]);
            p1[e] = PackPair(z0 - DType<T>::ToF(back.v[0]), z1 - DType<T>::ToF(back.v[1]), static_cast<const T*>(nullptr));
        }
        // Keys behind the sequence are not read into the sums, whatever they hold: their values become zeros.
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (!whole) {
            keep0 = (2 * c < behind ? 0xffffu : 0u) | (2 * c + 1 < behind ? 0xffff0000u : 0u);
            keep1 = (2 * c + 8 < behind ? 0xffffu : 0u) | (2 * c + 9 < behind ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int k = 0; k < 4 * B64; ++k) {
            uint32_t f[4]; // dims 16 k to + 7: [0] keys 0 to 7, [1] keys 8 to 15; dims + 8 to + 15: [2], [3]
            LoadMatrices<true>(at + (B64 + (k >> 2)) * kBox + (valueAt ^ ((k & 3) << 5)), f);
            f[0] &= keep0;
            f[1] &= keep1;
            f[2] &= keep0;
            f[3] &= keep1;
            WarpMma<T>(acc[2 * k], p0, f[0], f[1]);
            WarpMma<T>(acc[2 * k + 1], p0, f[2], f[3]);
            WarpMma<T>(acc[2 * k], p1, f[0], f[1]);
            WarpMma<T>(acc[2 * k + 1], p1, f[2], f[3]);
        }
        __syncwarp(); // all lanes have read the step
        if (lane == 0 && step + kStages * stride < steps) {
            fetch(step + kStages * stride, stage);
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
        phase ^= stage == 0 ? 1u : 0u;
    }
    if (*failed != 0 && lane == 0) { // own copies end before the block does
        for (int x = 0; x < kStages; ++x) {
            BarDrain(&full[warp][x], 0);
            BarDrain(&full[warp][x], 1);
        }
    }
    __syncthreads(); // the rings become room for the rows
    if (threadIdx.x == 0 && *failed != 0) {
        atomicAdd(&g_stepTimeouts, 1u);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        total[r] += __shfl_xor_sync(0xffffffffu, total[r], 1);
        total[r] += __shfl_xor_sync(0xffffffffu, total[r], 2);
        const int32_t row = g + 8 * r;
        if (row < mostRows) {
#pragma unroll
            for (int e = 0; e < 8 * B64; ++e) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int32_t d = 8 * e + 2 * c + x;
                    if (d < s.dim) {
                        shared[(warp * mostRows + row) * s.dim + d] = acc[e][2 * r + x];
                    }
                }
            }
            if (c == 0) {
                part.warpTop[warp][row] = top[r];
                part.warpSum[warp][row] = *failed != 0 ? NAN : total[r]; // the row is formed again
            }
        }
    }
    JoinRows<T, W>(m, b, u, r0, mostRows, n, shared, part);
}

// Shared memory of any of these: the rows of 16 (of at most 128 values) or 4 (256), the rings.
constexpr size_t kRing = static_cast<size_t>(kStages) * 2 * kBox; // of a warp, per block of 64 dims
constexpr size_t MostShared(int warps) { return 2 * kRing * warps + 1024; }
static_assert((kWarps + 1) * 16 * 128 * 4 <= MostShared(kWarps) && (kWarps + 1) * 4 * 256 * 4 <= MostShared(kWarps) &&
                  (2 * kWarps + 1) * 16 * 128 * 4 <= MostShared(2 * kWarps),
              "rows fit");

template <typename Kernel, typename... More>
cudaError_t Launch(Kernel kernel, std::atomic<uint64_t>& asked, const StepArgs& m, int r, int warps, size_t ring, int64_t units,
                   cudaStream_t stream, const More&... more)
{
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(units * m.splits));
    config.blockDim = dim3(32 * warps);
    config.dynamicSmemBytes = std::max(static_cast<size_t>(warps + 1) * r * m.a.s.dim * 4, ring);
    config.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(m.splits);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    const cudaError_t ask = AskOnce(kernel, asked, static_cast<int>(MostShared(warps)), true);
    if (ask != cudaSuccess) {
        return ask;
    }
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, m, more...);
    CountLaunch();
    return e != cudaSuccess ? e : cudaGetLastError();
}

// rows, chunks a lane, keys in flight: what the registers of a thread hold
template <typename T>
cudaError_t LaunchFor(const StepArgs& m, int r, int n, bool vec, int64_t units, cudaStream_t stream)
{
#define OPSCV_STEP(R, N, U)                                                                                       \
    if (r == R && n == N) {                                                                                       \
        static std::atomic<uint64_t> asked[2];                                                                    \
        return vec ? Launch(AttnStepKernel<T, R, N, U, true>, asked[0], m, r, kWarps, 0, units, stream) :                 \
                     Launch(AttnStepKernel<T, R, N, U, false>, asked[1], m, r, kWarps, 0, units, stream);                 \
    }
    OPSCV_STEP(1, 1, 4)
    OPSCV_STEP(2, 1, 4)
    OPSCV_STEP(4, 1, 4)
    OPSCV_STEP(1, 2, 4)
    OPSCV_STEP(2, 2, 4)
    if constexpr (sizeof(T) == 2) {
        OPSCV_STEP(4, 2, 2)
        OPSCV_STEP(1, 4, 2)
        OPSCV_STEP(2, 4, 2)
    } else {
        OPSCV_STEP(4, 2, 4)
        OPSCV_STEP(1, 4, 2)
        OPSCV_STEP(2, 4, 2)
        OPSCV_STEP(4, 4, 2)
        OPSCV_STEP(1, 8, 1)
        OPSCV_STEP(2, 8, 1)
    }
#undef OPSCV_STEP
    return cudaErrorInvalidValue;
}

} // namespace

namespace {

// Rows a block, and which kernel: `products` of a warp, or fp32 arithmetic with n chunks a lane.
struct StepPlan {
    bool vec, products;
    int n, r;
    int64_t rowGroups;
};
StepPlan PlanStep(Dt dt, const AttnArgs& a)
{
    const AttnShape& s = a.s;
    StepPlan p;
    const int64_t rows = static_cast<int64_t>(s.lq) * a.group;
    const int v = dt == Dt::F32 ? 4 : 8;
    const int n = static_cast<int>(CeilDiv(s.dim, 8 * v)); // chunks a lane
    p.n = n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8;
    const int values = p.n * v; // a lane, of q and of the sums, for each row
    auto rowsApart = [&](const AttnTensor& x) { return Aligned(x.p, 16) && x.b % v == 0 && x.l % v == 0 && x.h % v == 0; };
    p.vec = s.dim % v == 0 && rowsApart(a.q) && rowsApart(a.k) && rowsApart(a.v);
    p.products = dt != Dt::F32 && s.dim % 2 == 0 && s.dim <= kMmaMostDim && rowsApart(a.q) &&
                 AttnTmaReadable(a.k, s.lk, s.kvHeads, s.batch) && AttnTmaReadable(a.v, s.lk, s.kvHeads, s.batch);
    const int most = p.products ? kMostRows : values > 16 ? 2 : 4;
    p.r = rows >= most ? most : static_cast<int>(p.products || rows < 3 ? rows : 4);
    p.rowGroups = CeilDiv(rows, p.r > 0 ? p.r : 1);
    return p;
}

} // namespace

// Up to 8 queries always. More where the blocks of the other kernels, which walk all keys of 32 to 128 queries, leave most of the SMs
// idle: as long as there are few groups of rows (each reads the keys again) and keys enough to share out. bf16, heads of 128, 32 on 8, one
// sequence of 32768 keys: 16 queries (32 groups) 94 us against 517, 64 (128 groups) 326 against 515, 128 (256 groups) 633 against 516;
// 8 sequences of 8192: 9 queries (192 groups) 172 against 152. fp32, 16 heads of 64, 4096 keys: 64 queries (256 groups) 136 us against 274,
// 128 queries (512 groups) 275 against 274; wider heads, whose tiles are slower: 32 of 128 on 8, 32768 keys, 64 queries (512 groups) 2768
// us against 3712; bf16, 8 heads of 256, 8192 keys, 128 queries (512 groups) 578 us against 2128.
bool AttnStepTakes(Dt dt, const AttnArgs& a)
{
    const AttnShape& s = a.s;
    if (s.lk == 0 || s.lq <= 8) {
        return s.lk > 0;
    }
    const int64_t keys = std::min<int64_t>(s.lk, static_cast<int64_t>(s.window) + s.sinks + s.lq);
    const StepPlan p = PlanStep(dt, a);
    return keys >= 1024 && p.rowGroups * s.batch * s.kvHeads <= (p.products ? 128 : s.dim > 64 ? 512 : 256);
}

cudaError_t AttnStep(Dt dt, const AttnArgs& a, cudaStream_t stream)
{
    const AttnShape& s = a.s;
    StepArgs m{};
    m.a = a;
    const StepPlan plan = PlanStep(dt, a);
    const bool vec = plan.vec, products = plan.products;
    const int n = plan.n, r = plan.r;
    m.rowGroups = static_cast<int32_t>(plan.rowGroups);
    const int64_t units = static_cast<int64_t>(s.batch) * s.kvHeads * m.rowGroups;
    // Blocks of a cluster share out the keys of a unit, up to about two blocks an SM (a block's start and end cost as much as some
    // hundred keys, so more are slower: 32 sequences of window 1024 with 8 key heads take 31 us as 256 blocks, 44 as 512 or 1024; 8 of
    // 16384 keys 272 us as 64 blocks, 85 as 256, 113 as 512), and down to the 64 keys of one step of each warp.
    const int64_t keys = static_cast<int64_t>(s.window) + s.sinks + s.lq < s.lk ? static_cast<int64_t>(s.window) + s.sinks + s.lq : s.lk;
    int splits = 1;
    while (splits < 16 && 2 * splits * units <= 2 * NumSMs() && keys >= 2 * splits * kStepKeys * kWarps) {
        splits *= 2;
    }
    m.splits = splits;
    if (units * splits > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    if (products) {
        CUtensorMap mk, mv;
        cudaError_t e = AttnMakeMap(&mk, dt, a.k, s.dim, s.lk, s.kvHeads, s.batch, kStepKeys);
        e = e != cudaSuccess ? e : AttnMakeMap(&mv, dt, a.v, s.dim, s.lk, s.kvHeads, s.batch, kStepKeys);
        if (e != cudaSuccess) {
            return e;
        }
        // Where the blocks take at most half of the SMs, they have twice the warps: the chain of a warp's steps, not memory, is their limit
        // (32768 keys, 16 heads of 128 on 4, 64 blocks: 26.5 us against 41.8; of 64 on 2, 65536 keys, 32 blocks: 30.8 against 47.2). With more
        // blocks, clusters of 16 such large ones wait for one another's SMs (8192 keys, 32 heads of 128 on 8, 128 blocks: 24.6 against 18.5).
        const bool more = 2 * units * splits <= NumSMs() && keys >= static_cast<int64_t>(splits) * kStepKeys * 8 * kWarps;
        const int warps = more ? 2 * kWarps : kWarps;
        const size_t ring = (s.dim > 64 ? 2 : 1) * kRing * warps + 1024;
        auto launch = [&](auto wide, auto narrow, auto wideMore, auto narrowMore, std::atomic<uint64_t>* asked) {
            return warps == kWarps ? (s.dim > 64 ? Launch(wide, asked[0], m, r, warps, ring, units, stream, r, mk, mv) :
                                                   Launch(narrow, asked[1], m, r, warps, ring, units, stream, r, mk, mv)) :
                                     (s.dim > 64 ? Launch(wideMore, asked[2], m, r, warps, ring, units, stream, r, mk, mv) :
                                                   Launch(narrowMore, asked[3], m, r, warps, ring, units, stream, r, mk, mv));
        };
        static std::atomic<uint64_t> asked[8];
        if (dt == Dt::F16) {
            return launch(AttnStepMmaKernel<__half, 2, kWarps>, AttnStepMmaKernel<__half, 1, kWarps>,
                          AttnStepMmaKernel<__half, 2, 2 * kWarps>, AttnStepMmaKernel<__half, 1, 2 * kWarps>, asked);
        }
        return launch(AttnStepMmaKernel<__nv_bfloat16, 2, kWarps>, AttnStepMmaKernel<__nv_bfloat16, 1, kWarps>,
                      AttnStepMmaKernel<__nv_bfloat16, 2, 2 * kWarps>, AttnStepMmaKernel<__nv_bfloat16, 1, 2 * kWarps>, asked + 4);
    }
    switch (dt) {
        case Dt::F32: return LaunchFor<float>(m, r, n, vec, units, stream);
        case Dt::F16: return LaunchFor<__half>(m, r, n, vec, units, stream);
        default: return LaunchFor<__nv_bfloat16>(m, r, n, vec, units, stream);
    }
}

uint32_t AttnStepTimeouts()
{
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_stepTimeouts, sizeof(v)) == cudaSuccess ? v : 0;
}

} // namespace opscv
