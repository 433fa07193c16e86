// Attention over a sliding window with sinks on the tensor cores: 16-bit tensors with heads of up to 128 values.
#include "tcgen05.cuh"
#include "window_attention.cuh"

namespace opscv {

namespace {

__device__ unsigned int g_attentionTimeouts = 0;

constexpr int kTile = 128;                        // queries of a block, keys of a step
constexpr uint32_t kHalfBytes = kTile * 128;      // 64 of the up to 128 values of 128 rows
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// The running maximum stays as it is while the scores outgrow it by no more than a factor of 2^8: weights up to 2^8 lose nothing in
// a floating-point type, and most tiles then need no rescaling of the accumulators.
constexpr float kGrowth = 8.0f;

struct MmaArgs {
    AttnArgs a;
    int32_t tiles;  // of queries, per head
    int32_t halves; // of the heads' values: 1 or 2
    bool vecOut;    // rows of out can be written 16 bytes at a time
};

// The steps over keys of a block whose queries sit at [low, high]: first the sinks in front of the window, in steps from key 0,
// then the window, in steps from its first key (TMA boxes may start anywhere along the tokens).
struct KeySteps {
    int32_t sinkEnd, first, sinkSteps, steps;
};
__device__ __forceinline__ KeySteps StepsOf(const AttnShape& s, int32_t low, int32_t high)
{
    KeySteps r{0, 0, 0, 0};
    if (high >= 0) {
        low = low > 0 ? low : 0;
        r.first = low >= s.window ? low - s.window + 1 : 0;
        r.sinkEnd = s.sinks < r.first ? s.sinks : r.first;
        r.sinkSteps = (r.sinkEnd + kTile - 1) / kTile;
        r.steps = r.sinkSteps + (high - r.first + kTile) / kTile;
    }
    return r;
}
__device__ __forceinline__ int32_t StepKey(const KeySteps& r, int32_t n)
{
    return n < r.sinkSteps ? n * kTile : r.first + (n - r.sinkSteps) * kTile;
}

// Bits 0 to n - 1 of a word, n cut to [0, 32].
__device__ __forceinline__ uint32_t Below(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// ---- forward -----------------------------------------------------------------------------------------------------------------
// A block has 128 queries of a head. Warp 4's first thread loads the tiles and issues the products; warps 0 to 3 have a query a
// thread: S = Q K^T arrives in tensor memory, the thread forms the weights of its row, writes them over S as 16-bit values, and
// O += P V takes them from there, so that neither S nor P touches shared memory. Two blocks share an SM (256 columns of tensor memory
// and 97 KB each): while one forms its weights, the other's products run.
struct ForwardShared {
    uint64_t qFull, kFull, vFull, sFull, pFull, oFull;
    uint32_t tmem;
    uint32_t failed;
};

template <typename T, int HALVES>
__global__ void __launch_bounds__(160, 2)
    AttnForwardMmaKernel(const __grid_constant__ MmaArgs m, const __grid_constant__ CUtensorMap mapQ,
                         const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV)
{
    extern __shared__ unsigned char raw[];
    __shared__ ForwardShared sh;
    constexpr uint32_t kBytes = HALVES * kHalfBytes;
    unsigned char* base = raw + (1024 - (SharedAddr(raw) & 1023)) % 1024;
    unsigned char *sq = base, *sk = base + kBytes, *sv = base + 2 * kBytes;
    const AttnShape& s = m.a.s;
    const int32_t tile = blockIdx.x % m.tiles;
    const int32_t bh = blockIdx.x / m.tiles;
    const int32_t b = bh / s.heads, h = bh % s.heads;
    const Lengths n = LengthsOf(s, b);
    const int32_t i0 = tile * kTile;
    const int32_t iLast = min(i0 + kTile, n.q) - 1; // of the queries that count
    const int32_t low = n.shift + i0, high = iLast >= i0 ? n.shift + iLast : -1;
    const KeySteps steps = StepsOf(s, low, high);
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        sh.failed = 0;
        BarInit(&sh.qFull, 1);
        BarInit(&sh.kFull, 1);
        BarInit(&sh.vFull, 1);
        BarInit(&sh.sFull, 1);
        BarInit(&sh.pFull, 128);
        BarInit(&sh.oFull, 1);
        BarInitDone();
    }
    if (warp == 4) {
        TmemAlloc(&sh.tmem, 256);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmem = sh.tmem;
    const uint32_t tS = tmem, tO = tmem + 128;
    volatile uint32_t* failed = &sh.failed;

    if (warp == 4) {
        if ((threadIdx.x & 31) == 0 && steps.steps > 0) {
            const int32_t u = h / m.a.group;
            auto load = [&](unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int32_t row, int32_t head) {
                BarExpect(bar, kBytes);
#pragma unroll
                for (int c = 0; c < HALVES; ++c) {
                    TmaLoad4(dst + c * kHalfBytes, map, bar, 64 * c, row, head, b);
                }
            };
            load(sq, &mapQ, &sh.qFull, i0, h);
            load(sk, &mapK, &sh.kFull, StepKey(steps, 0), u);
            load(sv, &mapV, &sh.vFull, StepKey(steps, 0), u);
            const int32_t kSteps = (s.dim + 15) / 16;
            const uint32_t descS = ProductDesc<T>(kTile, false, s.scale < 0.0f);
            const uint32_t descO = ProductDesc<T>(kSteps * 16, true, false);
            const uint32_t aq = SharedAddr(sq), ak = SharedAddr(sk), av = SharedAddr(sv);
            BarWait(&sh.qFull, 0, failed);
            for (int32_t it = 0; it < steps.steps; ++it) {
                const uint32_t phase = it & 1;
                BarWait(&sh.kFull, phase, failed);
                TcFenceAfter();
                for (int32_t k = 0; k < kSteps; ++k) {
                    const uint32_t off = (k >> 2) * kHalfBytes + (k & 3) * 32;
                    MmaShared(tS, OperandDesc(aq + off, 16), OperandDesc(ak + off, 16), descS, k > 0);
                }
                MmaCommit(&sh.sFull);
                BarWait(&sh.sFull, phase, failed);
                if (*failed != 0) {
                    BarDrain(&sh.qFull, 0);
                    BarDrain(&sh.kFull, phase);
                    BarDrain(&sh.vFull, phase);
                    break;
                }
                if (it + 1 < steps.steps) {
                    load(sk, &mapK, &sh.kFull, StepKey(steps, it + 1), u);
                }
                BarWait(&sh.vFull, phase, failed);
                BarWait(&sh.pFull, phase, failed);
                if (*failed != 0) {
                    BarDrain(&sh.vFull, phase);
                    if (it + 1 < steps.steps) {
                        BarDrain(&sh.kFull, phase ^ 1);
                    }
                    break;
                }
                TcFenceAfter();
#pragma unroll
                for (int32_t k = 0; k < kTile / 16; ++k) {
                    MmaTmem(tO, tS + 8 * k, OperandDesc(av + k * 2048, kHalfBytes), descO, it > 0 || k > 0);
                }
                MmaCommit(&sh.oFull);
                BarWait(&sh.oFull, phase, failed);
                if (it + 1 < steps.steps) {
                    load(sv, &mapV, &sh.vFull, StepKey(steps, it + 1), u);
                }
            }
        }
        __syncwarp();
    } else {
        const int32_t i = i0 + threadIdx.x;
        const int32_t p = i <= iLast ? n.shift + i : -1;
        const Seen seen = SeenOf(s, p);
        const uint32_t lanes = static_cast<uint32_t>(warp) << 21; // 32 warp, in the lane half of an address
        const float factor = fabsf(s.scale) * kLog2e;             // scores in powers of two
        const int32_t wLow = low + 32 * warp, wHigh = wLow + 31;
        float top = -INFINITY, total = 0.0f;
        for (int32_t it = 0; it < steps.steps; ++it) {
            const int32_t j0 = StepKey(steps, it);
            BarWait(&sh.sFull, it & 1, failed);
            if (__any_sync(0xffffffffu, *failed != 0)) {
                break;
            }
            TcFenceAfter();
            uint32_t x[kTile];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                TmemLoad32(tS + lanes + 32 * c, x + 32 * c);
            }
            TmemLoadWait();
            const bool whole = it >= steps.sinkSteps && j0 + kTile - 1 <= wLow && j0 > wHigh - s.window && i0 + 32 * warp + 31 <= iLast;
            if (!whole) {
                // visible columns of the step: those of the window, or those of the sinks. A window step may hold sinks as well:
                // those behind the block's first key, in front of the row's window.
                const bool sinkStep = it < steps.sinkSteps;
                const int32_t from = sinkStep ? 0 : seen.first - j0;
                const int32_t to = p < 0 ? 0 : sinkStep ? steps.sinkEnd - j0 : p - j0 + 1;
                const int32_t sinkTo = sinkStep ? 0 : seen.sinkEnd - j0;
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {
                    const uint32_t live = (Below(to - c) & ~Below(from - c)) | Below(sinkTo - c);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        x[c + e] = (live >> e & 1) != 0 ? x[c + e] : 0xff800000u;
                    }
                }
            }
            float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < kTile; c += 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    part[e] = fmaxf(fmaxf(part[e], __uint_as_float(x[c + 2 * e])), __uint_as_float(x[c + 2 * e + 1]));
                }
            }
            const float most = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * factor;
            const float grown = fmaxf(top, most);
            const bool grow = grown > top + kGrowth; // always from -infinity to a number
            if (it == 0) {
                top = grown;
            } else if (__any_sync(0xffffffffu, grow)) {
                const float fade = grow ? Exp2(top - grown) : 1.0f;
                top = grow ? grown : top;
                total *= fade;
#pragma unroll 1
                for (int c = 0; c < 8 * HALVES; ++c) {
                    uint32_t o[8];
                    TmemLoad8(tO + lanes + 8 * c, o);
                    TmemLoadWait();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * fade);
                    }
                    TmemStore8(tO + lanes + 8 * c, o);
                }
            }
            const float off = top == -INFINITY ? 0.0f : -top;
            const F2 factor2 = MakeF2(factor, factor), off2 = MakeF2(off, off);
            F2 sum2[2] = {MakeF2(0.0f, 0.0f), MakeF2(0.0f, 0.0f)};
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const F2 z = Fma2(MakeF2(__uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1])), factor2, off2);
                    float e0, e1;
                    SplitF2(z, e0, e1);
                    e0 = Exp2(e0);
                    e1 = Exp2(e1);
                    sum2[e & 1] = Add2(sum2[e & 1], MakeF2(e0, e1));
                    w[e] = PackPair(e0, e1, static_cast<const T*>(nullptr));
                }
                TmemStore16(tS + lanes + c / 2, w);
            }
            float a0, a1;
            SplitF2(Add2(sum2[0], sum2[1]), a0, a1);
            total += a0 + a1;
            TmemStoreWait();
            TcFenceBefore();
            BarArrive(&sh.pFull);
        }
        // ---- the rows of out
        if (steps.steps > 0) {
            BarWait(&sh.oFull, (steps.steps - 1) & 1, failed);
            TcFenceAfter();
        }
        const float inverse = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total; // NaN stays
        bool bad = seen.count > 0 && !(total > 0.0f && total <= 3.0e38f);
        T* out = i < s.lq ? OutRowOf<T>(m.a.out, b, i, h) : nullptr;
#pragma unroll
        for (int c = 0; c < 2 * HALVES; ++c) {
            uint32_t o[32];
            if (steps.steps > 0) {
                TmemLoad32(tO + lanes + 32 * c, o);
                TmemLoadWait();
            }
            if (32 * c < s.dim) {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float v = seen.count > 0 ? __uint_as_float(o[e]) * inverse : 0.0f;
                    bad = bad || (32 * c + e < s.dim && !(fabsf(v) <= 3.4e38f));
                    o[e] = __float_as_uint(v);
                }
                if (out != nullptr) {
                    if (m.vecOut) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (32 * c + e < s.dim) {
                                float v[8];
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    v[k] = __uint_as_float(o[e + k]);
                                }
                                StorePack<T, 8>(out + 32 * c + e, v);
                            }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (32 * c + e < s.dim) {
                                out[32 * c + e] = DType<T>::FromF(__uint_as_float(o[e]));
                            }
                        }
                    }
                }
            }
        }
        if (out != nullptr && m.a.lse != nullptr) {
            m.a.lse[(static_cast<int64_t>(b) * s.heads + h) * s.lq + i] = seen.count > 0 ? (top + log2f(total)) * kLn2 : -INFINITY;
        }
        // rows that are not finite again, without the masked keys' part
        uint32_t rows = __ballot_sync(0xffffffffu, bad && out != nullptr);
        __syncwarp();
        while (rows != 0) {
            const int r = __ffs(rows) - 1;
            rows &= rows - 1;
            AttnForwardRow<T>(m.a, b, h, i0 + 32 * warp + r);
        }
        __syncwarp();
        if (*failed != 0 && out != nullptr) {
            for (int32_t d = 0; d < s.dim; ++d) {
                out[d] = DType<T>::FromF(NAN);
            }
        }
    }
    TcFenceBefore();
    __syncthreads();
    if (warp == 4) {
        TcFenceAfter();
        TmemFree(tmem, 256);
    }
    if (threadIdx.x == 0 && sh.failed != 0) {
        atomicAdd(&g_attentionTimeouts, 1u);
    }
}

// ---- launches ------------------------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled Encoder()
{
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return static_cast<EncodeTiled>(nullptr);
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// Boxes of 64 values by 128 tokens of one head; what lies outside the tensor arrives as zeros.
cudaError_t MakeMap(CUtensorMap* map, Dt dt, const AttnTensor& t, int32_t dim, int32_t tokens, int32_t heads, int32_t batch)
{
    const EncodeTiled encode = Encoder();
    if (encode == nullptr) {
        return cudaErrorNotSupported;
    }
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(heads),
                                static_cast<cuuint64_t>(batch)};
    const cuuint64_t row = static_cast<cuuint64_t>(CeilDiv(dim, 8)) * 16;
    // the stride along a single token, head or sequence is of no account, but has to be a valid one
    const cuuint64_t strides[3] = {tokens > 1 ? static_cast<cuuint64_t>(t.l) * 2 : row, heads > 1 ? static_cast<cuuint64_t>(t.h) * 2 : row,
                                   batch > 1 ? static_cast<cuuint64_t>(t.b) * 2 : row};
    const cuuint32_t box[4] = {64, kTile, 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, dt == Dt::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void*>(t.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

bool TmaStride(int64_t stride, int32_t extent) { return extent <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); }

} // namespace

// A tensor that boxes can be loaded from: 16-byte aligned rows, heads and sequences, none of them at one address.
bool AttnTmaReadable(const AttnTensor& t, int32_t tokens, int32_t heads, int32_t batch)
{
    return Aligned(t.p, 16) && TmaStride(t.l, tokens) && TmaStride(t.h, heads) && TmaStride(t.b, batch);
}

cudaError_t AttnForwardMma(Dt dt, const AttnArgs& a, cudaStream_t stream)
{
    const AttnShape& s = a.s;
    MmaArgs m{};
    m.a = a;
    m.tiles = static_cast<int32_t>(CeilDiv(s.lq, kTile));
    m.halves = s.dim > 64 ? 2 : 1;
    m.vecOut = s.dim % 8 == 0 && Aligned(a.out.p, 16) && a.out.l % 8 == 0 && a.out.h % 8 == 0 && a.out.b % 8 == 0;
    CUtensorMap mq, mk, mv;
    cudaError_t e = MakeMap(&mq, dt, a.q, s.dim, s.lq, s.heads, s.batch);
    e = e != cudaSuccess ? e : MakeMap(&mk, dt, a.k, s.dim, s.lk, s.kvHeads, s.batch);
    e = e != cudaSuccess ? e : MakeMap(&mv, dt, a.v, s.dim, s.lk, s.kvHeads, s.batch);
    if (e != cudaSuccess) {
        return e;
    }
    const int shared = 3 * m.halves * static_cast<int>(kHalfBytes) + 1024;
    const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(s.batch) * s.heads * m.tiles);
    auto launch = [&](auto kernel) {
        const cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
        if (set != cudaSuccess) {
            return set;
        }
        kernel<<<grid, 160, shared, stream>>>(m, mq, mk, mv);
        CountLaunch();
        return cudaGetLastError();
    };
    if (dt == Dt::F16) {
        return m.halves == 1 ? launch(AttnForwardMmaKernel<__half, 1>) : launch(AttnForwardMmaKernel<__half, 2>);
    }
    return m.halves == 1 ? launch(AttnForwardMmaKernel<__nv_bfloat16, 1>) : launch(AttnForwardMmaKernel<__nv_bfloat16, 2>);
}

uint32_t AttentionTimeouts()
{
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_attentionTimeouts, sizeof(v)) == cudaSuccess ? v : 0xffffffffu;
}

} // namespace opscv
