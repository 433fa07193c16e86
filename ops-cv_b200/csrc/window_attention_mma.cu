// Attention over a sliding window with sinks on the tensor cores: 16-bit tensors with heads of up to 128 values.
#include <algorithm>

#include "tcgen05.cuh"
#include "window_attention.cuh"

namespace opscv {

namespace {

__device__ unsigned int g_attentionTimeouts = 0;

constexpr int kTile = 128;                        // rows of a tile
constexpr uint32_t kHalfBytes = kTile * 128;      // 64 of the up to 128 values of 128 rows
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Softmax in one pass with a running maximum and sum (M. Milakov, N. Gimelshein, "Online normalizer calculation for softmax", 2018). The
// maximum stays as it is while the scores outgrow it by no more than a factor of 2^8: any reference will do as long as the weights keep
// their bits, which weights up to 2^8 do in a floating-point type, and most tiles then need no rescaling of the accumulators.
constexpr float kGrowth = 8.0f;

struct MmaArgs {
    AttnArgs a;
    int32_t tiles;  // of queries, per head
    int32_t halves; // of the heads' values: 1 or 2
    bool vecOut;    // rows of out can be written 16 bytes at a time
};

// The steps of KEYS keys over those of a block whose queries sit at [low, high]: first the sinks in front of the window, in steps from
// key 0, then the window, in steps from its first key (TMA boxes may start anywhere along the tokens).
template <int KEYS>
struct KeySteps {
    int32_t sinkEnd = 0, first = 0, sinkSteps = 0, steps = 0;
    __device__ __forceinline__ KeySteps(const AttnShape& s, int32_t low, int32_t high)
    {
        if (high >= 0) {
            low = low > 0 ? low : 0;
            first = low >= s.window ? low - s.window + 1 : 0;
            sinkEnd = s.sinks < first ? s.sinks : first;
            sinkSteps = (sinkEnd + KEYS - 1) / KEYS;
            steps = sinkSteps + (high - first + KEYS) / KEYS;
        }
    }
    __device__ __forceinline__ int32_t Key(int32_t n) const { return n < sinkSteps ? n * KEYS : first + (n - sinkSteps) * KEYS; }
};

// Bits 0 to n - 1 of a word, n cut to [0, 32].
__device__ __forceinline__ uint32_t Below(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// of the threads that have the rows
template <int THREADS>
__device__ __forceinline__ void RowBarrier()
{
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// ---- what lies behind a sequence's lengths ---------------------------------------------------------------------------------
// Its weights are 0, but 0 times a NaN would send every row of the tile to the warps that form rows again (4 x 4096 tokens, window 1024: 24 ms
// in place of 0.13, backward 98 in place of 0.38). So a tile that reaches behind the end comes on a barrier of the loading thread's own
// (`tail`), which then copies zeros over the last rows, on the barrier that the products wait for. Other tiles, and the warps that
// multiply and form weights, have no part in it (zeros written by the product warp cost the backward 2 % where nothing is padded).
__device__ uint4 g_zeroRows[kTile * 128 / sizeof(uint4)];

// Bytes of rows [from, ROWS) of an operand of HALVES blocks of 64 values, and zeros for them on `bar`, which expects them.
template <int ROWS, int HALVES>
__device__ __forceinline__ uint32_t BytesFrom(int32_t from)
{
    return HALVES * (ROWS - max(from, 0)) * 128;
}
template <int ROWS, int HALVES>
__device__ __forceinline__ void ZerosFrom(unsigned char* operand, int32_t from, uint64_t* bar)
{
#pragma unroll
    for (int c = 0; c < HALVES; ++c) {
        BulkLoad(operand + (c * ROWS + max(from, 0)) * 128, g_zeroRows, BytesFrom<ROWS, 1>(from), bar);
    }
}

// A tile that reaches behind the end, at row `row` of a head, its rows from `from` on as zeros: on `tail` first, then on `bar`. false: a wait
// ran out. Apart from the loops that call it, which keep their registers (in line, the forward took 1 to 2 % longer where nothing is padded).
template <int ROWS, int HALVES>
__device__ __noinline__ bool LoadTail(unsigned char* dst, const CUtensorMap* map, int32_t row, int32_t head, int32_t b, int32_t from,
                                      uint64_t* tail, uint32_t phase, uint64_t* bar, volatile uint32_t* failed)
{
    BarExpect(tail, HALVES * ROWS * 128);
#pragma unroll
    for (int c = 0; c < HALVES; ++c) {
        TmaLoad4(dst + c * ROWS * 128, map, tail, 64 * c, row, head, b);
    }
    BarWait(tail, phase, failed);
    if (*failed != 0) {
        return false;
    }
    BarExpect(bar, BytesFrom<ROWS, HALVES>(from));
    ZerosFrom<ROWS, HALVES>(dst, from, bar);
    return true;
}

// columns of an accumulator times a factor a row
template <int N>
__device__ __forceinline__ void TmemScale(uint32_t addr, float f)
{
#pragma unroll 1
    for (int c = 0; c < N; c += 8) {
        uint32_t o[8];
        TmemLoad8(addr + c, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
        }
        TmemStore8(addr + c, o);
    }
    TmemStoreWait();
}

// N values of a row of an output, of which `left` exist
template <typename T, int N>
__device__ __forceinline__ void StoreRow(T* out, const float (&v)[N], int32_t left, bool vec)
{
    if (vec) {
#pragma unroll
        for (int e = 0; e < N; e += 8) {
            if (e < left) {
                float w[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    w[k] = v[e + k];
                }
                StorePack<T, 8>(out + e, w);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (e < left) {
                out[e] = DType<T>::FromF(v[e]);
            }
        }
    }
}

// -infinity where a column's bit is not set
template <int N>
__device__ __forceinline__ void MaskColumns(uint32_t* x, const uint32_t (&live)[N / 32])
{
#pragma unroll
    for (int e = 0; e < N; ++e) {
        x[e] = (live[e >> 5] >> (e & 31) & 1) != 0 ? x[e] : 0xff800000u;
    }
}
// the columns [from, to) and [0, sinkTo) of N
template <int N>
__device__ __forceinline__ void LiveColumns(uint32_t (&live)[N / 32], int32_t from, int32_t to, int32_t sinkTo)
{
#pragma unroll
    for (int w = 0; w < N / 32; ++w) {
        live[w] = (Below(to - 32 * w) & ~Below(from - 32 * w)) | Below(sinkTo - 32 * w);
    }
}

// ---- forward -----------------------------------------------------------------------------------------------------------------
// A block has 128 queries of a head and walks its keys 64 at a time. Warp 4's first thread loads the tiles, warp 5 issues the products;
// warps 0 to 3 have a thread a query, with all 64 scores of a step in its registers: S = Q K^T arrives in tensor memory, the thread forms
// the weights, writes them over S as 16-bit values, and O += P V takes them from there, so that neither S nor P touches shared memory and
// a row's maximum and sum need no exchange (two threads a row: 333 us at 8192 tokens without a window, one: 301). S has two places (O, at
// most 128 columns, and twice 64), so the next step's scores are there when the threads come to them. Two blocks share an SM (256 columns
// of tensor memory, 97 KB of shared memory and 192 threads each), one's exponentials under the other's products.
//
// Bound by the chain of a row's thread: scores from tensor memory, their maximum, 64 exponentials, weights back. The running maximum moves
// only where a row has outgrown it by 2^8 (at the start, mostly); O is rescaled then and not otherwise. The weights are rounded to the
// tensors' type, as the product takes both operands in one type: half a step each, as much as the rounding of the result itself; the sum
// that they are divided by is of the weights before that. A second 16-bit part, as for few queries, would double the product. 8192
// tokens, 16 heads of 128 on 4:
// 301 us (906 TFLOP/s) without a window; 106 us (window 1024, 4 sinks; with the tensor pipe and the special-function units 37 % busy).
constexpr int kRowThreads = 128;
constexpr int kKeys = 64;
constexpr uint32_t kKeyHalf = kKeys * 128;

struct ForwardShared {
    uint64_t qFull, kFull[2], vFull[2], tail, sFull[2], pFull[2], pvDone[2], allDone, drain;
    uint32_t tmem, failed;
};

// KS: steps of 16 values of a head.
template <typename T, int KS>
__global__ void __launch_bounds__(192, 2)
    AttnForwardMmaKernel(const __grid_constant__ MmaArgs m, const __grid_constant__ CUtensorMap mapQ,
                         const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV)
{
    extern __shared__ unsigned char raw[];
    __shared__ ForwardShared sh;
    constexpr int HALVES = KS > 4 ? 2 : 1;
    constexpr uint32_t kBytes = HALVES * kHalfBytes, kKeyBytes = HALVES * kKeyHalf;
    unsigned char* base = raw + (1024 - (SharedAddr(raw) & 1023)) % 1024;
    unsigned char *sq = base, *sk = base + kBytes, *sv = sk + 2 * kKeyBytes;
    const AttnShape& s = m.a.s;
    const int32_t tile = m.tiles - 1 - static_cast<int32_t>(blockIdx.x % m.tiles); // the tiles that see most keys first
    const int32_t bh = blockIdx.x / m.tiles;
    const int32_t b = bh / s.heads, h = bh % s.heads;
    const Lengths n = LengthsOf(s, b);
    const int32_t i0 = tile * kTile;
    const int32_t iLast = min(i0 + kTile, n.q) - 1; // of the queries that count
    const int32_t low = n.shift + i0, high = iLast >= i0 ? n.shift + iLast : -1;
    const KeySteps<kKeys> steps(s, low, high);
    const int32_t count = steps.steps;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        sh.failed = 0;
        BarInit(&sh.qFull, 1);
        for (int e = 0; e < 2; ++e) {
            BarInit(&sh.kFull[e], 1);
            BarInit(&sh.vFull[e], 1);
            BarInit(&sh.sFull[e], 1);
            BarInit(&sh.pFull[e], kRowThreads);
            BarInit(&sh.pvDone[e], 1);
        }
        BarInit(&sh.tail, 1);
        BarInit(&sh.allDone, 1);
        BarInit(&sh.drain, 1);
        BarInitDone();
    }
    if (warp == 5) {
        TmemAlloc(&sh.tmem, 256);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tO = sh.tmem, tS = tO + 128; // S of even steps at 0 and of odd ones at 64 from there
    volatile uint32_t* failed = &sh.failed;

    if (warp == 4) {
        if ((threadIdx.x & 31) == 0 && count > 0) {
            const int32_t u = h / m.a.group;
            BarExpect(&sh.qFull, kBytes);
#pragma unroll
            for (int c = 0; c < HALVES; ++c) {
                TmaLoad4(sq + c * kHalfBytes, &mapQ, &sh.qFull, 64 * c, i0, h, b);
            }
            auto load = [&](unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int32_t row) {
                BarExpect(bar, kKeyBytes);
#pragma unroll
                for (int c = 0; c < HALVES; ++c) {
                    TmaLoad4(dst + c * kKeyHalf, map, bar, 64 * c, row, u, b);
                }
            };
            const int32_t end = n.kv < s.lk ? n.kv : INT32_MAX; // tiles that reach behind it come with zeros there
            int32_t ks = 0, vs = 0, tails = 0;                  // loads so far
            for (int32_t it = 0; it < count; ++it) {
                const int32_t st = it & 1, j0 = steps.Key(it);
                if (it >= 2) {
                    BarWait(&sh.sFull[st], (it / 2 - 1) & 1, failed); // the scores that read the place before
                }
                if (*failed != 0) {
                    break;
                }
                load(sk + st * kKeyBytes, &mapK, &sh.kFull[st], j0);
                ++ks;
                if (it >= 2) {
                    BarWait(&sh.pvDone[st], (it / 2 - 1) & 1, failed);
                }
                if (*failed != 0) {
                    break;
                }
                if (j0 + kKeys > end) { // the scores of its keys are replaced as they are
                    if (!LoadTail<kKeys, HALVES>(sv + st * kKeyBytes, &mapV, j0, u, b, n.kv - j0, &sh.tail, tails++ & 1, &sh.vFull[st],
                                                 failed)) {
                        break;
                    }
                } else {
                    load(sv + st * kKeyBytes, &mapV, &sh.vFull[st], j0);
                }
                ++vs;
            }
            // own copies end before the block does, whatever became of the others
            BarDrain(&sh.qFull, 0);
            if (tails > 0) {
                BarDrain(&sh.tail, (tails - 1) & 1);
            }
            for (int32_t e = ks > 2 ? ks - 2 : 0; e < ks; ++e) {
                BarDrain(&sh.kFull[e & 1], (e / 2) & 1);
            }
            for (int32_t e = vs > 2 ? vs - 2 : 0; e < vs; ++e) {
                BarDrain(&sh.vFull[e & 1], (e / 2) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        if (count > 0) {
            const bool lead = ElectOne();
            const uint32_t descS = ProductDesc<T>(kKeys, false, s.scale < 0.0f);
            const uint32_t descO = ProductDesc<T>(KS * 16, true, false);
            const uint64_t dq = OperandDesc(SharedAddr(sq), 16), dk = OperandDesc(SharedAddr(sk), 16), dv = OperandDesc(SharedAddr(sv), kKeyHalf);
            // a descriptor's address is in units of 16 bytes
            auto scores = [&](int32_t st) {
                if (lead) {
                    const uint64_t k0 = dk + st * (kKeyBytes >> 4);
#pragma unroll
                    for (int32_t k = 0; k < KS; ++k) {
                        MmaShared(tS + st * kKeys, dq + ((k >> 2) * (kHalfBytes >> 4) + (k & 3) * 2),
                                  k0 + ((k >> 2) * (kKeyHalf >> 4) + (k & 3) * 2), descS, k > 0);
                    }
                    MmaCommit(&sh.sFull[st]);
                }
                __syncwarp();
            };
            BarWait(&sh.qFull, 0, failed);
            for (int32_t it = 0; it < 2 && it < count; ++it) {
                BarWait(&sh.kFull[it], 0, failed);
                TcFenceAfter();
                scores(it);
            }
            for (int32_t it = 0; it < count; ++it) {
                const int32_t st = it & 1;
                const uint32_t phase = (it / 2) & 1;
                BarWait(&sh.vFull[st], phase, failed);
                BarWait(&sh.pFull[st], phase, failed);
                if (__any_sync(0xffffffffu, *failed != 0)) {
                    break;
                }
                TcFenceAfter();
                if (lead) {
                    const uint64_t v0 = dv + st * (kKeyBytes >> 4);
#pragma unroll
                    for (int32_t k = 0; k < kKeys / 16; ++k) {
                        MmaTmem(tO, tS + st * kKeys + k * 8, v0 + k * (2048 >> 4), descO, it > 0 || k > 0);
                    }
                    MmaCommit(&sh.pvDone[st]);
                }
                __syncwarp();
                if (it + 2 < count) {
                    BarWait(&sh.kFull[st], phase ^ 1, failed);
                    BarWait(&sh.pvDone[st], phase, failed); // the weights, which the next scores go over, have been read
                    TcFenceAfter();
                    scores(st);
                }
            }
            if (lead) {
                MmaCommit(&sh.allDone);
            }
            __syncwarp();
            BarWait(&sh.allDone, 0, failed);
            if (*failed != 0) {
                if (lead) {
                    MmaCommit(&sh.drain);
                }
                __syncwarp();
                BarDrain(&sh.drain, 0);
            }
        }
        __syncwarp();
    } else {
        const int32_t quad = warp & 3, r = quad * 32 + (threadIdx.x & 31);
        const int32_t i = i0 + r;
        const int32_t p = i <= iLast ? n.shift + i : -1;
        const Seen seen = SeenOf(s, p);
        const uint32_t lanes = static_cast<uint32_t>(quad) << 21; // 32 quad, in the lane half of an address
        const uint32_t to32 = tO + lanes;
        const float factor = fabsf(s.scale) * kLog2e;             // scores in powers of two
        const int32_t wLow = low + 32 * quad, wHigh = wLow + 31;
        const bool rowsWhole = i0 + 32 * quad + 31 <= iLast;
        const F2 factor2 = MakeF2(factor, factor);
        float top = -INFINITY, total = 0.0f;
        for (int32_t it = 0; it < count; ++it) {
            const int32_t j0 = steps.Key(it);
            const uint32_t tx = tS + (it & 1) * kKeys + lanes;
            BarWait(&sh.sFull[it & 1], (it / 2) & 1, failed);
            if (__any_sync(0xffffffffu, *failed != 0)) {
                break;
            }
            TcFenceAfter();
            const bool sinkStep = it < steps.sinkSteps;
            const bool masked = sinkStep || !rowsWhole || j0 + kKeys - 1 > wLow || j0 <= wHigh - s.window;
            uint32_t x[64];
            auto read = [&] {
                TmemLoad64(tx, x);
                if (masked) {
                    // Visible columns of the step: those of the window, or those of the sinks. A window step may hold sinks as well:
                    // those behind the block's first key, in front of the row's window.
                    uint32_t live[2];
                    LiveColumns<64>(live, sinkStep ? 0 : seen.first - j0, p < 0 ? 0 : sinkStep ? steps.sinkEnd - j0 : p - j0 + 1,
                                    sinkStep ? 0 : seen.sinkEnd - j0);
                    MaskColumns<64>(x, live);
                }
            };
            uint32_t w[32];
            float sum = 0.0f;
            auto weigh = [&] {
                const float off = top == -INFINITY ? 0.0f : -top;
                const F2 off2 = MakeF2(off, off);
                F2 sum2[2] = {MakeF2(0.0f, 0.0f), MakeF2(0.0f, 0.0f)};
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    float e0, e1;
                    SplitF2(Fma2(MakeF2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), factor2, off2), e0, e1);
                    e0 = Exp2(e0);
                    e1 = Exp2(e1);
                    sum2[e & 1] = Add2(sum2[e & 1], MakeF2(e0, e1));
                    w[e] = PackPair(e0, e1, static_cast<const T*>(nullptr));
                }
                float a0, a1;
                SplitF2(Add2(sum2[0], sum2[1]), a0, a1);
                sum = a0 + a1;
            };
            read();
            float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 64; c += 8) {
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
                BarWait(&sh.pvDone[(it - 1) & 1], ((it - 1) / 2) & 1, failed);
                TcFenceAfter();
                TmemScale<64 * HALVES>(to32, fade);
            }
            weigh();
            total += sum;
            TmemStore32(tx, w);
            TmemStoreWait();
            TcFenceBefore();
            BarArrive(&sh.pFull[it & 1]);
        }
        // ---- the rows of out
        if (count > 0) {
            BarWait(&sh.allDone, 0, failed);
            TcFenceAfter();
        }
        const float inverse = total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total; // NaN stays
        bool bad = seen.count > 0 && !(total > 0.0f && total <= 3.0e38f);
        T* out = i < s.lq ? OutRowOf<T>(m.a.out, b, i, h) : nullptr;
#pragma unroll
        for (int c = 0; c < 2 * HALVES; ++c) {
            const int32_t d0 = 32 * c;
            uint32_t o[32];
            if (count > 0) {
                TmemLoad32(to32 + 32 * c, o);
            }
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                v[e] = seen.count > 0 ? __uint_as_float(o[e]) * inverse : 0.0f;
                bad = bad || (d0 + e < s.dim && !(fabsf(v[e]) <= 3.4e38f));
            }
            if (out != nullptr && d0 < s.dim) {
                StoreRow<T>(out + d0, v, s.dim - d0, m.vecOut);
            }
        }
        if (out != nullptr && m.a.lse != nullptr) {
            m.a.lse[(static_cast<int64_t>(b) * s.heads + h) * s.lq + i] = seen.count > 0 ? (top + log2f(total)) * kLn2 : -INFINITY;
        }
        const uint32_t rows = __ballot_sync(0xffffffffu, bad && out != nullptr);
        __syncwarp();
        // rows that are not finite again, without the masked keys' part
        uint32_t again = rows;
        while (again != 0) {
            const int e = __ffs(again) - 1;
            again &= again - 1;
            AttnForwardRow<T>(m.a, b, h, i0 + 32 * quad + e);
        }
        if (*failed != 0 && out != nullptr) {
            for (int32_t d = 0; d < s.dim; ++d) {
                out[d] = DType<T>::FromF(NAN);
            }
        }
    }
    TcFenceBefore();
    __syncthreads();
    if (warp == 5) {
        TcFenceAfter();
        TmemFree(sh.tmem, 256);
    }
    if (threadIdx.x == 0 && sh.failed != 0) {
        atomicAdd(&g_attentionTimeouts, 1u);
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------------
// Two kinds of blocks, each with the sums that it owns in tensor memory, so that no sum crosses blocks but for the sinks' (below) and all
// are formed in a fixed order: gradK and gradV by blocks of 128 keys that walk the queries that see them, gradQ by blocks of 128 queries
// that walk their keys. S and dP are formed twice for that (7 products where one kind would do 5 and add gradQ up in memory, in an order
// of chance). They go in one launch, the longer ones first, so that the others fill the SMs that the last of them leave. A block has an SM
// to itself: warps 0 to 15 have a row each four threads (32 columns each), warp 16 loads, warp 17 issues the products; with two threads
// a row, the chain of one thread's exponentials was longer than the products. 8192 tokens, 16 heads of 128 on 4: 858 us (801 TFLOP/s of
// the 5 products) without a window; 2 x 4096, window 1024, 4 sinks: 302 us, the tensor pipe 45 % busy. The weights are scaled by 2^8
// (folded into the statistics), which keeps small ones out of fp16's subnormal range. Weights and ds are rounded to the tensors' type for
// their products, half a step each; delta is formed from `out` as it is stored, the only form of it that the call has.
constexpr int kSides = 4;
constexpr int kColumns = kTile / kSides;
constexpr int kGradThreads = kTile * kSides;
constexpr int kLoadWarp = kGradThreads / 32, kProductWarp = kLoadWarp + 1;
constexpr float kWeightShift = 8.0f;
constexpr float kWeightScale = 0.00390625f; // 2^-8
struct BackwardArgs {
    AttnArgs a;
    int32_t qTiles, kTiles;
    uint32_t kvBlocks;
    float* lse2;  // [batch, heads, stride]: lse in powers of two less kWeightShift; +infinity where a query sees nothing, so that its
                  // weights are 0
    float* delta; // [batch, heads, stride], 0 there
    int64_t stride;
    int32_t sinkTiles, farChunks; // see GradKvBlock
    float* partial;
    bool vecQ, vecK, vecV;
};

// delta and lse2 of the rows of a head (blockIdx.y), a row by 16 lanes, kStatRows rows by each at a time.
constexpr int kStatRows = 4;
template <typename T>
__global__ void __launch_bounds__(256) AttnStatisticsKernel(const __grid_constant__ BackwardArgs m, bool vec)
{
    const AttnShape& s = m.a.s;
    const int32_t lane = threadIdx.x & 15, first = blockIdx.x * (16 * kStatRows) + (threadIdx.x >> 4);
    for (int32_t bh = blockIdx.y; bh < s.batch * s.heads; bh += gridDim.y) {
        const int32_t b = bh / s.heads, h = bh - b * s.heads;
        const Lengths n = LengthsOf(s, b);
        const T* g = RowOf<T>(m.a.gradOut, b, 0, h);
        const T* o = RowOf<T>(m.a.out, b, 0, h);
        const int64_t stats = bh * m.stride, rows = static_cast<int64_t>(bh) * s.lq;
        float sum[kStatRows], lse[kStatRows];
        Pack<T, 8> x[kStatRows], y[kStatRows];
        bool live[kStatRows];
#pragma unroll
        for (int r = 0; r < kStatRows; ++r) {
            const int32_t i = first + 16 * r;
            live[r] = i < n.q && n.shift + i >= 0;
            lse[r] = live[r] ? m.a.lse[rows + i] : INFINITY;
            sum[r] = 0.0f;
            if (vec && live[r] && lane * 8 < s.dim) {
                x[r] = *reinterpret_cast<const Pack<T, 8>*>(g + i * m.a.gradOut.l + lane * 8);
                y[r] = *reinterpret_cast<const Pack<T, 8>*>(o + i * m.a.out.l + lane * 8);
            }
        }
#pragma unroll
        for (int r = 0; r < kStatRows; ++r) {
            const int32_t i = first + 16 * r;
            if (vec && live[r] && lane * 8 < s.dim) {
                float u[8], v[8];
                UnpackToF<T, 8>(x[r], u);
                UnpackToF<T, 8>(y[r], v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sum[r] = fmaf(u[e], v[e], sum[r]);
                }
            } else if (!vec && live[r]) {
                for (int32_t d = lane; d < s.dim; d += 16) {
                    sum[r] = fmaf(DType<T>::ToF(g[i * m.a.gradOut.l + d]), DType<T>::ToF(o[i * m.a.out.l + d]), sum[r]);
                }
            }
#pragma unroll
            for (int e = 8; e > 0; e >>= 1) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], e);
            }
            if (lane == 0 && i < m.stride) {
                m.lse2[stats + i] = live[r] ? fmaf(lse[r], kLog2e, -kWeightShift) : INFINITY;
                m.delta[stats + i] = sum[r];
            }
        }
    }
}

// fp16 alone: the rows of ds are scaled to its range by powers of two that follow the exponent (as it is stored, 0 to 255) of the
// largest value so far. Returns the factor for what the accumulator holds already (1: as it is).
struct RowScale {
    float scale = 1.0f;
    int32_t e = 0;
    bool set = false;
    __device__ __forceinline__ float Follow(uint32_t exponent)
    {
        const int32_t x = static_cast<int32_t>(exponent) - 127;
        if (exponent == 0 || (set && x + e <= 13)) { // below 2^14 when scaled
            return 1.0f;
        }
        const float before = scale;
        const bool was = set;
        e = 8 - x; // the largest becomes 2^8 to 2^9
        e = e > 100 ? 100 : (e < -100 ? -100 : e);
        scale = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
        set = true;
        return was ? scale / before : 1.0f; // nothing but zeros before the first
    }
};
__device__ __forceinline__ uint32_t ExponentOf(float positive) { return __float_as_uint(positive) >> 23; }

// 128 x 128 products over KS steps of 16 values, both operands with the values along their 128 bytes, halves of 64 kHalfBytes apart
template <int KS>
__device__ __forceinline__ void InnerProducts(uint32_t d, uint64_t a, uint64_t b, uint32_t desc)
{
#pragma unroll
    for (int32_t k = 0; k < KS; ++k) {
        const uint64_t off = (k >> 2) * (kHalfBytes >> 4) + (k & 3) * 2;
        MmaShared(d, a + off, b + off, desc, k > 0);
    }
}
// the products of 128 weights a row (tensor memory: 32 in 16 columns at `a`, the next at a + 32, ...) with 128 rows of values
__device__ __forceinline__ void OuterProducts(uint32_t d, uint32_t a, uint64_t rows, uint32_t desc, bool add)
{
#pragma unroll
    for (int32_t k = 0; k < kTile / 16; ++k) {
        MmaTmem(d, a + (k >> 1) * kColumns + (k & 1) * 8, rows + k * (2048 >> 4), desc, add || k > 0);
    }
}

// 32 weights of a row, scaled, as 16-bit values
template <typename T>
__device__ __forceinline__ void StoreWeights(uint32_t addr, const uint32_t (&x)[kColumns], float scale)
{
    uint32_t w[kColumns / 2];
#pragma unroll
    for (int c = 0; c < kColumns / 2; ++c) {
        w[c] = PackPair(__uint_as_float(x[2 * c]) * scale, __uint_as_float(x[2 * c + 1]) * scale, static_cast<const T*>(nullptr));
    }
    TmemStore16(addr, w);
}
template <int N>
__device__ __forceinline__ void TmemLoadOwn(uint32_t addr, uint32_t* o)
{
    if constexpr (N == 32) {
        TmemLoad32(addr, o);
    } else {
        TmemLoad16(addr, o);
    }
}
// The exponent of the largest of a row's threads' values.
__device__ __forceinline__ uint32_t LargestOfRow(uint8_t (&most)[kSides][kTile], int32_t side, int32_t r, float mine, uint64_t* exchanged,
                                                 uint32_t phase, volatile uint32_t* failed)
{
    most[side][r] = static_cast<uint8_t>(ExponentOf(mine));
    BarArrive(exchanged);
    BarWait(exchanged, phase, failed);
    uint32_t e = 0;
#pragma unroll
    for (int x = 0; x < kSides; ++x) {
        e = max(e, static_cast<uint32_t>(most[x][r]));
    }
    return e;
}

struct GradQShared {
    uint64_t qFull, kFull[3], kEmpty[3], vFull[2], vEmpty[2], tail, sFull[2], dpFull, dsReady, dqDone, allDone, exchanged, drain;
    uint32_t tmem, failed, bad[4];
    uint8_t most[2][kSides][kTile]; // fp16: exponents of a row's largest ds, of even and odd steps, of its threads
};

// Tensor memory: S of even and odd steps at 0 and 128 (ds of a step goes over its S), dP at 256, gradQ at 384. The products of a step in
// the order dP(n + 1), gradQ(n), S(n + 2): the row threads form the weights of step n + 1 from an S that is there already while the
// first two run.
template <typename T, int KS>
__device__ __forceinline__ void GradQBlock(const BackwardArgs& m, const CUtensorMap& mapQ, const CUtensorMap& mapG, const CUtensorMap& mapK,
                                           const CUtensorMap& mapV, uint32_t block, unsigned char* raw, GradQShared& sh)
{
    constexpr int HALVES = KS > 4 ? 2 : 1;
    constexpr uint32_t kBytes = HALVES * kHalfBytes;
    unsigned char* base = raw + (1024 - (SharedAddr(raw) & 1023)) % 1024;
    unsigned char *sq = base, *sg = base + kBytes, *sk = base + 2 * kBytes, *sv = base + 5 * kBytes;
    const AttnShape& s = m.a.s;
    const int32_t tile = m.qTiles - 1 - static_cast<int32_t>(block % m.qTiles); // the tiles that see most keys first
    const int32_t bh = block / m.qTiles;
    const int32_t b = bh / s.heads, h = bh % s.heads;
    const Lengths n = LengthsOf(s, b);
    const int32_t i0 = tile * kTile;
    const int32_t iLast = min(i0 + kTile, n.q) - 1;
    const int32_t low = n.shift + i0, high = iLast >= i0 ? n.shift + iLast : -1;
    const KeySteps<kTile> steps(s, low, high);
    const int32_t count = steps.steps;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        sh.failed = 0;
        BarInit(&sh.qFull, 1);
        for (int e = 0; e < 3; ++e) {
            BarInit(&sh.kFull[e], 1);
            BarInit(&sh.kEmpty[e], 1);
        }
        for (int e = 0; e < 2; ++e) {
            BarInit(&sh.vFull[e], 1);
            BarInit(&sh.vEmpty[e], 1);
            BarInit(&sh.sFull[e], 1);
        }
        BarInit(&sh.tail, 1);
        BarInit(&sh.dpFull, 1);
        BarInit(&sh.dsReady, kGradThreads);
        BarInit(&sh.dqDone, 1);
        BarInit(&sh.allDone, 1);
        BarInit(&sh.exchanged, kGradThreads);
        BarInit(&sh.drain, 1);
        BarInitDone();
    }
    if (threadIdx.x < 4) {
        sh.bad[threadIdx.x] = 0;
    }
    if (warp == kProductWarp) {
        TmemAlloc(&sh.tmem, 512);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tS = sh.tmem, tDp = tS + 256, tDq = tS + 384;
    volatile uint32_t* failed = &sh.failed;

    if (warp == kLoadWarp) {
        if ((threadIdx.x & 31) == 0 && count > 0) {
            const int32_t u = h / m.a.group;
            auto load = [&](unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int32_t row, int32_t head) {
#pragma unroll
                for (int c = 0; c < HALVES; ++c) {
                    TmaLoad4(dst + c * kHalfBytes, map, bar, 64 * c, row, head, b);
                }
            };
            BarExpect(&sh.qFull, 2 * kBytes);
            load(sq, &mapQ, &sh.qFull, i0, h);
            load(sg, &mapG, &sh.qFull, i0, h);
            const int32_t end = n.kv < s.lk ? n.kv : INT32_MAX; // tiles that reach behind it come with zeros there
            int32_t it = 0, tails = 0;
            for (; it < count; ++it) {
                const int32_t j0 = steps.Key(it), ks = it % 3, vs = it & 1;
                if (it >= 3) {
                    BarWait(&sh.kEmpty[ks], (it / 3 - 1) & 1, failed);
                }
                if (it >= 2) {
                    BarWait(&sh.vEmpty[vs], (it / 2 - 1) & 1, failed);
                }
                if (*failed != 0) {
                    break;
                }
                if (j0 + kTile > end) { // of the products for dP and gradQ
                    const int32_t from = n.kv - j0;
                    if (!LoadTail<kTile, HALVES>(sk + ks * kBytes, &mapK, j0, u, b, from, &sh.tail, tails++ & 1, &sh.kFull[ks], failed)) {
                        break;
                    }
                    if (!LoadTail<kTile, HALVES>(sv + vs * kBytes, &mapV, j0, u, b, from, &sh.tail, tails++ & 1, &sh.vFull[vs], failed)) {
                        BarDrain(&sh.kFull[ks], (it / 3) & 1);
                        break;
                    }
                    continue;
                }
                BarExpect(&sh.kFull[ks], kBytes);
                load(sk + ks * kBytes, &mapK, &sh.kFull[ks], j0, u);
                BarExpect(&sh.vFull[vs], kBytes);
                load(sv + vs * kBytes, &mapV, &sh.vFull[vs], j0, u);
            }
            // own copies end before the block does, whatever became of the others
            BarDrain(&sh.qFull, 0);
            if (tails > 0) {
                BarDrain(&sh.tail, (tails - 1) & 1);
            }
            for (int32_t e = it > 3 ? it - 3 : 0; e < it; ++e) {
                BarDrain(&sh.kFull[e % 3], (e / 3) & 1);
            }
            for (int32_t e = it > 2 ? it - 2 : 0; e < it; ++e) {
                BarDrain(&sh.vFull[e & 1], (e / 2) & 1);
            }
        }
        __syncwarp();
    } else if (warp == kProductWarp) {
        if (count > 0) {
            const bool lead = ElectOne();
            const uint32_t descS = ProductDesc<T>(kTile, false, s.scale < 0.0f), descDp = ProductDesc<T>(kTile, false, false);
            const uint32_t descDq = ProductDesc<T>(KS * 16, true, false);
            const uint64_t dq = OperandDesc(SharedAddr(sq), 16), dg = OperandDesc(SharedAddr(sg), 16);
            const uint64_t dk = OperandDesc(SharedAddr(sk), 16), dkRows = OperandDesc(SharedAddr(sk), kHalfBytes),
                           dv = OperandDesc(SharedAddr(sv), 16);
            auto scores = [&](int32_t it, int32_t ks) { // ks: it modulo 3
                BarWait(&sh.kFull[ks], (it / 3) & 1, failed);
                TcFenceAfter();
                if (lead) {
                    InnerProducts<KS>(tS + (it & 1) * 128, dq, dk + ks * (kBytes >> 4), descS);
                    MmaCommit(&sh.sFull[it & 1]);
                }
                __syncwarp();
            };
            auto products = [&](int32_t it) {
                BarWait(&sh.vFull[it & 1], (it / 2) & 1, failed);
                TcFenceAfter();
                if (lead) {
                    InnerProducts<KS>(tDp, dg, dv + (it & 1) * (kBytes >> 4), descDp);
                    MmaCommit(&sh.dpFull);
                    MmaCommit(&sh.vEmpty[it & 1]);
                }
                __syncwarp();
            };
            BarWait(&sh.qFull, 0, failed);
            scores(0, 0);
            products(0);
            if (count > 1) {
                scores(1, 1);
            }
            int32_t ks = 0;
            for (int32_t it = 0; it < count; ++it) {
                BarWait(&sh.dsReady, it & 1, failed);
                if (__any_sync(0xffffffffu, *failed != 0)) {
                    break;
                }
                TcFenceAfter();
                if (it + 1 < count) {
                    products(it + 1);
                }
                if (lead) {
                    OuterProducts(tDq, tS + (it & 1) * 128, dkRows + ks * (kBytes >> 4), descDq, it > 0);
                    MmaCommit(&sh.kEmpty[ks]);
                    MmaCommit(&sh.dqDone);
                }
                __syncwarp();
                if (it + 2 < count) {
                    BarWait(&sh.dqDone, it & 1, failed); // ds(it), which the next scores go over, has been read
                    scores(it + 2, ks == 0 ? 2 : ks - 1);
                }
                ks = ks == 2 ? 0 : ks + 1;
            }
            if (lead) {
                MmaCommit(&sh.allDone);
            }
            __syncwarp();
            BarWait(&sh.allDone, 0, failed);
            if (*failed != 0) {
                if (lead) {
                    MmaCommit(&sh.drain);
                }
                __syncwarp();
                BarDrain(&sh.drain, 0);
            }
        }
        __syncwarp();
    } else {
        constexpr int kOwn = 64 * HALVES / kSides; // columns of the sums that a thread has
        const int32_t side = warp >> 2, r = (warp & 3) * 32 + (threadIdx.x & 31);
        const int32_t i = i0 + r;
        const int32_t p = i <= iLast ? n.shift + i : -1;
        const Seen seen = SeenOf(s, p);
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
        const float factor = fabsf(s.scale) * kLog2e;
        const int64_t row = static_cast<int64_t>(bh) * m.stride + i;
        const float lse2 = p >= 0 ? m.lse2[row] : INFINITY, delta = p >= 0 ? m.delta[row] : 0.0f;
        const F2 factor2 = MakeF2(factor, factor), off2 = MakeF2(-lse2, -lse2), delta2 = MakeF2(-delta, -delta);
        RowScale range;
        for (int32_t it = 0; it < count; ++it) {
            const int32_t j0 = steps.Key(it) + kColumns * side;
            const uint32_t tx = tS + (it & 1) * 128 + kColumns * side + lanes;
            BarWait(&sh.sFull[it & 1], (it >> 1) & 1, failed);
            if (__any_sync(0xffffffffu, *failed != 0)) {
                break;
            }
            TcFenceAfter();
            uint32_t x[kColumns];
            TmemLoad32(tx, x);
            {
                const bool sinkStep = it < steps.sinkSteps;
                const int32_t from = sinkStep ? 0 : seen.first - j0;
                const int32_t to = p < 0 ? 0 : sinkStep ? steps.sinkEnd - j0 : p - j0 + 1;
                const int32_t sinkTo = sinkStep ? 0 : seen.sinkEnd - j0;
                if (!__all_sync(0xffffffffu, from <= 0 && to >= kColumns)) {
                    uint32_t live[1];
                    LiveColumns<kColumns>(live, from, to, sinkTo);
                    MaskColumns<kColumns>(x, live);
                }
            }
#pragma unroll
            for (int e = 0; e < kColumns; e += 2) {
                float e0, e1;
                SplitF2(Fma2(MakeF2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), factor2, off2), e0, e1);
                x[e] = __float_as_uint(Exp2(e0));
                x[e + 1] = __float_as_uint(Exp2(e1));
            }
            BarWait(&sh.dpFull, it & 1, failed);
            TcFenceAfter();
            float most = 0.0f;
            {
                uint32_t y[kColumns];
                TmemLoad32(tDp + kColumns * side + lanes, y);
#pragma unroll
                for (int e = 0; e < kColumns; e += 2) {
                    const F2 d = Mul2(Add2(MakeF2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), delta2),
                                      MakeF2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
                    float d0, d1;
                    SplitF2(d, d0, d1);
                    x[e] = __float_as_uint(d0);
                    x[e + 1] = __float_as_uint(d1);
                    if constexpr (DType<T>::kIsHalf) {
                        most = fmaxf(most, fmaxf(fabsf(d0), fabsf(d1)));
                    }
                }
            }
            float scale = 1.0f;
            if constexpr (DType<T>::kIsHalf) {
                const float change = range.Follow(LargestOfRow(sh.most[it & 1], side, r, most, &sh.exchanged, it & 1, failed));
                scale = range.scale;
                if (it > 0 && __any_sync(0xffffffffu, change != 1.0f)) { // in all warps of the rows alike
                    BarWait(&sh.dqDone, (it - 1) & 1, failed);
                    TcFenceAfter();
                    TmemScale<kOwn>(tDq + lanes + kOwn * side, change);
                }
            }
            StoreWeights<T>(tx, x, scale);
            TmemStoreWait();
            TcFenceBefore();
            BarArrive(&sh.dsReady);
        }
        if (count > 0) {
            BarWait(&sh.allDone, 0, failed);
            TcFenceAfter();
        }
        T* out = i < s.lq ? OutRowOf<T>(m.a.gradQ, b, i, h) : nullptr;
        const float last = s.scale * kWeightScale / range.scale;
        bool bad = false;
        {
            const int32_t d0 = kOwn * side;
            uint32_t o[kOwn];
            if (count > 0) {
                TmemLoadOwn<kOwn>(tDq + lanes + d0, o);
            }
            float v[kOwn];
#pragma unroll
            for (int e = 0; e < kOwn; ++e) {
                v[e] = p >= 0 ? __uint_as_float(o[e]) * last : 0.0f;
                bad = bad || (d0 + e < s.dim && !(fabsf(v[e]) <= 3.4e38f));
            }
            if (out != nullptr && d0 < s.dim) {
                StoreRow<T>(out + d0, v, s.dim - d0, m.vecQ);
            }
        }
        const uint32_t rows = __ballot_sync(0xffffffffu, bad && out != nullptr);
        if ((threadIdx.x & 31) == 0 && rows != 0) {
            atomicOr(&sh.bad[warp & 3], rows);
        }
        RowBarrier<kGradThreads>();
        // rows that are not finite again, without the masked keys' part, shared out among the rows' warps
        uint32_t again = sh.bad[warp & 3] & (0x11111111u << side);
        while (again != 0) {
            const int e = __ffs(again) - 1;
            again &= again - 1;
            AttnGradQRow<T>(m.a, b, h, i0 + 32 * (warp & 3) + e);
        }
        if (*failed != 0 && out != nullptr && side == 0) {
            for (int32_t d = 0; d < s.dim; ++d) {
                out[d] = DType<T>::FromF(NAN);
            }
        }
    }
    TcFenceBefore();
    __syncthreads();
    if (warp == kProductWarp) {
        TcFenceAfter();
        TmemFree(sh.tmem, 512);
    }
    if (threadIdx.x == 0 && sh.failed != 0) {
        atomicAdd(&g_attentionTimeouts, 1u);
    }
}

struct GradKvShared {
    uint64_t kvFull, full[2], empty[2], tail, sFull, dpFull, pReady, dsReady, dvDone, dkDone, exchanged, drain;
    uint32_t tmem, failed, bad[4];
    uint8_t most[2][kSides][kTile]; // fp16: exponents of a row's largest ds, of even and odd steps, of its threads
};

// Tensor memory: S^T at 0 (the weights go over it), dP^T at 128 (ds goes over it), gradV at 256, gradK at 384; rows are keys, columns
// queries. The products of a step in the order gradV(n), S(n + 1), gradK(n), dP(n + 1): the exponentials of step n + 1 run under the last
// two, the rest of ds(n) under the first two.
//
// Sinks are seen by every later query. Were that left to the block of their keys, it would walk the whole sequence while the others
// walk a window; so the queries behind the window of such a tile are shared out among farChunks further blocks. Their sums and the
// tile's own go to `partial` ([tile][1 + farChunks][gradK, gradV][128][dim], fp32), which AttnSinkGradKernel adds up in order.
template <typename T, int KS>
__device__ __forceinline__ void GradKvBlock(const BackwardArgs& m, const CUtensorMap& mapQ, const CUtensorMap& mapG, const CUtensorMap& mapK,
                                            const CUtensorMap& mapV, uint32_t block, unsigned char* raw, GradKvShared& sh)
{
    constexpr int HALVES = KS > 4 ? 2 : 1;
    constexpr uint32_t kBytes = HALVES * kHalfBytes;
    constexpr uint32_t kStage = 2 * kBytes + 2 * kTile * 4;
    unsigned char* base = raw + (1024 - (SharedAddr(raw) & 1023)) % 1024;
    unsigned char *sk = base, *sv = base + kBytes, *sqg = base + 2 * kBytes;  // two stages of Q and gradOut
    float* stats = reinterpret_cast<float*>(base + 6 * kBytes);              // two stages of lse2 and delta
    const AttnShape& s = m.a.s;
    const int32_t perHead = m.kTiles + m.sinkTiles * m.farChunks;
    const int32_t bu = block / perHead;
    const int32_t b = bu / s.kvHeads, u = bu % s.kvHeads;
    int32_t tile = block % perHead, chunk = -1;
    if (tile >= m.kTiles) {
        chunk = (tile - m.kTiles) % m.farChunks;
        tile = (tile - m.kTiles) / m.farChunks;
    }
    const bool split = m.farChunks > 0 && tile < m.sinkTiles;
    const Lengths n = LengthsOf(s, b);
    const int32_t j0 = tile * kTile;
    const int32_t jLast = min(j0 + kTile, n.kv) - 1;
    const int32_t end = n.kv - 1; // position of the last query
    // positions [low, high] of the queries that this block walks
    int32_t low = max(j0, max(n.shift, 0)), high = min(end, jLast + s.window - 1);
    if (chunk >= 0) {
        low = max(low, jLast + s.window);
        high = end;
    } else if (j0 < s.sinks && !split) {
        high = end;
    }
    if (jLast < j0) {
        high = low - 1;
    }
    int32_t iBase = (low - n.shift) & ~3; // rows of the statistics are read 16 bytes at a time
    const int32_t perGroup = high >= low ? (high - n.shift - iBase + kTile) / kTile : 0;
    int32_t begin = 0, stop = perGroup * m.a.group;
    if (chunk >= 0) {
        const int32_t share = (stop + m.farChunks - 1) / m.farChunks;
        begin = min(stop, chunk * share);
        stop = min(stop, begin + share);
    }
    const int32_t count = stop - begin;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        sh.failed = 0;
        BarInit(&sh.kvFull, 1);
        for (int e = 0; e < 2; ++e) {
            BarInit(&sh.full[e], 1);
            BarInit(&sh.empty[e], 1);
        }
        BarInit(&sh.tail, 1);
        BarInit(&sh.sFull, 1);
        BarInit(&sh.dpFull, 1);
        BarInit(&sh.pReady, kGradThreads);
        BarInit(&sh.dsReady, kGradThreads);
        BarInit(&sh.dvDone, 1);
        BarInit(&sh.dkDone, 1);
        BarInit(&sh.exchanged, kGradThreads);
        BarInit(&sh.drain, 1);
        BarInitDone();
    }
    if (threadIdx.x < 4) {
        sh.bad[threadIdx.x] = 0;
    }
    if (warp == kProductWarp) {
        TmemAlloc(&sh.tmem, 512);
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tS = sh.tmem, tDp = tS + 128, tDv = tS + 256, tDk = tS + 384;
    volatile uint32_t* failed = &sh.failed;

    if (warp == kLoadWarp) {
        if ((threadIdx.x & 31) == 0 && count > 0) {
            auto load = [&](unsigned char* dst, const CUtensorMap* map, uint64_t* bar, int32_t row, int32_t head) {
#pragma unroll
                for (int c = 0; c < HALVES; ++c) {
                    TmaLoad4(dst + c * kHalfBytes, map, bar, 64 * c, row, head, b);
                }
            };
            BarExpect(&sh.kvFull, 2 * kBytes);
            load(sk, &mapK, &sh.kvFull, j0, u);
            load(sv, &mapV, &sh.kvFull, j0, u);
            const int32_t last = n.q < s.lq ? n.q : INT32_MAX; // tiles that reach behind it come with zeros there
            int32_t it = 0, tails = 0;
            for (; it < count; ++it) {
                const int32_t st = it & 1, h = u * m.a.group + (begin + it) / perGroup;
                const int32_t i0 = iBase + (begin + it) % perGroup * kTile;
                if (it >= 2) {
                    BarWait(&sh.empty[st], (it / 2 - 1) & 1, failed);
                }
                if (*failed != 0) {
                    break;
                }
                unsigned char *q = sqg + st * 2 * kBytes, *g = q + kBytes;
                if (i0 + kTile > last) { // of the products for dP and of both outer ones
                    BarExpect(&sh.tail, 2 * kBytes);
                    load(q, &mapQ, &sh.tail, i0, h);
                    load(g, &mapG, &sh.tail, i0, h);
                    BarWait(&sh.tail, tails++ & 1, failed);
                    if (*failed != 0) {
                        break;
                    }
                    BarExpect(&sh.full[st], 2 * BytesFrom<kTile, HALVES>(n.q - i0) + 2 * kTile * 4);
                    ZerosFrom<kTile, HALVES>(q, n.q - i0, &sh.full[st]);
                    ZerosFrom<kTile, HALVES>(g, n.q - i0, &sh.full[st]);
                } else {
                    BarExpect(&sh.full[st], kStage);
                    load(q, &mapQ, &sh.full[st], i0, h);
                    load(g, &mapG, &sh.full[st], i0, h);
                }
                const int64_t row = (static_cast<int64_t>(b) * s.heads + h) * m.stride + i0;
                BulkLoad(stats + st * 2 * kTile, m.lse2 + row, kTile * 4, &sh.full[st]);
                BulkLoad(stats + st * 2 * kTile + kTile, m.delta + row, kTile * 4, &sh.full[st]);
            }
            BarDrain(&sh.kvFull, 0);
            if (tails > 0) {
                BarDrain(&sh.tail, (tails - 1) & 1);
            }
            for (int32_t e = it > 2 ? it - 2 : 0; e < it; ++e) {
                BarDrain(&sh.full[e & 1], (e / 2) & 1);
            }
        }
        __syncwarp();
    } else if (warp == kProductWarp) {
        if (count > 0) {
            const bool lead = ElectOne();
            const uint32_t descS = ProductDesc<T>(kTile, false, s.scale < 0.0f), descDp = ProductDesc<T>(kTile, false, false);
            const uint32_t descOut = ProductDesc<T>(KS * 16, true, false);
            const uint64_t dk = OperandDesc(SharedAddr(sk), 16), dv = OperandDesc(SharedAddr(sv), 16);
            // Q and gradOut as rows of values (inner products) and as columns (outer ones)
            const uint64_t dq = OperandDesc(SharedAddr(sqg), 16), dqRows = OperandDesc(SharedAddr(sqg), kHalfBytes);
            constexpr uint64_t kPlace = 2 * kBytes >> 4, kGrad = kBytes >> 4;
            auto inner = [&](uint32_t d, uint64_t a, uint64_t rows, uint32_t desc, uint64_t* bar) {
                if (lead) {
                    InnerProducts<KS>(d, a, rows, desc);
                    MmaCommit(bar);
                }
                __syncwarp();
            };
            BarWait(&sh.kvFull, 0, failed);
            BarWait(&sh.full[0], 0, failed);
            TcFenceAfter();
            inner(tS, dk, dq, descS, &sh.sFull);
            inner(tDp, dv, dq + kGrad, descDp, &sh.dpFull);
            for (int32_t it = 0; it < count; ++it) {
                const uint32_t phase = it & 1;
                const uint64_t at = (it & 1) * kPlace, next = ((it + 1) & 1) * kPlace;
                BarWait(&sh.pReady, phase, failed);
                if (__any_sync(0xffffffffu, *failed != 0)) {
                    break;
                }
                TcFenceAfter();
                if (lead) {
                    OuterProducts(tDv, tS, dqRows + at + kGrad, descOut, it > 0);
                    MmaCommit(&sh.dvDone);
                }
                __syncwarp();
                if (it + 1 < count) {
                    BarWait(&sh.full[(it + 1) & 1], ((it + 1) / 2) & 1, failed);
                    BarWait(&sh.dvDone, phase, failed); // the weights, which the next scores go over, have been read
                    TcFenceAfter();
                    inner(tS, dk, dq + next, descS, &sh.sFull);
                }
                BarWait(&sh.dsReady, phase, failed);
                if (__any_sync(0xffffffffu, *failed != 0)) {
                    break;
                }
                TcFenceAfter();
                if (lead) {
                    OuterProducts(tDk, tDp, dqRows + at, descOut, it > 0);
                    MmaCommit(&sh.empty[it & 1]);
                    MmaCommit(&sh.dkDone);
                }
                __syncwarp();
                if (it + 1 < count) {
                    BarWait(&sh.dkDone, phase, failed);
                    TcFenceAfter();
                    inner(tDp, dv, dq + next + kGrad, descDp, &sh.dpFull);
                }
            }
            BarWait(&sh.dkDone, (count - 1) & 1, failed);
            if (*failed != 0) {
                if (lead) {
                    MmaCommit(&sh.drain);
                }
                __syncwarp();
                BarDrain(&sh.drain, 0);
            }
        }
        __syncwarp();
    } else {
        constexpr int kOwn = 64 * HALVES / kSides; // columns of the sums that a thread has
        const int32_t side = warp >> 2, r = (warp & 3) * 32 + (threadIdx.x & 31);
        const int32_t j = j0 + r;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
        const float factor = fabsf(s.scale) * kLog2e;
        const F2 factor2 = MakeF2(factor, factor);
        // positions [from, to) of the queries that see key j, of those that this block walks
        const int32_t from = max(j, low);
        const int32_t to = j >= n.kv ? 0 : (j < s.sinks || s.window > high + 1 - j) ? high + 1 : j + s.window;
        RowScale range;
        for (int32_t it = 0; it < count; ++it) {
            const int32_t st = it & 1;
            const int32_t p0 = n.shift + iBase + (begin + it) % perGroup * kTile + kColumns * side;
            BarWait(&sh.full[st], (it >> 1) & 1, failed); // the statistics
            BarWait(&sh.sFull, it & 1, failed);
            if (__any_sync(0xffffffffu, *failed != 0)) {
                break;
            }
            TcFenceAfter();
            uint32_t x[kColumns];
            TmemLoad32(tS + kColumns * side + lanes, x);
            if (!__all_sync(0xffffffffu, from <= p0 && to >= p0 + kColumns)) {
                uint32_t live[1];
                LiveColumns<kColumns>(live, from - p0, to - p0, 0);
                MaskColumns<kColumns>(x, live);
            }
            const float4* lse = reinterpret_cast<const float4*>(stats + st * 2 * kTile + kColumns * side);
            const float4* del = reinterpret_cast<const float4*>(stats + st * 2 * kTile + kTile + kColumns * side);
#pragma unroll
            for (int e = 0; e < kColumns; e += 4) {
                const float4 l = lse[e / 4];
                float z[4];
                SplitF2(Fma2(MakeF2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), factor2, MakeF2(-l.x, -l.y)), z[0], z[1]);
                SplitF2(Fma2(MakeF2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3])), factor2, MakeF2(-l.z, -l.w)), z[2], z[3]);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[e + k] = __float_as_uint(Exp2(z[k]));
                }
            }
            StoreWeights<T>(tS + kColumns * side + lanes, x, 1.0f);
            TmemStoreWait();
            TcFenceBefore();
            BarArrive(&sh.pReady);
            BarWait(&sh.dpFull, it & 1, failed);
            TcFenceAfter();
            float most = 0.0f;
            {
                uint32_t y[kColumns];
                TmemLoad32(tDp + kColumns * side + lanes, y);
#pragma unroll
                for (int e = 0; e < kColumns; e += 4) {
                    const float4 d = del[e / 4];
                    float z[4];
                    SplitF2(Mul2(Add2(MakeF2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), MakeF2(-d.x, -d.y)),
                                 MakeF2(__uint_as_float(x[e]), __uint_as_float(x[e + 1]))),
                            z[0], z[1]);
                    SplitF2(Mul2(Add2(MakeF2(__uint_as_float(y[e + 2]), __uint_as_float(y[e + 3])), MakeF2(-d.z, -d.w)),
                                 MakeF2(__uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]))),
                            z[2], z[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        x[e + k] = __float_as_uint(z[k]);
                        if constexpr (DType<T>::kIsHalf) {
                            most = fmaxf(most, fabsf(z[k]));
                        }
                    }
                }
            }
            float scale = 1.0f;
            if constexpr (DType<T>::kIsHalf) {
                const float change = range.Follow(LargestOfRow(sh.most[it & 1], side, r, most, &sh.exchanged, it & 1, failed));
                scale = range.scale;
                if (it > 0 && __any_sync(0xffffffffu, change != 1.0f)) {
                    BarWait(&sh.dkDone, (it - 1) & 1, failed);
                    TcFenceAfter();
                    TmemScale<kOwn>(tDk + lanes + kOwn * side, change);
                }
            }
            StoreWeights<T>(tDp + kColumns * side + lanes, x, scale);
            TmemStoreWait();
            TcFenceBefore();
            BarArrive(&sh.dsReady);
        }
        if (count > 0) {
            BarWait(&sh.dkDone, (count - 1) & 1, failed);
            TcFenceAfter();
        }
        const bool lives = j < s.lk;
        bool bad = false;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const float last = which == 0 ? s.scale * kWeightScale / range.scale : kWeightScale;
            const uint32_t from32 = (which == 0 ? tDk : tDv) + lanes;
            float* part = split ? m.partial + (((static_cast<int64_t>(bu) * m.sinkTiles + tile) * (1 + m.farChunks) + 1 + chunk) * 2 + which) *
                                                  kTile * s.dim + static_cast<int64_t>(r) * s.dim :
                                  nullptr;
            T* out = lives && !split ? OutRowOf<T>(which == 0 ? m.a.gradK : m.a.gradV, b, j, u) : nullptr;
            const int32_t d0 = kOwn * side;
            uint32_t o[kOwn];
            if (count > 0) {
                TmemLoadOwn<kOwn>(from32 + d0, o);
            }
            float v[kOwn];
#pragma unroll
            for (int e = 0; e < kOwn; ++e) {
                v[e] = count > 0 && j < n.kv ? __uint_as_float(o[e]) * last : 0.0f;
                bad = bad || (d0 + e < s.dim && !(fabsf(v[e]) <= 3.4e38f));
            }
            if (out != nullptr && d0 < s.dim) {
                StoreRow<T>(out + d0, v, s.dim - d0, which == 0 ? m.vecK : m.vecV);
            }
            if (part != nullptr) {
#pragma unroll
                for (int e = 0; e < kOwn; ++e) {
                    if (d0 + e < s.dim && (chunk < 0 || j < s.sinks)) { // further blocks have sums of sinks alone
                        part[d0 + e] = *failed != 0 ? NAN : v[e];
                    }
                }
            }
        }
        const uint32_t rows = __ballot_sync(0xffffffffu, bad && lives && !split);
        if ((threadIdx.x & 31) == 0 && rows != 0) {
            atomicOr(&sh.bad[warp & 3], rows);
        }
        RowBarrier<kGradThreads>();
        uint32_t again = sh.bad[warp & 3] & (0x11111111u << side);
        while (again != 0) {
            const int e = __ffs(again) - 1;
            again &= again - 1;
            AttnGradKvRow<T>(m.a, b, u, j0 + 32 * (warp & 3) + e);
        }
        if (*failed != 0 && lives && !split && side == 0) {
            T *gk = OutRowOf<T>(m.a.gradK, b, j, u), *gv = OutRowOf<T>(m.a.gradV, b, j, u);
            for (int32_t d = 0; d < s.dim; ++d) {
                gk[d] = gv[d] = DType<T>::FromF(NAN);
            }
        }
    }
    TcFenceBefore();
    __syncthreads();
    if (warp == kProductWarp) {
        TcFenceAfter();
        TmemFree(sh.tmem, 512);
    }
    if (threadIdx.x == 0 && sh.failed != 0) {
        atomicAdd(&g_attentionTimeouts, 1u);
    }
}

template <typename T, int KS>
__global__ void __launch_bounds__(kGradThreads + 64, 1)
    AttnGradMmaKernel(const __grid_constant__ BackwardArgs m, const __grid_constant__ CUtensorMap mapQ,
                      const __grid_constant__ CUtensorMap mapG, const __grid_constant__ CUtensorMap mapK,
                      const __grid_constant__ CUtensorMap mapV)
{
    extern __shared__ unsigned char raw[];
    __shared__ union {
        GradQShared q;
        GradKvShared kv;
    } sh;
    if (blockIdx.x < m.kvBlocks) {
        GradKvBlock<T, KS>(m, mapQ, mapG, mapK, mapV, blockIdx.x, raw, sh.kv);
    } else {
        GradQBlock<T, KS>(m, mapQ, mapG, mapK, mapV, blockIdx.x - m.kvBlocks, raw, sh.q);
    }
}

// gradK and gradV of the keys of tiles with sinks: the blocks' sums in order, a warp per key, a lane per four values of both.
template <typename T>
__global__ void __launch_bounds__(128) AttnSinkGradKernel(const __grid_constant__ BackwardArgs m)
{
    const AttnShape& s = m.a.s;
    const int lane = threadIdx.x & 31;
    const int64_t key = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int64_t tileIndex = key / kTile; // (batch, key head, tile)
    const int32_t r = static_cast<int32_t>(key % kTile);
    const int32_t tile = static_cast<int32_t>(tileIndex % m.sinkTiles);
    const int32_t bu = static_cast<int32_t>(tileIndex / m.sinkTiles);
    const int32_t b = bu / s.kvHeads, u = bu % s.kvHeads, j = tile * kTile + r;
    if (bu >= s.batch * s.kvHeads || j >= s.lk) {
        return;
    }
    const int32_t slots = j < s.sinks ? 1 + m.farChunks : 1;
    const float* part = m.partial + tileIndex * (1 + m.farChunks) * 2 * kTile * s.dim + static_cast<int64_t>(r) * s.dim;
    const int64_t other = static_cast<int64_t>(kTile) * s.dim; // from gradK to gradV
    float sum[2][4] = {};
#pragma unroll 4
    for (int32_t c = 0; c < slots; ++c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (lane + 32 * e < s.dim) {
                sum[0][e] += part[2 * c * other + lane + 32 * e];
                sum[1][e] += part[(2 * c + 1) * other + lane + 32 * e];
            }
        }
    }
    T *gk = OutRowOf<T>(m.a.gradK, b, j, u), *gv = OutRowOf<T>(m.a.gradV, b, j, u);
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (lane + 32 * e < s.dim) {
            gk[lane + 32 * e] = DType<T>::FromF(sum[0][e]);
            gv[lane + 32 * e] = DType<T>::FromF(sum[1][e]);
            bad = bad || !(fabsf(sum[0][e]) <= 3.4e38f) || !(fabsf(sum[1][e]) <= 3.4e38f);
        }
    }
    if (__any_sync(0xffffffffu, bad)) {
        __syncwarp();
        AttnGradKvRow<T>(m.a, b, u, j);
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

bool TmaStride(int64_t stride, int32_t extent) { return extent <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); }

// launch(the steps of 16 values that a head takes): a kernel for each number, so that no head is padded by 16 values or more. 2 x 4096
// tokens, 16 heads on 4, window 1024, bf16, forward and backward: heads of 48 87 and 237 us (88 and 245 in the kernel of 64), of 112 106
// and 314 us (108 and 325 in that of 128).
template <typename Launch>
cudaError_t BySteps(int32_t dim, Launch launch)
{
    switch (CeilDiv(dim, 16)) {
        case 1: return launch(std::integral_constant<int, 1>{});
        case 2: return launch(std::integral_constant<int, 2>{});
        case 3: return launch(std::integral_constant<int, 3>{});
        case 4: return launch(std::integral_constant<int, 4>{});
        case 5: return launch(std::integral_constant<int, 5>{});
        case 6: return launch(std::integral_constant<int, 6>{});
        case 7: return launch(std::integral_constant<int, 7>{});
        default: return launch(std::integral_constant<int, 8>{});
    }
}

template <typename T>
cudaError_t LaunchForward(const MmaArgs& m, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, unsigned grid, int shared,
                          cudaStream_t stream)
{
    return BySteps(m.a.s.dim, [&](auto steps) {
        const auto kernel = AttnForwardMmaKernel<T, decltype(steps)::value>;
        static std::atomic<uint64_t> asked;
        const cudaError_t set = AskOnce(kernel, asked, shared);
        if (set != cudaSuccess) {
            return set;
        }
        kernel<<<grid, 192, shared, stream>>>(m, mq, mk, mv);
        CountLaunch();
        return cudaGetLastError();
    });
}

} // namespace

cudaError_t AttnMakeMap(CUtensorMap* map, Dt dt, const AttnTensor& t, int32_t dim, int32_t tokens, int32_t heads, int32_t batch,
                        int32_t boxTokens)
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
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(boxTokens), 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, dt == Dt::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                              const_cast<void*>(t.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

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
    cudaError_t e = AttnMakeMap(&mq, dt, a.q, s.dim, s.lq, s.heads, s.batch, kTile);
    e = e != cudaSuccess ? e : AttnMakeMap(&mk, dt, a.k, s.dim, s.lk, s.kvHeads, s.batch, kKeys);
    e = e != cudaSuccess ? e : AttnMakeMap(&mv, dt, a.v, s.dim, s.lk, s.kvHeads, s.batch, kKeys);
    if (e != cudaSuccess) {
        return e;
    }
    const int shared = 3 * m.halves * static_cast<int>(kHalfBytes) + 1024;
    const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(s.batch) * s.heads * m.tiles);
    if (dt == Dt::F16) {
        return LaunchForward<__half>(m, mq, mk, mv, grid, shared, stream);
    }
    return LaunchForward<__nv_bfloat16>(m, mq, mk, mv, grid, shared, stream);
}

namespace {

bool VecRows(const AttnTensor& t, int32_t dim) { return dim % 8 == 0 && Aligned(t.p, 16) && t.l % 8 == 0 && t.h % 8 == 0 && t.b % 8 == 0; }

// Further blocks for the sinks' far queries (GradKvBlock): as many as bring their walks down to that of an ordinary block.
struct FarPlan {
    int32_t sinkTiles = 0, chunks = 0;
};
FarPlan PlanFar(const AttnShape& s)
{
    FarPlan f;
    const int64_t sinks = s.sinks < s.lk ? s.sinks : s.lk;
    const int64_t group = s.heads / s.kvHeads;
    const int64_t near = group * (CeilDiv(static_cast<int64_t>(s.window) + kTile, kTile) + 1);
    const int64_t far = group * CeilDiv(s.lq > s.window ? s.lq - s.window : 0, kTile);
    if (sinks > 0 && 2 * far > near) {
        f.sinkTiles = static_cast<int32_t>(CeilDiv(sinks, kTile));
        const int64_t chunks = CeilDiv(far, near);
        f.chunks = AttnFarChunks(static_cast<int64_t>(s.batch) * s.kvHeads, f.sinkTiles, chunks);
        f.sinkTiles = f.chunks > 0 ? f.sinkTiles : 0;
    }
    return f;
}
int64_t StatsStride(const AttnShape& s) { return CeilDiv(s.lq, 4) * 4 + kTile; }
uint64_t StatsBytes(const AttnShape& s) { return (static_cast<uint64_t>(s.batch) * s.heads * StatsStride(s) * 4 + 255) & ~255ull; }

} // namespace

namespace {

struct BackwardLaunch {
    const BackwardArgs& m;
    const CUtensorMap &mq, &mg, &mk, &mv;
    dim3 statBlocks;
    unsigned blocks;
    int shared;
    bool vecStats;
};
template <typename T>
cudaError_t LaunchBackward(const BackwardLaunch& l, cudaStream_t stream)
{
    const BackwardArgs& m = l.m;
    return BySteps(m.a.s.dim, [&](auto steps) {
        const auto kernel = AttnGradMmaKernel<T, decltype(steps)::value>;
        static std::atomic<uint64_t> asked;
        const cudaError_t set = AskOnce(kernel, asked, l.shared);
        if (set != cudaSuccess) {
            return set;
        }
        AttnStatisticsKernel<T><<<l.statBlocks, 256, 0, stream>>>(m, l.vecStats); // rows x heads
        kernel<<<l.blocks, kGradThreads + 64, l.shared, stream>>>(m, l.mq, l.mg, l.mk, l.mv);
        CountLaunch(2);
        if (m.farChunks > 0) {
            const int64_t keys = static_cast<int64_t>(m.a.s.batch) * m.a.s.kvHeads * m.sinkTiles * kTile;
            AttnSinkGradKernel<T><<<static_cast<unsigned>(CeilDiv(keys, 4)), 128, 0, stream>>>(m);
            CountLaunch();
        }
        return cudaGetLastError();
    });
}

} // namespace

uint64_t AttnBackwardMmaWorkspace(const AttnShape& s)
{
    const FarPlan f = PlanFar(s);
    return 2 * StatsBytes(s) + static_cast<uint64_t>(s.batch) * s.kvHeads * f.sinkTiles * (f.chunks + 1) * 2 * kTile * s.dim * 4;
}

cudaError_t AttnBackwardMma(Dt dt, const AttnArgs& a, void* workspace, cudaStream_t stream)
{
    const AttnShape& s = a.s;
    const FarPlan f = PlanFar(s);
    BackwardArgs m{};
    m.a = a;
    m.qTiles = static_cast<int32_t>(CeilDiv(s.lq, kTile));
    m.kTiles = static_cast<int32_t>(CeilDiv(s.lk, kTile));
    m.stride = StatsStride(s);
    m.lse2 = static_cast<float*>(workspace);
    m.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + StatsBytes(s));
    m.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + 2 * StatsBytes(s));
    m.a.delta = m.delta;
    m.a.deltaStride = m.stride;
    m.sinkTiles = f.sinkTiles;
    m.farChunks = f.chunks;
    m.vecQ = VecRows(a.gradQ, s.dim);
    m.vecK = VecRows(a.gradK, s.dim);
    m.vecV = VecRows(a.gradV, s.dim);
    const int64_t heads = static_cast<int64_t>(s.batch) * s.heads;
    const dim3 statBlocks(static_cast<unsigned>(CeilDiv(m.stride, 16 * kStatRows)), static_cast<unsigned>(heads < 65535 ? heads : 65535));
    const int64_t kvBlocks = static_cast<int64_t>(s.batch) * s.kvHeads * (m.kTiles + static_cast<int64_t>(m.sinkTiles) * m.farChunks);
    if (kvBlocks > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    CUtensorMap mq, mg, mk, mv;
    cudaError_t e = AttnMakeMap(&mq, dt, a.q, s.dim, s.lq, s.heads, s.batch, kTile);
    e = e != cudaSuccess ? e : AttnMakeMap(&mg, dt, a.gradOut, s.dim, s.lq, s.heads, s.batch, kTile);
    e = e != cudaSuccess ? e : AttnMakeMap(&mk, dt, a.k, s.dim, s.lk, s.kvHeads, s.batch, kTile);
    e = e != cudaSuccess ? e : AttnMakeMap(&mv, dt, a.v, s.dim, s.lk, s.kvHeads, s.batch, kTile);
    if (e != cudaSuccess) {
        return e;
    }
    const int32_t halves = s.dim > 64 ? 2 : 1;
    const int bytes = halves * static_cast<int>(kHalfBytes);
    // gradQ's tiles, gradK's and gradV's with two places of statistics
    const int shared = std::max(7 * bytes, 6 * bytes + 4 * kTile * 4) + 1024;
    const int64_t blocks = kvBlocks + static_cast<int64_t>(s.batch) * s.heads * m.qTiles;
    if (blocks > INT32_MAX || static_cast<int64_t>(s.batch) * s.kvHeads * m.sinkTiles * (kTile / 4) > INT32_MAX) {
        return cudaErrorInvalidConfiguration;
    }
    m.kvBlocks = static_cast<uint32_t>(kvBlocks);
    const bool vecStats = VecRows(a.gradOut, s.dim) && VecRows(a.out, s.dim);
    const BackwardLaunch l{m, mq, mg, mk, mv, statBlocks, static_cast<unsigned>(blocks), shared, vecStats};
    return dt == Dt::F16 ? LaunchBackward<__half>(l, stream) : LaunchBackward<__nv_bfloat16>(l, stream);
}

uint32_t AttentionTimeouts()
{
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_attentionTimeouts, sizeof(v)) == cudaSuccess ? v + AttnStepTimeouts() : 0xffffffffu;
}

} // namespace opscv
