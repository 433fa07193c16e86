// What the attention kernels share: the arguments, which keys a query sees, and a row of the result by one warp.
//
// Query i of a sequence with qLen queries and kvLen keys sits at position p = kvLen - qLen + i and sees the keys j <= p with
// j > p - window or j < sinks. With s_j = scale q.k_j:  out = sum_j exp(s_j - lse) v_j, lse = log sum_j exp(s_j).
// A query that sees nothing (behind qLen, or before the first key) has out 0 and lse -inf.
// Backward, with p_j = exp(s_j - lse) and delta = gradOut . out:
//   gradV_j += p_j gradOut, ds_j = p_j (gradOut . v_j - delta) scale, gradQ += ds_j k_j, gradK_j += ds_j q.
#pragma once

#include <algorithm>

#include <cuda.h> // CUtensorMap

#include "launch_util.cuh"
#include "sequence_kernels.h"

namespace opscv {

struct AttnArgs {
    AttnShape s;
    AttnTensor q, k, v, out, gradOut, gradQ, gradK, gradV;
    float* lse;         // [batch, heads, lq], null where it is not wanted
    const float* delta; // the same with rows of deltaStride (backward)
    int64_t deltaStride;
    int32_t group;      // heads / kvHeads
};

__device__ __forceinline__ int32_t LengthOf(const void* p, bool is64, int32_t b, int32_t most)
{
    if (p == nullptr) {
        return most;
    }
    const long long n = is64 ? static_cast<const long long*>(p)[b] : static_cast<const int*>(p)[b];
    return static_cast<int32_t>(n < 0 ? 0 : (n > most ? most : n)); // lengths outside the tensors are cut to them
}
struct Lengths {
    int32_t q, kv;
    int32_t shift; // position of query 0
};
__device__ __forceinline__ Lengths LengthsOf(const AttnShape& s, int32_t b)
{
    Lengths n;
    n.q = LengthOf(s.qLen, s.qLen64, b, s.lq);
    n.kv = LengthOf(s.kvLen, s.kvLen64, b, s.lk);
    n.shift = n.kv - n.q;
    return n;
}

// The keys that the query at position p sees: [0, sinkEnd) and [first, p]. p < 0: none.
struct Seen {
    int32_t sinkEnd, first, count;
};
__device__ __forceinline__ Seen SeenOf(const AttnShape& s, int32_t p)
{
    Seen r{0, 0, 0};
    if (p >= 0) {
        r.first = p >= s.window ? p - s.window + 1 : 0;
        r.sinkEnd = s.sinks < r.first ? s.sinks : r.first;
        r.count = r.sinkEnd + (p - r.first + 1);
    }
    return r;
}
__device__ __forceinline__ int32_t SeenKey(const Seen& r, int32_t n) { return n < r.sinkEnd ? n : r.first + (n - r.sinkEnd); }

template <typename T>
__device__ __forceinline__ const T* RowOf(const AttnTensor& t, int32_t b, int32_t l, int32_t h)
{
    return static_cast<const T*>(t.p) + b * t.b + l * t.l + h * t.h;
}
template <typename T>
__device__ __forceinline__ T* OutRowOf(const AttnTensor& t, int32_t b, int32_t l, int32_t h)
{
    return const_cast<T*>(RowOf<T>(t, b, l, h));
}

__device__ __forceinline__ float WarpSum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}
__device__ __forceinline__ float WarpMax(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    }
    return v;
}

template <typename T>
__device__ __forceinline__ float DotRows(const T* a, const T* b, int32_t dim)
{
    float s = 0.0f;
    for (int32_t d = 0; d < dim; ++d) {
        s = fmaf(DType<T>::ToF(a[d]), DType<T>::ToF(b[d]), s);
    }
    return s;
}

constexpr int kLaneDims = kMaxAttnDim / 32; // dims d = lane + 32 c of a row belong to a lane

// ---- rows of the results by one warp ---------------------------------------------------------------------------------------
// These touch the visible keys (or queries) and nothing else, so what lies in masked places cannot reach the result. The tiled
// kernels multiply masked pairs by a weight of zero, which is the same unless the masked value is an infinity or a NaN; they hand
// the rows that came out not finite to these.
// 32 keys at a time: a lane forms the score of its key, then all lanes add the 32 weighted rows to the dims that they own.
template <typename T>
__device__ __noinline__ void AttnForwardRow(const AttnArgs& a, int32_t b, int32_t h, int32_t i)
{
    const int lane = threadIdx.x & 31;
    const Lengths n = LengthsOf(a.s, b);
    const Seen seen = SeenOf(a.s, i < n.q ? n.shift + i : -1);
    const T* q = RowOf<T>(a.q, b, i, h);
    const int32_t u = h / a.group;
    float acc[kLaneDims] = {};
    float top = -INFINITY, total = 0.0f;
    for (int32_t at = 0; at < seen.count; at += 32) {
        const bool live = at + lane < seen.count;
        const int32_t j = live ? SeenKey(seen, at + lane) : 0;
        const float s = live ? DotRows(q, RowOf<T>(a.k, b, j, u), a.s.dim) * a.s.scale : -INFINITY;
        const float next = fmaxf(top, WarpMax(s));
        const float base = next == -INFINITY ? 0.0f : next;
        const float fade = expf(top - base); // 0 at first
        const float w = live ? expf(s - base) : 0.0f; // a NaN score stays one
        total = total * fade + WarpSum(w);
        top = next;
#pragma unroll
        for (int c = 0; c < kLaneDims; ++c) {
            acc[c] *= fade;
        }
        const int32_t m = seen.count - at < 32 ? seen.count - at : 32;
        for (int32_t r = 0; r < m; ++r) {
            const float wr = __shfl_sync(0xffffffffu, w, r);
            const T* v = RowOf<T>(a.v, b, __shfl_sync(0xffffffffu, j, r), u);
#pragma unroll
            for (int c = 0; c < kLaneDims; ++c) {
                const int32_t d = lane + 32 * c;
                if (d < a.s.dim) {
                    acc[c] = fmaf(wr, DType<T>::ToF(v[d]), acc[c]);
                }
            }
        }
    }
    T* out = OutRowOf<T>(a.out, b, i, h);
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) {
        const int32_t d = lane + 32 * c;
        if (d < a.s.dim) {
            out[d] = DType<T>::FromF(seen.count > 0 ? acc[c] / total : 0.0f);
        }
    }
    if (lane == 0 && a.lse != nullptr) {
        a.lse[(static_cast<int64_t>(b) * a.s.heads + h) * a.s.lq + i] = seen.count > 0 ? top + logf(total) : -INFINITY;
    }
}

template <typename T>
__device__ __noinline__ void AttnGradQRow(const AttnArgs& a, int32_t b, int32_t h, int32_t i)
{
    const int lane = threadIdx.x & 31;
    const Lengths n = LengthsOf(a.s, b);
    const Seen seen = SeenOf(a.s, i < n.q ? n.shift + i : -1);
    const T* q = RowOf<T>(a.q, b, i, h);
    const T* g = RowOf<T>(a.gradOut, b, i, h);
    const int32_t u = h / a.group;
    const int64_t head = static_cast<int64_t>(b) * a.s.heads + h;
    const float lse = a.lse[head * a.s.lq + i], delta = a.delta[head * a.deltaStride + i];
    float acc[kLaneDims] = {};
    for (int32_t at = 0; at < seen.count; at += 32) {
        const bool live = at + lane < seen.count;
        const int32_t j = live ? SeenKey(seen, at + lane) : 0;
        float ds = 0.0f;
        if (live) {
            const float p = expf(DotRows(q, RowOf<T>(a.k, b, j, u), a.s.dim) * a.s.scale - lse);
            ds = p * (DotRows(g, RowOf<T>(a.v, b, j, u), a.s.dim) - delta) * a.s.scale;
        }
        const int32_t m = seen.count - at < 32 ? seen.count - at : 32;
        for (int32_t r = 0; r < m; ++r) {
            const float dr = __shfl_sync(0xffffffffu, ds, r);
            const T* k = RowOf<T>(a.k, b, __shfl_sync(0xffffffffu, j, r), u);
#pragma unroll
            for (int c = 0; c < kLaneDims; ++c) {
                const int32_t d = lane + 32 * c;
                if (d < a.s.dim) {
                    acc[c] = fmaf(dr, DType<T>::ToF(k[d]), acc[c]);
                }
            }
        }
    }
    T* out = OutRowOf<T>(a.gradQ, b, i, h);
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) {
        const int32_t d = lane + 32 * c;
        if (d < a.s.dim) {
            out[d] = DType<T>::FromF(acc[c]);
        }
    }
}

// The queries that see key j: positions [j, last], the last of the window or, for a sink, of the sequence.
template <typename T>
__device__ __noinline__ void AttnGradKvRow(const AttnArgs& a, int32_t b, int32_t u, int32_t j)
{
    const int lane = threadIdx.x & 31;
    const Lengths n = LengthsOf(a.s, b);
    const int32_t end = n.shift + n.q; // one behind the last position
    int32_t last = j < a.s.sinks || a.s.window > end - j ? end - 1 : j + a.s.window - 1;
    if (j >= n.kv) {
        last = -1;
    }
    const int32_t first = j > n.shift ? j : n.shift;
    const T* k = RowOf<T>(a.k, b, j, u);
    const T* v = RowOf<T>(a.v, b, j, u);
    float accK[kLaneDims] = {}, accV[kLaneDims] = {};
    for (int32_t h = u * a.group; h < (u + 1) * a.group; ++h) {
        const int64_t head = static_cast<int64_t>(b) * a.s.heads + h;
        for (int32_t at = first; at <= last; at += 32) {
            const int32_t i = at + lane - n.shift;
            float p = 0.0f, ds = 0.0f;
            if (at + lane <= last) {
                p = expf(DotRows(RowOf<T>(a.q, b, i, h), k, a.s.dim) * a.s.scale - a.lse[head * a.s.lq + i]);
                ds = p * (DotRows(RowOf<T>(a.gradOut, b, i, h), v, a.s.dim) - a.delta[head * a.deltaStride + i]) * a.s.scale;
            }
            const int32_t m = last - at + 1 < 32 ? last - at + 1 : 32;
            for (int32_t r = 0; r < m; ++r) {
                const float pr = __shfl_sync(0xffffffffu, p, r), dr = __shfl_sync(0xffffffffu, ds, r);
                const T* q = RowOf<T>(a.q, b, at - n.shift + r, h);
                const T* g = RowOf<T>(a.gradOut, b, at - n.shift + r, h);
#pragma unroll
                for (int c = 0; c < kLaneDims; ++c) {
                    const int32_t d = lane + 32 * c;
                    if (d < a.s.dim) {
                        accV[c] = fmaf(pr, DType<T>::ToF(g[d]), accV[c]);
                        accK[c] = fmaf(dr, DType<T>::ToF(q[d]), accK[c]);
                    }
                }
            }
        }
    }
    T* gk = OutRowOf<T>(a.gradK, b, j, u);
    T* gv = OutRowOf<T>(a.gradV, b, j, u);
#pragma unroll
    for (int c = 0; c < kLaneDims; ++c) {
        const int32_t d = lane + 32 * c;
        if (d < a.s.dim) {
            gk[d] = DType<T>::FromF(accK[c]);
            gv[d] = DType<T>::FromF(accV[c]);
        }
    }
}

// ---- few queries (window_attention_step.cu) ----------------------------------------------------------------------------------
bool AttnStepTakes(Dt dt, const AttnArgs& a);
cudaError_t AttnStep(Dt dt, const AttnArgs& a, cudaStream_t stream);
uint32_t AttnStepTimeouts();

// ---- fp32 arithmetic (window_attention_tiles.cu) -------------------------------------------------------------------------------
cudaError_t AttnForwardTiles(Dt dt, const AttnArgs& a, cudaStream_t stream);
// a.delta is the start of the workspace, and filled
uint64_t AttnBackwardTilesWorkspace(const AttnShape& s);
cudaError_t AttnBackwardTiles(Dt dt, const AttnArgs& a, void* workspace, cudaStream_t stream);

// ---- tensor-core kernels (window_attention_mma.cu) ---------------------------------------------------------------------------
bool AttnTmaReadable(const AttnTensor& t, int32_t tokens, int32_t heads, int32_t batch);
// Boxes of 64 values by boxTokens tokens of one head, in the 128-byte swizzle; what lies outside the tensor arrives as zeros.
cudaError_t AttnMakeMap(CUtensorMap* map, Dt dt, const AttnTensor& t, int32_t dim, int32_t tokens, int32_t heads, int32_t batch,
                        int32_t boxTokens);
// 16-bit tensors that boxes can be loaded from, heads of at most 128 values, scale != 0
cudaError_t AttnForwardMma(Dt dt, const AttnArgs& a, cudaStream_t stream);
// a.lse, a.out and a.gradOut too; the workspace holds delta and the statistics, and partial sums of the sinks' gradients
uint64_t AttnBackwardMmaWorkspace(const AttnShape& s);
cudaError_t AttnBackwardMma(Dt dt, const AttnArgs& a, void* workspace, cudaStream_t stream);
constexpr int kMmaMostDim = 128;

// Blocks that share out the far queries of a tile with sinks, of the `wanted` that bring their walks down to an ordinary one's; 0: the
// tile's own block walks them. Each costs memory for its sums, so there are no more than four of them an SM over all units and tiles:
// longer walks then end with the others, and the sums take some 150 MB at most. Backward, heads of 128, bf16, with 4, 8 and 16 an SM:
// 32 sequences of 2048, 8 heads, window 128, 300 sinks 904, 1266 and 1568 us; 64 of 4096, window 64, 4 sinks 3176, 3192 and 3246 (3438
// and 805 MB without a limit). Nor more than 64 a tile: 65536 tokens, one head, window 256: 144 us, 165 with 128; fp32, 16384 tokens,
// window 64: 171 us, 189 with 128, 194 with 32. The SMs are a constant, not the device's, because both phases have to come to one plan.
inline int32_t AttnFarChunks(int64_t units, int32_t sinkTiles, int64_t wanted)
{
    const int64_t enough = 4 * kNumSMsFallback / (units * sinkTiles > 0 ? units * sinkTiles : 1);
    return static_cast<int32_t>(std::min({wanted, enough, static_cast<int64_t>(64)}));
}

} // namespace opscv
