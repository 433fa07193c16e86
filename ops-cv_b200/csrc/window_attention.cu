// Attention over a sliding window with sinks: which kernels a call takes.
#include "window_attention.cuh"

namespace opscv {

namespace {

constexpr int kRowWarps = 4;

// delta = gradOut . out, a warp per row
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) AttnDeltaKernel(AttnArgs a, float* delta)
{
    const int lane = threadIdx.x & 31;
    const int32_t i = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    if (i >= a.s.lq) {
        return;
    }
    for (int32_t bh = blockIdx.y; bh < a.s.batch * a.s.heads; bh += gridDim.y) {
        const int32_t b = bh / a.s.heads, h = bh % a.s.heads;
        const T* g = RowOf<T>(a.gradOut, b, i, h);
        const T* o = RowOf<T>(a.out, b, i, h);
        float s = 0.0f;
        for (int32_t d = lane; d < a.s.dim; d += 32) {
            s = fmaf(DType<T>::ToF(g[d]), DType<T>::ToF(o[d]), s);
        }
        s = WarpSum(s);
        if (lane == 0) {
            delta[static_cast<int64_t>(bh) * a.s.lq + i] = s;
        }
    }
}

dim3 RowGrid(int32_t rows, int64_t others)
{
    return dim3(static_cast<unsigned>(CeilDiv(rows, kRowWarps)), static_cast<unsigned>(others < 65535 ? others : 65535));
}

// Whether a call can take the tensor-core kernels: scores of a scale near 0 keep to the others, where 0 times an infinity is handled.
bool MmaTakes(Dt dt, const AttnArgs& a)
{
    const AttnShape& s = a.s;
    return dt != Dt::F32 && s.dim <= kMmaMostDim && fabsf(s.scale) > 1e-30f && s.lk > 0 &&
           static_cast<int64_t>(s.batch) * s.heads * CeilDiv(s.lq, 128) <= INT32_MAX && AttnTmaReadable(a.q, s.lq, s.heads, s.batch) &&
           AttnTmaReadable(a.k, s.lk, s.kvHeads, s.batch) && AttnTmaReadable(a.v, s.lk, s.kvHeads, s.batch);
}

bool BackwardTakesMma(Dt dt, const AttnArgs& a)
{
    const AttnShape& s = a.s;
    return s.lq > 0 && s.heads > 0 && MmaTakes(dt, a) && AttnTmaReadable(a.gradOut, s.lq, s.heads, s.batch);
}

} // namespace

cudaError_t WindowAttentionFwd(Dt dt, const AttnShape& s, AttnTensor q, AttnTensor k, AttnTensor v, AttnTensor out, float* lse,
                               cudaStream_t stream)
{
    AttnArgs a{};
    a.s = s;
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.lse = lse;
    a.group = s.heads / s.kvHeads;
    if (AttnStepTakes(dt, a)) {
        return AttnStep(dt, a, stream);
    }
    if (MmaTakes(dt, a)) {
        return AttnForwardMma(dt, a, stream);
    }
    return AttnForwardTiles(dt, a, stream);
}

uint64_t WindowAttentionBwdWorkspace(Dt dt, const AttnShape& s, AttnTensor gradOut, AttnTensor q, AttnTensor k, AttnTensor v)
{
    AttnArgs a{};
    a.s = s;
    a.q = q;
    a.k = k;
    a.v = v;
    a.gradOut = gradOut;
    return BackwardTakesMma(dt, a) ? AttnBackwardMmaWorkspace(s) : AttnBackwardTilesWorkspace(s);
}

cudaError_t WindowAttentionBwd(Dt dt, const AttnShape& s, AttnTensor gradOut, AttnTensor q, AttnTensor k, AttnTensor v, AttnTensor out,
                               const float* lse, AttnTensor gradQ, AttnTensor gradK, AttnTensor gradV, void* workspace,
                               cudaStream_t stream)
{
    AttnArgs a{};
    a.s = s;
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.gradOut = gradOut;
    a.gradQ = gradQ;
    a.gradK = gradK;
    a.gradV = gradV;
    a.lse = const_cast<float*>(lse);
    float* delta = static_cast<float*>(workspace);
    a.delta = delta;
    a.deltaStride = s.lq;
    a.group = s.heads / s.kvHeads;
    if (BackwardTakesMma(dt, a)) {
        return AttnBackwardMma(dt, a, workspace, stream);
    }
    if (s.lq > 0 && s.heads > 0) { // without queries, the gradients of the keys are zeros
        const dim3 rows = RowGrid(s.lq, static_cast<int64_t>(s.batch) * s.heads);
        OPSCV_DISPATCH_DT(dt, T, AttnDeltaKernel<T><<<rows, 32 * kRowWarps, 0, stream>>>(a, delta));
        CountLaunch();
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) {
            return e;
        }
    }
    return AttnBackwardTiles(dt, a, workspace, stream);
}

} // namespace opscv
