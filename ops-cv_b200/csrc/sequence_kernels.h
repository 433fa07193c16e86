// Host-callable launchers of the token-sequence kernels (rms_norm.cu, rotary.cu, window_attention*.cu).
#pragma once

#include "kernels.h"

namespace opscv {

// The rows of a tensor whose last dimension is contiguous: row r starts at (r / inner) * s0 + (r % inner) * s1 elements.
struct RowStride {
    int64_t s0 = 0, s1 = 0;
};

struct NormShape {
    int64_t rows = 0;
    int64_t inner = 1; // rows of the inner of the two leading dimensions
    int32_t width = 0;
    double eps = 0.0;
    bool weight32 = false; // weight (and its gradient) in fp32, else in the tensors' type
};

// y = z * rstd * w with z = T(x + residual), rstd = 1 / sqrt(mean(z^2) + eps). residual, weight, sum and rstd may be null.
cudaError_t RmsNormFwd(Dt dt, const NormShape& n, const void* x, RowStride xs, const void* residual, RowStride rs,
                       const void* weight, void* y, RowStride ys, void* sum, RowStride ss, float* rstd, cudaStream_t s);

enum class Q8 : int32_t { E4M3 = 0, INT8 = 1 };
// The same norm, written as 8-bit values (contiguous rows) and a scale per row (group 0) or per `group` columns.
cudaError_t RmsNormQuant(Dt dt, const NormShape& n, const void* x, RowStride xs, const void* residual, RowStride rs,
                         const void* weight, Q8 type, int32_t group, void* q, float* scales, void* sum, RowStride ss,
                         cudaStream_t s);

// Floats of scratch that the backward's per-block sums of the weight's gradient take (0 without a weight).
int64_t RmsNormBwdScratch(Dt dt, const NormShape& n, bool weight);
// gradSum, weight (with gradWeight and scratch) may be null.
cudaError_t RmsNormBwd(Dt dt, const NormShape& n, const void* gradY, RowStride gs, const void* sum, RowStride ss,
                       const float* rstd, const void* weight, const void* gradSum, RowStride as, void* gradX,
                       RowStride xs, void* gradWeight, float* scratch, int64_t scratchFloats, cudaStream_t s);

// ---- rotary positions ----------------------------------------------------------------------------------------------
constexpr int kMaxRotaryAxes = 4;

enum class RotaryScaling : int32_t { NONE = 0, LINEAR = 1, BASE = 2, WAVELENGTH = 3, RAMP = 4 };
// frequencies[i], i < half, in double or float
cudaError_t RotaryFrequencies(void* out, bool is64, int32_t half, double base, RotaryScaling kind, double factor,
                              double originalLength, double low, double high, cudaStream_t s);

struct RotaryTensor { // [token, head, dim], dim contiguous; heads 0: absent
    const void* in = nullptr;
    void* out = nullptr;
    int32_t heads = 0;
    RowStride inTok, outTok; // tokens
    int64_t inHead = 0, outHead = 0;
};
struct RotaryShape {
    int64_t tokens = 0, inner = 1; // tokens of the inner of the two leading dimensions
    int32_t dim = 0, half = 0;     // the first 2 * half values of a head are turned, the others copied
    bool interleaved = false, inverse = false, freq64 = false, pos64 = false;
    int32_t axes = 1;
    int32_t ends[kMaxRotaryAxes] = {}; // frequencies [ends[a - 1], ends[a]) turn by positions of axis a
    int64_t posAxis = 0;               // stride of the axes of positions
    RowStride posTok;
    float scale = 1.0f;
};
cudaError_t RotaryTurn(Dt dt, const RotaryShape& r, const RotaryTensor& q, const RotaryTensor& k, const void* positions,
                       const void* frequencies, cudaStream_t s);

// ---- attention over a sliding window with sinks ------------------------------------------------------------------------------
struct AttnTensor { // [batch, token, head, dim], dim contiguous; strides in elements
    const void* p = nullptr;
    int64_t b = 0, l = 0, h = 0;
};
struct AttnShape {
    int32_t batch = 0, lq = 0, lk = 0, heads = 0, kvHeads = 0, dim = 0;
    int32_t window = 1, sinks = 0; // at most 2^30
    float scale = 1.0f;
    const void *qLen = nullptr, *kvLen = nullptr; // [batch], null: lq, lk
    bool qLen64 = false, kvLen64 = false;
};
constexpr int kMaxAttnDim = 256;

// out and lse ([batch, heads, lq] contiguous) of queries over keys and values.
cudaError_t WindowAttentionFwd(Dt dt, const AttnShape& a, AttnTensor q, AttnTensor k, AttnTensor v, AttnTensor out, float* lse,
                               cudaStream_t s);
// The strides and the alignment of the addresses decide which kernels a call takes; tensors in the workspace may be given by their
// offsets in it.
uint64_t WindowAttentionBwdWorkspace(Dt dt, const AttnShape& a, AttnTensor gradOut, AttnTensor q, AttnTensor k, AttnTensor v);
cudaError_t WindowAttentionBwd(Dt dt, const AttnShape& a, AttnTensor gradOut, AttnTensor q, AttnTensor k, AttnTensor v,
                               AttnTensor out, const float* lse, AttnTensor gradQ, AttnTensor gradK, AttnTensor gradV,
                               void* workspace, cudaStream_t s);

} // namespace opscv
