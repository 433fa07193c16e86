// First- and second-phase entry points of the token-sequence operators (include/aclnn_sequence.h).
#include <cmath>
#include <exception>
#include <optional>

#include "../../include/aclnn_sequence.h"
#include "host_common.h"
#include "sequence_kernels.h"

using namespace opscv;

namespace {

// The first phases allocate (executors, lists of steps): nothing thrown there leaves a C entry point.
template <typename F>
aclnnStatus Guarded(const char* api, uint64_t* workspaceSize, aclOpExecutor** executor, F plan)
{
    if (workspaceSize == nullptr || executor == nullptr) {
        return Fail(ACLNN_ERR_PARAM_NULLPTR, "%s: workspaceSize or executor is null", api);
    }
    aclOpExecutor* ex = nullptr;
    try {
        ex = NewExecutor(api);
        if (ex == nullptr) {
            return Fail(ACLNN_ERR_INNER_CREATE_EXECUTOR, "%s: cannot create executor", api);
        }
        WsPlan ws;
        const aclnnStatus st = plan(*ex, ws);
        if (st != ACLNN_SUCCESS) {
            ReleaseExecutor(ex);
            return st;
        }
        ex->workspaceSize = ws.Size();
        *workspaceSize = ws.Size();
        *executor = ex;
        return ACLNN_SUCCESS;
    } catch (const std::exception& e) {
        if (ex != nullptr) {
            ReleaseExecutor(ex);
        }
        return Fail(ACLNN_ERR_INNER, "%s: %s", api, e.what());
    }
}

#define OPSCV_REQUIRE(cond, ...)                             \
    do {                                                     \
        if (!(cond)) {                                       \
            return Fail(ACLNN_ERR_PARAM_INVALID, __VA_ARGS__); \
        }                                                    \
    } while (0)
#define OPSCV_NOT_NULL(cond, api)                                              \
    do {                                                                       \
        if (!(cond)) {                                                         \
            return Fail(ACLNN_ERR_PARAM_NULLPTR, "%s: null argument", api);    \
        }                                                                      \
    } while (0)

#define OPSCV_TRY(expr)                     \
    do {                                    \
        const aclnnStatus st_ = (expr);     \
        if (st_ != ACLNN_SUCCESS) {         \
            return st_;                     \
        }                                   \
    } while (0)

int64_t Last(const aclTensor* t) { return t->dims[t->dims.size() - 1]; }

bool LeadEqual(const aclTensor* a, const aclTensor* b, size_t lead)
{
    for (size_t i = 0; i < lead; ++i) {
        if (a->dims[i] != b->dims[i]) {
            return false;
        }
    }
    return true;
}

// An output with a stride of 0 along more than one element would be written by several threads.
bool WritesApart(const aclTensor* t)
{
    for (size_t i = 0; i < t->dims.size(); ++i) {
        if (t->dims[i] > 1 && t->strides[i] == 0) {
            return false;
        }
    }
    return true;
}

// of a tensor that goes to the kernels as it is
bool Dense(const aclTensor* t) { return IsEmpty(t) || IsContiguous(t); }

bool LastContiguous(const aclTensor* t)
{
    const size_t n = t->dims.size();
    return t->dims[n - 1] <= 1 || t->strides[n - 1] == 1;
}

char* DataOf(const aclTensor* t, int elem) { return static_cast<char*>(t->data) + t->offset * elem; }

// A tensor with elements has an address: a kernel would fault on none.
bool HasData(const aclTensor* t) { return t == nullptr || t->data != nullptr || IsEmpty(t); }
aclnnStatus CheckData(const char* api, std::initializer_list<const aclTensor*> ts)
{
    for (const aclTensor* t : ts) {
        if (!HasData(t)) {
            return Fail(ACLNN_ERR_PARAM_NULLPTR, "%s: a tensor has no data", api);
        }
    }
    return ACLNN_SUCCESS;
}

// One floating tensor of a call, as the kernels get it: the view itself, or a contiguous copy in the workspace.
struct Operand {
    const aclTensor* given = nullptr;
    aclTensor view;
    BufRef buf;
    bool output = false, staged = false;
};

aclTensor ContiguousLike(const aclTensor* t)
{
    aclTensor c = *t;
    int64_t s = 1;
    for (size_t i = c.dims.size(); i-- > 0;) {
        c.strides[i] = s;
        s *= c.dims[i];
    }
    c.offset = 0;
    return c;
}

// The leading dimensions of tensors that share them, as at most two: neighbours merge where every tensor allows it.
struct Lead {
    int64_t total = 1, inner = 1;
};
class LeadMerge {
public:
    explicit LeadMerge(size_t lead) : lead_(lead) {}
    // strides of t's dimensions [from, from + lead); `to` gets the result
    void Add(const aclTensor* t, size_t from, RowStride* to) { uses_[used_++] = {t, from, to}; } // at most five
    bool Run(Lead& out)
    {
        int64_t extent[2] = {1, 1}; // of the levels, and the dimension whose stride each has
        size_t last[2] = {0, 0};
        int count = 0;
        const Use& u0 = uses_[0];
        for (size_t i = 0; i < lead_; ++i) {
            const int64_t n = u0.t->dims[u0.from + i];
            if (n == 1) {
                continue;
            }
            bool joins = count > 0;
            for (int x = 0; x < used_; ++x) {
                const Use& u = uses_[x];
                if (joins) {
                    joins = u.t->strides[u.from + last[count - 1]] == u.t->strides[u.from + i] * n;
                }
            }
            if (joins) {
                extent[count - 1] *= n;
                last[count - 1] = i;
            } else if (count == 2) {
                return false;
            } else {
                extent[count] = n;
                last[count++] = i;
            }
        }
        out.total = extent[0] * extent[1];
        out.inner = count > 0 ? extent[count - 1] : 1;
        for (int x = 0; x < used_; ++x) {
            const Use& u = uses_[x];
            u.to->s1 = count > 0 ? u.t->strides[u.from + last[count - 1]] : 0;
            u.to->s0 = count == 2 ? u.t->strides[u.from + last[0]] : 0;
        }
        return true;
    }

private:
    struct Use {
        const aclTensor* t;
        size_t from;
        RowStride* to;
    };
    size_t lead_;
    Use uses_[5];
    int used_ = 0;
};

// Gives every operand its buffer: itself, or a staged copy where `stage` says so (or where it has to be).
aclnnStatus Place(const char* api, std::initializer_list<Operand*> ops, bool stageAll, aclOpExecutor& ex, WsPlan& ws)
{
    for (Operand* o : ops) {
        if (o->given == nullptr) {
            continue;
        }
        o->staged = !IsContiguous(o->given) && (stageAll || !LastContiguous(o->given));
        if (o->staged) {
            OPSCV_REQUIRE(ViewStageable(o->given), "%s: view not supported (more than four strided dimensions)", api);
            o->view = ContiguousLike(o->given);
            o->buf = o->output ? StageOutput(o->given, ws) : StageInput(o->given, ws, &ex);
        } else {
            o->view = *o->given;
            o->buf = BufRef{};
            o->buf.base = DataOf(o->given, ElemSize(o->given->dtype));
        }
    }
    return ACLNN_SUCCESS;
}
void Finish(std::initializer_list<Operand*> ops, aclOpExecutor& ex)
{
    for (Operand* o : ops) {
        if (o->given != nullptr && o->output && o->staged) {
            FinishOutput(o->given, o->buf, &ex);
        }
    }
}
Operand In(const aclTensor* t)
{
    Operand o;
    o.given = t;
    return o;
}
Operand Out(const aclTensor* t)
{
    Operand o;
    o.given = t;
    o.output = true;
    return o;
}

// Whether staging is needed at all is known only after the merge of the leading dimensions has been tried on the views.
template <typename AddAll>
bool MergesAsGiven(std::initializer_list<Operand*> ops, size_t lead, AddAll addAll, Lead& out)
{
    for (Operand* o : ops) {
        if (o->given != nullptr) {
            const bool direct = IsContiguous(o->given) || LastContiguous(o->given);
            o->view = direct ? *o->given : ContiguousLike(o->given);
        }
    }
    LeadMerge m(lead);
    addAll(m);
    return m.Run(out);
}

// ---- norm --------------------------------------------------------------------------------------------------------------------
aclnnStatus CheckNormTensor(const char* api, const aclTensor* x, const aclTensor* t, const char* name)
{
    if (t == nullptr) {
        return ACLNN_SUCCESS;
    }
    OPSCV_REQUIRE(t->dtype == x->dtype, "%s: %s must have the type of the others, got %s", api, name, DtypeName(t->dtype));
    OPSCV_REQUIRE(t->dims == x->dims, "%s: %s must have the shape of the others", api, name);
    return ACLNN_SUCCESS;
}

aclnnStatus CheckNorm(const char* api, const aclTensor* x, const aclTensor* weight)
{
    OPSCV_REQUIRE(DtypeSupported(x->dtype), "%s: dtype %s not supported (FLOAT, FLOAT16, BF16)", api, DtypeName(x->dtype));
    OPSCV_REQUIRE(x->dims.size() >= 1, "%s: at least one dimension is needed", api);
    OPSCV_REQUIRE(Last(x) >= 1 && Last(x) <= INT32_MAX / 2, "%s: the last extent must be in [1, 2^30)", api);
    if (weight != nullptr) {
        OPSCV_REQUIRE(weight->dtype == x->dtype || weight->dtype == ACL_FLOAT, "%s: weight must have the tensors' type or FLOAT, got %s",
                      api, DtypeName(weight->dtype));
        OPSCV_REQUIRE(weight->dims.size() == 1 && weight->dims[0] == Last(x), "%s: weight must be [%ld]", api, (long)Last(x));
    }
    return ACLNN_SUCCESS;
}

// fp32 tensor with x's leading dimensions, and `last` values for each where last > 0
aclnnStatus CheckPerRow(const char* api, const aclTensor* x, const aclTensor* t, int64_t last, const char* name)
{
    if (t == nullptr) {
        return ACLNN_SUCCESS;
    }
    const size_t lead = x->dims.size() - 1;
    OPSCV_REQUIRE(t->dtype == ACL_FLOAT, "%s: %s must be FLOAT, got %s", api, name, DtypeName(t->dtype));
    OPSCV_REQUIRE(t->dims.size() == lead + (last > 0 ? 1 : 0) && LeadEqual(x, t, lead) && (last <= 0 || Last(t) == last),
                  "%s: %s does not have the rows' shape", api, name);
    OPSCV_REQUIRE(Dense(t), "%s: %s must be contiguous", api, name);
    return ACLNN_SUCCESS;
}

// The kernels take eps and scales in fp32.
bool Finite32(double v) { return std::isfinite(static_cast<float>(v)); }
bool EpsOk(double eps) { return Finite32(eps) && eps >= 0.0; }

NormShape ShapeOf(const aclTensor* x, const aclTensor* weight, double eps)
{
    NormShape n;
    n.width = static_cast<int32_t>(Last(x));
    n.eps = eps;
    n.weight32 = weight != nullptr && weight->dtype == ACL_FLOAT;
    return n;
}

// ---- rotary ------------------------------------------------------------------------------------------------------------------
// Positions that broadcast along a dimension between others do not merge with them; such go through a copy, axis by axis, in which the
// dimensions that broadcast in front of all others stay as they are. Those that stand for themselves in three dimensions or more do not:
// the kernel reads two.
class PositionsCopy {
public:
    PositionsCopy(const aclTensor* positions, size_t axesDim) : given_(positions), axesDim_(axesDim), axis_(*positions), copied_(*positions)
    {
        const size_t rank = positions->dims.size();
        from_ = axesDim;
        while (from_ < rank && (positions->dims[from_] == 1 || positions->strides[from_] == 0)) {
            ++from_;
        }
        axis_.dims.assign(positions->dims.begin() + from_, positions->dims.end());
        axis_.strides.assign(positions->strides.begin() + from_, positions->strides.end());
        int64_t stride = 1;
        for (size_t i = rank; i-- > from_;) {
            copied_.strides[i] = stride;
            stride *= positions->dims[i];
        }
    }
    bool Possible() const
    {
        int levels = 0;
        int64_t last = 0;
        for (size_t i = 0; i < axis_.dims.size(); ++i) {
            const int64_t n = axis_.dims[i], stride = axis_.strides[i];
            if (n == 1 || stride == 0) {
                continue;
            }
            levels += levels == 0 || last != stride * n ? 1 : 0;
            last = stride;
        }
        return levels <= 2 && !IsContiguous(&axis_) && ViewStageable(&axis_);
    }
    const aclTensor& View() const { return copied_; } // strides of one axis; that between axes comes with Stage
    // the copies, and the stride between their axes
    BufRef Stage(WsPlan& ws, aclOpExecutor* ex, int64_t* axisStride)
    {
        const int64_t axes = axesDim_ != 0 ? given_->dims[0] : 1;
        BufRef first;
        for (int64_t a = 0; a < axes; ++a) {
            aclTensor one = axis_;
            one.offset += axesDim_ != 0 ? a * given_->strides[0] : 0;
            const BufRef at = StageInput(&one, ws, ex);
            if (a == 0) {
                first = at;
            } else if (a == 1) {
                *axisStride = static_cast<int64_t>(at.wsOff - first.wsOff) / ElemSize(given_->dtype);
            }
        }
        return first;
    }

private:
    const aclTensor* given_;
    size_t axesDim_, from_ = 0;
    aclTensor axis_, copied_;
};

aclnnStatus PlanRotary(const char* api, const aclTensor* q, const aclTensor* k, const aclTensor* positions,
                       const aclTensor* frequencies, const aclIntArray* sections, bool interleaved, double scale, bool inverse,
                       aclTensor* qOut, aclTensor* kOut, aclOpExecutor& ex, WsPlan& ws)
{
    OPSCV_NOT_NULL(q != nullptr && positions != nullptr && frequencies != nullptr && qOut != nullptr, api);
    OPSCV_NOT_NULL((k == nullptr) == (kOut == nullptr), api);
    OPSCV_REQUIRE(DtypeSupported(q->dtype), "%s: dtype %s not supported (FLOAT, FLOAT16, BF16)", api, DtypeName(q->dtype));
    const size_t rank = q->dims.size();
    OPSCV_REQUIRE(rank >= 2, "%s: q must be [..., heads, dim]", api);
    const size_t lead = rank - 2;
    OPSCV_REQUIRE(qOut->dims == q->dims && qOut->dtype == q->dtype, "%s: the output must have q's shape and type", api);
    if (k != nullptr) {
        OPSCV_REQUIRE(k->dtype == q->dtype && kOut->dtype == q->dtype, "%s: q and k must have one type", api);
        OPSCV_REQUIRE(k->dims.size() == rank && LeadEqual(q, k, lead) && Last(k) == Last(q),
                      "%s: k must be [..., heads, dim] with q's leading dimensions and dim", api);
        OPSCV_REQUIRE(kOut->dims == k->dims, "%s: the output must have k's shape", api);
    }
    OPSCV_REQUIRE(positions->dtype == ACL_INT32 || positions->dtype == ACL_INT64, "%s: positions must be INT32 or INT64, got %s",
                  api, DtypeName(positions->dtype));
    OPSCV_REQUIRE(frequencies->dtype == ACL_DOUBLE || frequencies->dtype == ACL_FLOAT,
                  "%s: frequencies must be DOUBLE or FLOAT, got %s", api, DtypeName(frequencies->dtype));
    OPSCV_REQUIRE(frequencies->dims.size() == 1 && Dense(frequencies), "%s: frequencies must be one contiguous dimension",
                  api);
    const int64_t half = frequencies->dims[0];
    OPSCV_REQUIRE(half >= 1 && 2 * half <= Last(q) && half <= 2048, "%s: %ld frequencies do not fit a head of %ld values", api,
                  (long)half, (long)Last(q));
    OPSCV_REQUIRE(Finite32(scale), "%s: scale must be finite in fp32", api);
    const size_t axesDim = sections != nullptr ? 1 : 0;
    RotaryShape r;
    if (sections != nullptr) {
        const size_t n = sections->v.size();
        OPSCV_REQUIRE(n >= 1 && n <= kMaxRotaryAxes, "%s: 1 to %d sections are supported, got %zu", api, kMaxRotaryAxes, n);
        int64_t end = 0;
        for (size_t i = 0; i < n; ++i) {
            OPSCV_REQUIRE(sections->v[i] >= 0 && sections->v[i] <= half, "%s: a section is a whole number of frequencies", api);
            end += sections->v[i];
            r.ends[i] = static_cast<int32_t>(end);
        }
        OPSCV_REQUIRE(end == half, "%s: the sections add up to %ld, not to the %ld frequencies", api, (long)end, (long)half);
        r.axes = static_cast<int32_t>(n);
    }
    OPSCV_REQUIRE(positions->dims.size() == lead + axesDim && (axesDim == 0 || positions->dims[0] == r.axes),
                  "%s: positions must be %s", api, axesDim != 0 ? "[sections, ...] with q's leading dimensions" : "q's leading dimensions");
    for (size_t i = 0; i < lead; ++i) {
        OPSCV_REQUIRE(positions->dims[axesDim + i] == q->dims[i], "%s: positions do not have q's leading dimensions", api);
    }
    const int64_t heads = q->dims[lead], kHeads = k != nullptr ? k->dims[lead] : 0;
    OPSCV_REQUIRE(Last(q) <= (1 << 20) && heads <= (1 << 20) && kHeads <= (1 << 20) && (heads + kHeads) * Last(q) <= (1 << 24),
                  "%s: a token of more than 2^24 values is not supported", api);
    OPSCV_REQUIRE(WritesApart(qOut) && (kOut == nullptr || WritesApart(kOut)), "%s: an output's elements overlap", api);
    OPSCV_TRY(CheckData(api, {q, k, positions, frequencies, qOut, kOut}));
    if (Numel(q) == 0 && (k == nullptr || Numel(k) == 0)) {
        return ACLNN_SUCCESS;
    }
    Operand oq = In(q), ok = In(k), oqo = Out(qOut), oko = Out(kOut);
    aclTensor pos = *positions;
    RotaryTensor tq, tk;
    Lead merged;
    auto addAll = [&](LeadMerge& m) {
        m.Add(&oq.view, 0, &tq.inTok);
        m.Add(&oqo.view, 0, &tq.outTok);
        if (k != nullptr) {
            m.Add(&ok.view, 0, &tk.inTok);
            m.Add(&oko.view, 0, &tk.outTok);
        }
        m.Add(&pos, axesDim, &r.posTok);
    };
    const auto all = {&oq, &ok, &oqo, &oko};
    // the views as they are; with copied positions; with copies of the others; with copies of all
    bool merges = MergesAsGiven(all, lead, addAll, merged);
    std::optional<PositionsCopy> copy;
    bool copies = false;
    if (!merges) {
        copy.emplace(positions, axesDim);
        if (!copy->Possible()) {
            copy.reset();
        }
    }
    if (copy) {
        pos = copy->View();
        merges = copies = MergesAsGiven(all, lead, addAll, merged);
        pos = copies ? pos : *positions;
    }
    OPSCV_TRY(Place(api, all, !merges, ex, ws));
    if (!merges) {
        LeadMerge asGiven(lead), withCopy(lead);
        addAll(asGiven);
        if (!asGiven.Run(merged)) {
            OPSCV_REQUIRE(copy, "%s: positions with more than two strided leading dimensions are not supported", api);
            copies = true;
            pos = copy->View();
            addAll(withCopy);
            withCopy.Run(merged); // contiguous tensors merge to one dimension, the copy to two
        }
    }
    r.posAxis = axesDim != 0 ? positions->strides[0] : 0;
    BufRef posBuf;
    posBuf.base = DataOf(positions, ElemSize(positions->dtype));
    if (copies) {
        posBuf = copy->Stage(ws, &ex, &r.posAxis);
    }
    r.tokens = merged.total;
    r.inner = merged.inner;
    r.dim = static_cast<int32_t>(Last(q));
    r.half = static_cast<int32_t>(half);
    r.interleaved = interleaved;
    r.inverse = inverse;
    r.freq64 = frequencies->dtype == ACL_DOUBLE;
    r.pos64 = positions->dtype == ACL_INT64;
    r.scale = static_cast<float>(scale);
    tq.heads = static_cast<int32_t>(heads);
    tq.inHead = oq.view.strides[lead];
    tq.outHead = oqo.view.strides[lead];
    if (k != nullptr) {
        tk.heads = static_cast<int32_t>(kHeads);
        tk.inHead = ok.view.strides[lead];
        tk.outHead = oko.view.strides[lead];
    }
    const void* freq = DataOf(frequencies, r.freq64 ? 8 : 4);
    const Dt dt = ToDt(q->dtype);
    const BufRef bq = oq.buf, bk = ok.buf, bqo = oqo.buf, bko = oko.buf;
    ex.steps.push_back([=](char* w, cudaStream_t s) {
        RotaryTensor a = tq, b = tk;
        a.in = bq.At(w);
        a.out = bqo.At(w);
        if (b.heads > 0) {
            b.in = bk.At(w);
            b.out = bko.At(w);
        }
        return RotaryTurn(dt, r, a, b, posBuf.At(w), freq, s);
    });
    Finish(all, ex);
    return ACLNN_SUCCESS;
}

// ---- attention ---------------------------------------------------------------------------------------------------------------
aclnnStatus CheckAttention(const char* api, const aclTensor* q, const aclTensor* k, const aclTensor* v, const aclTensor* qLengths,
                           const aclTensor* kvLengths, int64_t window, int64_t sinks, double scale, AttnShape& s)
{
    OPSCV_REQUIRE(DtypeSupported(q->dtype), "%s: dtype %s not supported (FLOAT, FLOAT16, BF16)", api, DtypeName(q->dtype));
    OPSCV_REQUIRE(k->dtype == q->dtype && v->dtype == q->dtype, "%s: q, k and v must have one type", api);
    OPSCV_REQUIRE(q->dims.size() == 4 && k->dims.size() == 4, "%s: q and k must be [batch, tokens, heads, dim]", api);
    OPSCV_REQUIRE(v->dims == k->dims, "%s: v must have k's shape", api);
    OPSCV_REQUIRE(k->dims[0] == q->dims[0] && k->dims[3] == q->dims[3], "%s: q and k must have one batch and one dim", api);
    OPSCV_REQUIRE(k->dims[2] >= 1 && q->dims[2] % k->dims[2] == 0, "%s: %ld heads are not a multiple of %ld key heads", api,
                  (long)q->dims[2], (long)k->dims[2]);
    OPSCV_REQUIRE(q->dims[3] >= 1 && q->dims[3] <= kMaxAttnDim, "%s: dim must be in [1, %d], got %ld", api, kMaxAttnDim,
                  (long)q->dims[3]);
    constexpr int64_t most = 1 << 30;
    OPSCV_REQUIRE(q->dims[1] <= most && k->dims[1] <= most && q->dims[0] <= most && q->dims[2] <= most &&
                      q->dims[0] * q->dims[2] <= most && k->dims[2] <= most && k->dims[0] * k->dims[2] <= most,
                  "%s: extents above 2^30 are not supported", api);
    // (query, head) pairs of a key head are counted in 32 bits where queries are few
    OPSCV_REQUIRE(q->dims[2] / k->dims[2] <= (1 << 24), "%s: more than 2^24 heads to a key head are not supported", api);
    for (const aclTensor* n : {qLengths, kvLengths}) {
        OPSCV_REQUIRE(n == nullptr || n->dtype == ACL_INT32 || n->dtype == ACL_INT64, "%s: lengths must be INT32 or INT64, got %s",
                      api, DtypeName(n->dtype));
        OPSCV_REQUIRE(n == nullptr || (n->dims.size() == 1 && n->dims[0] == q->dims[0] && Dense(n)),
                      "%s: lengths must be [batch] and contiguous", api);
    }
    OPSCV_REQUIRE(window >= 1, "%s: window must be at least 1, got %ld", api, (long)window);
    OPSCV_REQUIRE(sinks >= 0, "%s: sinks must not be negative, got %ld", api, (long)sinks);
    OPSCV_REQUIRE(Finite32(scale), "%s: scale must be finite in fp32", api);
    s.batch = static_cast<int32_t>(q->dims[0]);
    s.lq = static_cast<int32_t>(q->dims[1]);
    s.lk = static_cast<int32_t>(k->dims[1]);
    s.heads = static_cast<int32_t>(q->dims[2]);
    s.kvHeads = static_cast<int32_t>(k->dims[2]);
    s.dim = static_cast<int32_t>(q->dims[3]);
    s.window = static_cast<int32_t>(window < most ? window : most);
    s.sinks = static_cast<int32_t>(sinks < most ? sinks : most);
    s.scale = static_cast<float>(scale);
    if (qLengths != nullptr) {
        s.qLen64 = qLengths->dtype == ACL_INT64;
        s.qLen = DataOf(qLengths, s.qLen64 ? 8 : 4);
    }
    if (kvLengths != nullptr) {
        s.kvLen64 = kvLengths->dtype == ACL_INT64;
        s.kvLen = DataOf(kvLengths, s.kvLen64 ? 8 : 4);
    }
    return ACLNN_SUCCESS;
}

aclnnStatus CheckLse(const char* api, const aclTensor* q, const aclTensor* lse)
{
    OPSCV_REQUIRE(lse->dtype == ACL_FLOAT && Dense(lse) && lse->dims.size() == 3 && lse->dims[0] == q->dims[0] &&
                      lse->dims[1] == q->dims[2] && lse->dims[2] == q->dims[1],
                  "%s: lse must be [batch, heads, queries], FLOAT and contiguous", api);
    return ACLNN_SUCCESS;
}

AttnTensor AttnOf(const Operand& o, char* w)
{
    AttnTensor t;
    t.p = o.buf.At(w);
    t.b = o.view.strides[0];
    t.l = o.view.strides[1];
    t.h = o.view.strides[2];
    return t;
}

} // namespace

extern "C" {

aclnnStatus aclnnResidualRmsNormGetWorkspaceSize(const aclTensor* x, const aclTensor* residual, const aclTensor* weight,
                                                 double eps, aclTensor* y, aclTensor* sum, aclTensor* rstd,
                                                 uint64_t* workspaceSize, aclOpExecutor** executor)
{
    static const char* api = "aclnnResidualRmsNorm";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan& ws) -> aclnnStatus {
        OPSCV_NOT_NULL(x != nullptr && y != nullptr, api);
        OPSCV_TRY(CheckNorm(api, x, weight));
        OPSCV_TRY(CheckNormTensor(api, x, residual, "residual"));
        OPSCV_TRY(CheckNormTensor(api, x, y, "y"));
        OPSCV_TRY(CheckNormTensor(api, x, sum, "sum"));
        OPSCV_TRY(CheckPerRow(api, x, rstd, 0, "rstd"));
        OPSCV_REQUIRE(EpsOk(eps), "%s: eps must be finite in fp32 and not negative", api);
        OPSCV_REQUIRE(WritesApart(y) && (sum == nullptr || WritesApart(sum)), "%s: an output's elements overlap", api);
        OPSCV_TRY(CheckData(api, {x, residual, weight, y, sum, rstd}));
        if (Numel(x) == 0) {
            return ACLNN_SUCCESS;
        }
        NormShape n = ShapeOf(x, weight, eps);
        const size_t lead = x->dims.size() - 1;
        Operand ox = In(x), orr = In(residual), oy = Out(y), os = Out(sum);
        RowStride xs, rs, ys, ss;
        Lead merged;
        auto addAll = [&](LeadMerge& m) {
            m.Add(&ox.view, 0, &xs);
            m.Add(&oy.view, 0, &ys);
            if (residual != nullptr) {
                m.Add(&orr.view, 0, &rs);
            }
            if (sum != nullptr) {
                m.Add(&os.view, 0, &ss);
            }
        };
        const auto all = {&ox, &orr, &oy, &os};
        const bool merges = MergesAsGiven(all, lead, addAll, merged);
        OPSCV_TRY(Place(api, all, !merges, ex, ws));
        if (!merges) {
            LeadMerge m(lead);
            addAll(m);
            m.Run(merged); // contiguous tensors merge to one
        }
        n.rows = merged.total;
        n.inner = merged.inner;
        const BufRef bw = weight != nullptr ? StageInput(weight, ws, &ex) : BufRef{};
        const BufRef bx = ox.buf, br = orr.buf, by = oy.buf, bs = os.buf;
        const bool hasR = residual != nullptr, hasS = sum != nullptr, hasW = weight != nullptr;
        float* rstdAt = rstd != nullptr ? reinterpret_cast<float*>(DataOf(rstd, 4)) : nullptr;
        const Dt dt = ToDt(x->dtype);
        ex.steps.push_back([=](char* w, cudaStream_t s) {
            return RmsNormFwd(dt, n, bx.At(w), xs, hasR ? br.At(w) : nullptr, rs, hasW ? bw.At(w) : nullptr, by.At(w), ys,
                              hasS ? bs.At(w) : nullptr, ss, rstdAt, s);
        });
        Finish(all, ex);
        return ACLNN_SUCCESS;
    });
}

aclnnStatus aclnnResidualRmsNorm(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnResidualRmsNorm", workspace, workspaceSize, executor, stream);
}

aclnnStatus aclnnResidualRmsNormBackwardGetWorkspaceSize(const aclTensor* gradY, const aclTensor* sum, const aclTensor* rstd,
                                                         const aclTensor* weight, const aclTensor* gradSum, aclTensor* gradX,
                                                         aclTensor* gradWeight, uint64_t* workspaceSize,
                                                         aclOpExecutor** executor)
{
    static const char* api = "aclnnResidualRmsNormBackward";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan& ws) -> aclnnStatus {
        OPSCV_NOT_NULL(gradY != nullptr && sum != nullptr && rstd != nullptr && gradX != nullptr, api);
        OPSCV_TRY(CheckNorm(api, sum, weight));
        OPSCV_TRY(CheckNormTensor(api, sum, gradY, "gradY"));
        OPSCV_TRY(CheckNormTensor(api, sum, gradSum, "gradSum"));
        OPSCV_TRY(CheckNormTensor(api, sum, gradX, "gradX"));
        OPSCV_TRY(CheckPerRow(api, sum, rstd, 0, "rstd"));
        if (gradWeight != nullptr) {
            OPSCV_REQUIRE(weight != nullptr, "%s: gradWeight without a weight", api);
            OPSCV_REQUIRE(gradWeight->dtype == weight->dtype && gradWeight->dims == weight->dims && Dense(gradWeight),
                          "%s: gradWeight must be contiguous, of weight's type and shape", api);
        }
        OPSCV_REQUIRE(WritesApart(gradX), "%s: an output's elements overlap", api);
        OPSCV_TRY(CheckData(api, {gradY, sum, rstd, weight, gradSum, gradX, gradWeight}));
        NormShape n = ShapeOf(sum, weight, 0.0);
        const Dt dt = ToDt(sum->dtype);
        void* gwAt = gradWeight != nullptr ? DataOf(gradWeight, ElemSize(gradWeight->dtype)) : nullptr;
        if (Numel(sum) == 0) { // no rows
            if (gwAt != nullptr) {
                ex.steps.push_back([=](char*, cudaStream_t s) {
                    return RmsNormBwd(dt, n, nullptr, {}, nullptr, {}, nullptr, nullptr, nullptr, {}, nullptr, {}, gwAt, nullptr,
                                      0, s);
                });
            }
            return ACLNN_SUCCESS;
        }
        const size_t lead = sum->dims.size() - 1;
        Operand og = In(gradY), oz = In(sum), oa = In(gradSum), ox = Out(gradX);
        RowStride gs, ss, as, xs;
        Lead merged;
        auto addAll = [&](LeadMerge& m) {
            m.Add(&og.view, 0, &gs);
            m.Add(&oz.view, 0, &ss);
            if (gradSum != nullptr) {
                m.Add(&oa.view, 0, &as);
            }
            m.Add(&ox.view, 0, &xs);
        };
        const auto all = {&og, &oz, &oa, &ox};
        const bool merges = MergesAsGiven(all, lead, addAll, merged);
        OPSCV_TRY(Place(api, all, !merges, ex, ws));
        if (!merges) {
            LeadMerge m(lead);
            addAll(m);
            m.Run(merged);
        }
        n.rows = merged.total;
        n.inner = merged.inner;
        const BufRef bw = weight != nullptr ? StageInput(weight, ws, &ex) : BufRef{};
        const int64_t floats = RmsNormBwdScratch(dt, n, gradWeight != nullptr);
        const uint64_t scratchOff = ws.Alloc(static_cast<uint64_t>(floats) * 4);
        const BufRef bg = og.buf, bz = oz.buf, ba = oa.buf, bx = ox.buf;
        const bool hasA = gradSum != nullptr, hasW = weight != nullptr;
        const float* rstdAt = reinterpret_cast<const float*>(DataOf(rstd, 4));
        ex.steps.push_back([=](char* w, cudaStream_t s) {
            return RmsNormBwd(dt, n, bg.At(w), gs, bz.At(w), ss, rstdAt, hasW ? bw.At(w) : nullptr, hasA ? ba.At(w) : nullptr, as,
                              bx.At(w), xs, gwAt, reinterpret_cast<float*>(w + scratchOff), floats, s);
        });
        Finish(all, ex);
        return ACLNN_SUCCESS;
    });
}

aclnnStatus aclnnResidualRmsNormBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnResidualRmsNormBackward", workspace, workspaceSize, executor, stream);
}

aclnnStatus aclnnResidualRmsNormQuantGetWorkspaceSize(const aclTensor* x, const aclTensor* residual, const aclTensor* weight,
                                                      double eps, int64_t group, aclTensor* out, aclTensor* scales,
                                                      aclTensor* sum, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    static const char* api = "aclnnResidualRmsNormQuant";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan& ws) -> aclnnStatus {
        OPSCV_NOT_NULL(x != nullptr && out != nullptr && scales != nullptr, api);
        OPSCV_TRY(CheckNorm(api, x, weight));
        OPSCV_TRY(CheckNormTensor(api, x, residual, "residual"));
        OPSCV_TRY(CheckNormTensor(api, x, sum, "sum"));
        OPSCV_REQUIRE(EpsOk(eps), "%s: eps must be finite in fp32 and not negative", api);
        OPSCV_REQUIRE(group == 0 || (group >= 32 && group % 32 == 0), "%s: group must be 0 or a multiple of 32, got %ld", api,
                      (long)group);
        OPSCV_REQUIRE(out->dtype == ACL_FLOAT8_E4M3FN || out->dtype == ACL_INT8, "%s: out must be FLOAT8_E4M3FN or INT8, got %s",
                      api, DtypeName(out->dtype));
        OPSCV_REQUIRE(out->dims == x->dims && Dense(out), "%s: out must be contiguous and have x's shape", api);
        const int64_t width = Last(x);
        const int64_t groups = group == 0 ? 1 : (width + group - 1) / group;
        OPSCV_REQUIRE(groups <= 10240, "%s: more than 10240 groups a row are not supported", api);
        OPSCV_TRY(CheckPerRow(api, x, scales, groups, "scales"));
        OPSCV_REQUIRE(sum == nullptr || WritesApart(sum), "%s: an output's elements overlap", api);
        OPSCV_TRY(CheckData(api, {x, residual, weight, out, scales, sum}));
        if (Numel(x) == 0) {
            return ACLNN_SUCCESS;
        }
        NormShape n = ShapeOf(x, weight, eps);
        const size_t lead = x->dims.size() - 1;
        Operand ox = In(x), orr = In(residual), os = Out(sum);
        RowStride xs, rs, ss;
        Lead merged;
        auto addAll = [&](LeadMerge& m) {
            m.Add(&ox.view, 0, &xs);
            if (residual != nullptr) {
                m.Add(&orr.view, 0, &rs);
            }
            if (sum != nullptr) {
                m.Add(&os.view, 0, &ss);
            }
        };
        const auto all = {&ox, &orr, &os};
        const bool merges = MergesAsGiven(all, lead, addAll, merged);
        OPSCV_TRY(Place(api, all, !merges, ex, ws));
        if (!merges) {
            LeadMerge m(lead);
            addAll(m);
            m.Run(merged);
        }
        n.rows = merged.total;
        n.inner = merged.inner;
        const BufRef bw = weight != nullptr ? StageInput(weight, ws, &ex) : BufRef{};
        const BufRef bx = ox.buf, br = orr.buf, bs = os.buf;
        const bool hasR = residual != nullptr, hasS = sum != nullptr, hasW = weight != nullptr;
        void* q = DataOf(out, 1);
        float* sc = reinterpret_cast<float*>(DataOf(scales, 4));
        const Dt dt = ToDt(x->dtype);
        const Q8 type = out->dtype == ACL_INT8 ? Q8::INT8 : Q8::E4M3;
        const int32_t g = group >= width ? 0 : static_cast<int32_t>(group); // one group: a row's scale
        ex.steps.push_back([=](char* w, cudaStream_t s) {
            return RmsNormQuant(dt, n, bx.At(w), xs, hasR ? br.At(w) : nullptr, rs, hasW ? bw.At(w) : nullptr, type, g, q, sc,
                                hasS ? bs.At(w) : nullptr, ss, s);
        });
        Finish(all, ex);
        return ACLNN_SUCCESS;
    });
}

aclnnStatus aclnnResidualRmsNormQuant(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnResidualRmsNormQuant", workspace, workspaceSize, executor, stream);
}

aclnnStatus aclnnRotaryEmbeddingGetWorkspaceSize(const aclTensor* q, const aclTensor* k, const aclTensor* positions,
                                                 const aclTensor* frequencies, const aclIntArray* sections, bool interleaved,
                                                 double scale, aclTensor* qOut, aclTensor* kOut, uint64_t* workspaceSize,
                                                 aclOpExecutor** executor)
{
    static const char* api = "aclnnRotaryEmbedding";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan& ws) -> aclnnStatus {
        return PlanRotary(api, q, k, positions, frequencies, sections, interleaved, scale, false, qOut, kOut, ex, ws);
    });
}

aclnnStatus aclnnRotaryEmbedding(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnRotaryEmbedding", workspace, workspaceSize, executor, stream);
}

aclnnStatus aclnnRotaryEmbeddingBackwardGetWorkspaceSize(const aclTensor* gradQOut, const aclTensor* gradKOut,
                                                         const aclTensor* positions, const aclTensor* frequencies,
                                                         const aclIntArray* sections, bool interleaved, double scale,
                                                         aclTensor* gradQ, aclTensor* gradK, uint64_t* workspaceSize,
                                                         aclOpExecutor** executor)
{
    static const char* api = "aclnnRotaryEmbeddingBackward";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan& ws) -> aclnnStatus {
        return PlanRotary(api, gradQOut, gradKOut, positions, frequencies, sections, interleaved, scale, true, gradQ, gradK, ex,
                          ws);
    });
}

aclnnStatus aclnnRotaryEmbeddingBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnRotaryEmbeddingBackward", workspace, workspaceSize, executor, stream);
}

aclnnStatus aclnnRotaryFrequenciesGetWorkspaceSize(double base, int64_t scaling, double factor, double originalLength, double low,
                                                   double high, aclTensor* out, uint64_t* workspaceSize,
                                                   aclOpExecutor** executor)
{
    static const char* api = "aclnnRotaryFrequencies";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan&) -> aclnnStatus {
        OPSCV_NOT_NULL(out != nullptr, api);
        OPSCV_REQUIRE(std::isfinite(base) && base > 1.0, "%s: base must be above 1", api);
        OPSCV_REQUIRE(scaling >= 0 && scaling <= 4, "%s: scaling %ld should be in [0, 4]", api, (long)scaling);
        OPSCV_REQUIRE(std::isfinite(factor) && factor >= 1.0, "%s: factor must be at least 1", api);
        if (scaling >= 3) {
            OPSCV_REQUIRE(std::isfinite(originalLength) && originalLength > 0.0, "%s: originalLength must be above 0", api);
            OPSCV_REQUIRE(std::isfinite(low) && std::isfinite(high) && low < high && (scaling == 3 ? low >= 0.0 : low > 0.0),
                          "%s: low and high do not bound a range of turns", api);
        }
        OPSCV_REQUIRE(out->dtype == ACL_DOUBLE || out->dtype == ACL_FLOAT, "%s: out must be DOUBLE or FLOAT, got %s", api,
                      DtypeName(out->dtype));
        OPSCV_REQUIRE(out->dims.size() == 1 && Dense(out) && out->dims[0] <= (1 << 20),
                      "%s: out must be one contiguous dimension", api);
        const int32_t half = static_cast<int32_t>(out->dims[0]);
        OPSCV_TRY(CheckData(api, {out}));
        if (half == 0) {
            return ACLNN_SUCCESS;
        }
        const bool is64 = out->dtype == ACL_DOUBLE;
        void* at = DataOf(out, is64 ? 8 : 4);
        ex.steps.push_back([=](char*, cudaStream_t s) {
            return RotaryFrequencies(at, is64, half, base, static_cast<RotaryScaling>(scaling), factor, originalLength, low, high, s);
        });
        return ACLNN_SUCCESS;
    });
}

aclnnStatus aclnnRotaryFrequencies(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnRotaryFrequencies", workspace, workspaceSize, executor, stream);
}

aclnnStatus aclnnWindowAttentionGetWorkspaceSize(const aclTensor* q, const aclTensor* k, const aclTensor* v,
                                                 const aclTensor* qLengths, const aclTensor* kvLengths, int64_t window,
                                                 int64_t sinks, double scale, aclTensor* out, aclTensor* lse,
                                                 uint64_t* workspaceSize, aclOpExecutor** executor)
{
    static const char* api = "aclnnWindowAttention";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan& ws) -> aclnnStatus {
        OPSCV_NOT_NULL(q != nullptr && k != nullptr && v != nullptr && out != nullptr, api);
        AttnShape shape;
        OPSCV_TRY(CheckAttention(api, q, k, v, qLengths, kvLengths, window, sinks, scale, shape));
        OPSCV_REQUIRE(out->dtype == q->dtype && out->dims == q->dims, "%s: out must have q's type and shape", api);
        OPSCV_REQUIRE(WritesApart(out), "%s: an output's elements overlap", api);
        if (lse != nullptr) {
            OPSCV_TRY(CheckLse(api, q, lse));
        }
        OPSCV_TRY(CheckData(api, {q, k, v, qLengths, kvLengths, out, lse}));
        if (Numel(q) == 0) {
            return ACLNN_SUCCESS;
        }
        Operand oq = In(q), ok = In(k), ov = In(v), oo = Out(out);
        OPSCV_TRY(Place(api, {&oq, &ok, &ov, &oo}, false, ex, ws));
        const Dt dt = ToDt(q->dtype);
        float* lseAt = lse != nullptr ? reinterpret_cast<float*>(DataOf(lse, 4)) : nullptr;
        ex.steps.push_back([=](char* w, cudaStream_t s) {
            return WindowAttentionFwd(dt, shape, AttnOf(oq, w), AttnOf(ok, w), AttnOf(ov, w), AttnOf(oo, w), lseAt, s);
        });
        Finish({&oo}, ex);
        return ACLNN_SUCCESS;
    });
}

aclnnStatus aclnnWindowAttention(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnWindowAttention", workspace, workspaceSize, executor, stream);
}

aclnnStatus aclnnWindowAttentionBackwardGetWorkspaceSize(const aclTensor* gradOut, const aclTensor* q, const aclTensor* k,
                                                         const aclTensor* v, const aclTensor* out, const aclTensor* lse,
                                                         const aclTensor* qLengths, const aclTensor* kvLengths, int64_t window,
                                                         int64_t sinks, double scale, aclTensor* gradQ, aclTensor* gradK,
                                                         aclTensor* gradV, uint64_t* workspaceSize, aclOpExecutor** executor)
{
    static const char* api = "aclnnWindowAttentionBackward";
    return Guarded(api, workspaceSize, executor, [&](aclOpExecutor& ex, WsPlan& ws) -> aclnnStatus {
        OPSCV_NOT_NULL(gradOut != nullptr && q != nullptr && k != nullptr && v != nullptr && out != nullptr && lse != nullptr &&
                           gradQ != nullptr && gradK != nullptr && gradV != nullptr,
                       api);
        AttnShape shape;
        OPSCV_TRY(CheckAttention(api, q, k, v, qLengths, kvLengths, window, sinks, scale, shape));
        for (const aclTensor* t : {gradOut, out, static_cast<const aclTensor*>(gradQ)}) {
            OPSCV_REQUIRE(t->dtype == q->dtype && t->dims == q->dims, "%s: gradOut, out and gradQ must have q's type and shape", api);
        }
        for (const aclTensor* t : {gradK, gradV}) {
            OPSCV_REQUIRE(t->dtype == q->dtype && t->dims == k->dims, "%s: gradK and gradV must have k's type and shape", api);
        }
        OPSCV_TRY(CheckLse(api, q, lse));
        OPSCV_REQUIRE(WritesApart(gradQ) && WritesApart(gradK) && WritesApart(gradV), "%s: an output's elements overlap", api);
        OPSCV_TRY(CheckData(api, {gradOut, q, k, v, out, lse, qLengths, kvLengths, gradQ, gradK, gradV}));
        if (Numel(q) == 0 && Numel(k) == 0) {
            return ACLNN_SUCCESS;
        }
        Operand og = In(gradOut), oq = In(q), ok = In(k), ov = In(v), oo = In(out);
        Operand gq = Out(gradQ), gk = Out(gradK), gv = Out(gradV);
        OPSCV_TRY(Place(api, {&og, &oq, &ok, &ov, &oo, &gq, &gk, &gv}, false, ex, ws));
        const Dt dt = ToDt(q->dtype);
        const uint64_t own = ws.Alloc(WindowAttentionBwdWorkspace(dt, shape, AttnOf(og, nullptr), AttnOf(oq, nullptr), AttnOf(ok, nullptr),
                                                                  AttnOf(ov, nullptr)));
        const float* lseAt = reinterpret_cast<const float*>(DataOf(lse, 4));
        ex.steps.push_back([=](char* w, cudaStream_t s) {
            return WindowAttentionBwd(dt, shape, AttnOf(og, w), AttnOf(oq, w), AttnOf(ok, w), AttnOf(ov, w), AttnOf(oo, w), lseAt,
                                      AttnOf(gq, w), AttnOf(gk, w), AttnOf(gv, w), w + own, s);
        });
        Finish({&gq, &gk, &gv}, ex);
        return ACLNN_SUCCESS;
    });
}

aclnnStatus aclnnWindowAttentionBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream)
{
    return RunExecutor("aclnnWindowAttentionBackward", workspace, workspaceSize, executor, stream);
}

} // extern "C"
