// What the operators beside MatMulNBits share on the host: a call's tensors checked one by one, the node object with its scratch, creation and capability answers.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstring>
#include <initializer_list>
#include <limits>
#include <mutex>
#include <string>
#include <type_traits>
#include <vector>

#include "provider.h"

namespace nxrt_rocm {

constexpr uint32_t kMaxInputs = 14, kMaxOutputs = 14;

inline const char* dtype_name(uint32_t dt)
{
    switch (dt) {
        case NXRT_DT_FLOAT32: return "Float32";
        case NXRT_DT_UINT8: return "Uint8";
        case NXRT_DT_INT8: return "Int8";
        case NXRT_DT_INT32: return "Int32";
        case NXRT_DT_INT64: return "Int64";
        case NXRT_DT_FLOAT16: return "Float16";
        case NXRT_DT_BFLOAT16: return "BFloat16";
        case NXRT_DT_FLOAT8E4M3FN: return "Float8E4M3FN";
        default: return "another dtype";
    }
}

inline uint64_t item_size(uint32_t dt)
{
    switch (dt) {
        case NXRT_DT_INT64: return 8;
        case NXRT_DT_FLOAT32:
        case NXRT_DT_INT32: return 4;
        case NXRT_DT_UINT8:
        case NXRT_DT_INT8:
        case NXRT_DT_FLOAT8E4M3FN: return 1;
        default: return 2;
    }
}
inline bool is_float(uint32_t dt) { return dt == NXRT_DT_FLOAT32 || dt == NXRT_DT_FLOAT16 || dt == NXRT_DT_BFLOAT16; }

struct Dims {
    const uint64_t* at;
    uint32_t n;
};
inline std::string text(const Dims& d)
{
    std::string out = "[";
    for (uint32_t i = 0; i < d.n; ++i) out += (i ? ", " : "") + std::to_string(d.at[i]);
    return out + "]";
}
inline std::string text(const NxrtRocmTensorView& v) { return text(Dims{v.shape, v.ndim}); }
inline bool is_shape(const NxrtRocmTensorView& v, std::initializer_list<uint64_t> want)
{
    return v.ndim == want.size() && std::equal(want.begin(), want.end(), v.shape);
}

// The product of the first `dims` extents; false where one of them or the product is beyond what a tensor can have, so that nothing below overflows.
constexpr uint64_t kMaxExtent = uint64_t{1} << 40;
inline bool elements_of(const NxrtRocmTensorView& v, uint32_t dims, uint64_t* out)
{
    uint64_t n = 1;
    for (uint32_t i = 0; i < dims; ++i) {
        if (v.shape[i] >= (uint64_t{1} << 31)) return false;
        n *= v.shape[i];
        if (n > kMaxExtent) return false;
    }
    *out = n;
    return true;
}

inline bool contiguous(const NxrtRocmTensorView& v)
{
    if (!v.strides) return true;
    uint64_t expect = 1;
    for (int i = static_cast<int>(v.ndim) - 1; i >= 0; --i) {
        if (v.shape[i] != 1 && static_cast<uint64_t>(v.strides[i]) != expect) return false;
        expect *= v.shape[i];
    }
    return true;
}

// A call whose first tensor has no rows has nothing to do, and none of its tensors needs memory behind it.
inline bool no_rows(const NxrtRocmTensorView* in, uint32_t n_in)
{
    if (!in || n_in < 1 || !in[0].shape) return false;
    for (uint32_t d = 0; d + 1 < in[0].ndim; ++d)
        if (in[0].shape[d] == 0) return true;
    return false;
}

inline uint8_t* at(const NxrtRocmTensorView& v) { return static_cast<uint8_t*>(v.data) + v.byte_offset; }

// One call's tensors, checked as they are asked for; the first thing that is wrong stays. Nothing is allocated where nothing is wrong: a short call
// takes less time on the GPU than a few dozen allocations here.
class Call {
public:
    Call(const char* op, const NxrtRocmEp& ep, const NxrtRocmTensorView* in, uint32_t n_in, const NxrtRocmTensorView* out, uint32_t n_out) : op_(op), ep_(ep), in_{in, n_in}, out_{out, n_out}
    {
        if ((n_in && !in) || (n_out && !out)) fail("null tensor view array");
    }
    bool failed() const { return failed_; }
    NxrtStatus status() const { return failed_ ? make_status(NXRT_INVALID_ARGUMENT, message_) : ok(); }
    void fail(const std::string& m)
    {
        if (!failed_) message_ = std::string(op_) + ": " + m;
        failed_ = true;
    }
    void arity(uint32_t least, uint32_t most, uint32_t out_most)
    {
        if (in_.n < least || in_.n > most) fail("expected " + std::to_string(least) + "..=" + std::to_string(most) + " inputs, got " + std::to_string(in_.n));
        if (out_.n < 1 || out_.n > out_most) fail("expected 1..=" + std::to_string(out_most) + " outputs, got " + std::to_string(out_.n));
    }
    const NxrtRocmTensorView* input(uint32_t i, const char* name) { return take(in_, i, name, inputs_, n_inputs_); }
    const NxrtRocmTensorView* output(uint32_t i, const char* name) { return take(out_, i, name, outputs_, n_outputs_); }
    const NxrtRocmTensorView* required(const NxrtRocmTensorView* v, const char* name)
    {
        if (!v) fail(std::string(name) + " is required and absent");
        return v;
    }
    void dtype(const NxrtRocmTensorView* v, const char* name, std::initializer_list<uint32_t> allowed)
    {
        if (!v || failed_) return;
        for (uint32_t dt : allowed)
            if (v->dtype == dt) return;
        std::string names;
        for (uint32_t dt : allowed) names += (names.empty() ? "" : " or ") + std::string(dtype_name(dt));
        fail(std::string(name) + " must have dtype " + names + ", got " + dtype_name(v->dtype));
    }
    void shape(const NxrtRocmTensorView* v, const char* name, std::initializer_list<uint64_t> want)
    {
        if (v && !failed_ && !is_shape(*v, want)) fail(std::string(name) + " must have shape " + text(Dims{want.begin(), static_cast<uint32_t>(want.size())}) + ", got " + text(*v));
    }
    // the dims of `like`, but for the last one
    bool is_like(const NxrtRocmTensorView& v, const NxrtRocmTensorView& like, uint64_t last) const
    {
        return v.ndim == like.ndim && std::equal(v.shape, v.shape + v.ndim - 1, like.shape) && v.shape[v.ndim - 1] == last;
    }
    void shape_like(const NxrtRocmTensorView* v, const char* name, const NxrtRocmTensorView* like, uint64_t last)
    {
        if (!v || !like || failed_ || is_like(*v, *like, last)) return;
        std::vector<uint64_t> want(like->shape, like->shape + like->ndim);
        want.back() = last;
        fail(std::string(name) + " must have shape " + text(Dims{want.data(), like->ndim}) + ", got " + text(*v));
    }
    void one_per_row(const NxrtRocmTensorView* v, const char* name, uint64_t rows)
    {
        uint64_t count = 0;
        if (v && !failed_ && (!elements_of(*v, v->ndim, &count) || count != rows)) fail(std::string(name) + " must have one element for each of the " + std::to_string(rows) + " rows, got " + text(*v));
    }
    // rank >= 1: the leading dims multiplied, and the last one
    void matrix(const NxrtRocmTensorView* v, const char* name, uint64_t* rows, uint64_t* last)
    {
        if (!v || failed_) return;
        if (v->ndim == 0) return fail(std::string(name) + " must have rank >= 1");
        uint64_t all = 0;
        if (!elements_of(*v, v->ndim, &all) || !elements_of(*v, v->ndim - 1, rows)) return fail(std::string(name) + " is too large: " + text(*v));
        *last = v->shape[v->ndim - 1];
    }
    // Outputs may not overlap inputs, but for output o on input i where `may(o, i)`, both begin at one address and have one type.
    template <typename F>
    void check_overlap(F may)
    {
        auto bytes = [](const Named& t) {
            uint64_t n = 0;
            return elements_of(*t.v, t.v->ndim, &n) ? n * item_size(t.v->dtype) : uint64_t{0};
        };
        auto meet = [&](const Named& a, const Named& b) { return at(*a.v) < at(*b.v) + bytes(b) && at(*b.v) < at(*a.v) + bytes(a); };
        for (uint32_t o = 0; o < n_outputs_ && !failed_; ++o) {
            const Named& out = outputs_[o];
            for (uint32_t i = 0; i < n_inputs_; ++i) {
                const Named& in = inputs_[i];
                if (meet(out, in) && !(may(out.index, in.index) && at(*out.v) == at(*in.v) && out.v->dtype == in.v->dtype)) return fail(std::string(out.name) + " overlaps " + in.name);
            }
            for (uint32_t q = 0; q < o; ++q)
                if (meet(out, outputs_[q])) return fail(std::string(out.name) + " overlaps " + outputs_[q].name);
        }
    }
    void check_overlap()
    {
        check_overlap([](uint32_t, uint32_t) { return false; });
    }
    // state that a call changes where it is: an input and an output that are one tensor
    void in_place(const NxrtRocmTensorView* in, const NxrtRocmTensorView* out, const char* name)
    {
        if (failed_ || !in || !out) return;
        if (at(*in) != at(*out) || in->dtype != out->dtype || in->ndim != out->ndim || !std::equal(in->shape, in->shape + in->ndim, out->shape))
            fail(std::string(name) + " is changed where it is: the output must be the input's tensor");
    }

private:
    struct Views {
        const NxrtRocmTensorView* at;
        uint32_t n;
    };
    struct Named {
        const char* name;
        uint32_t index;
        const NxrtRocmTensorView* v;
    };
    const NxrtRocmTensorView* take(const Views& views, uint32_t i, const char* name, Named* seen, uint32_t& count)
    {
        if (failed_ || i >= views.n || !views.at[i].data) return nullptr;
        const NxrtRocmTensorView& v = views.at[i];
        uint64_t all = 0;
        if (v.ndim && !v.shape) fail(std::string(name) + " has a null shape");
        else if (!elements_of(v, v.ndim, &all)) fail(std::string(name) + " is too large: " + text(v));
        else if (!contiguous(v)) fail(std::string(name) + " must be contiguous on the ROCm execution provider");
        else if (v.device_type != NXRT_DEVICE_ROCM || v.device_index != ep_.device)
            fail(std::string(name) + " must live on ROCm device " + std::to_string(ep_.device) + " (allocate it with this provider and copy the data in)");
        else if (reinterpret_cast<uintptr_t>(at(v)) % item_size(v.dtype) != 0) fail(std::string(name) + " is not aligned to its elements");
        else seen[count++] = Named{name, i, &v};
        return failed_ ? nullptr : &v;
    }
    const char* op_;
    const NxrtRocmEp& ep_;
    const Views in_, out_;
    Named inputs_[2 * kMaxInputs], outputs_[kMaxOutputs];         // (an input may be asked for twice)
    uint32_t n_inputs_ = 0, n_outputs_ = 0;
    bool failed_ = false;
    std::string message_;
};

}  // namespace nxrt_rocm

using nxrt_rocm::hip_status;
using nxrt_rocm::make_status;
using nxrt_rocm::ok;

struct NxrtRocmNode {
    NxrtRocmEp* ep;
    std::mutex mu;                         // one call at a time: scratch, copies and variant are per node
    const char* variant = "none";
    void* scratch = nullptr;
    uint64_t scratch_bytes = 0;
    std::vector<void*> retired;            // outgrown scratch that a recorded graph may still name

    explicit NxrtRocmNode(NxrtRocmEp* provider) : ep(provider) { ep->retain(); }
    NxrtRocmNode(const NxrtRocmNode&) = delete;
    NxrtRocmNode& operator=(const NxrtRocmNode&) = delete;
    virtual ~NxrtRocmNode()
    {
        if ((scratch || !retired.empty()) && ep->bind().code == NXRT_OK) {
            rocm_ffi_stream_sync(ep->stream);
            if (scratch) rocm_ffi_free(scratch);
            for (void* old : retired) rocm_ffi_free(old);
        }
        nxrt_rocm_ep_release(ep);
    }
    virtual const char* op() const = 0;
    virtual NxrtStatus workspace(const NxrtTensorDesc* in, uint32_t n, uint64_t* bytes) const = 0;
    virtual NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void* ws, uint64_t ws_bytes) = 0;

    std::string err(const std::string& m) const { return std::string(op()) + ": " + m; }

    // Once the provider has recorded a graph, one may name the scratch, and it stays until the node is released. Before that it is freed when the stream has drained: a
    // host whose prompts grow holds one scratch a node, not one a length.
    void drop_scratch()
    {
        if (!scratch) return;
        if (ep->captures.load() != 0) {
            retired.push_back(scratch);
        } else {
            rocm_ffi_stream_sync(ep->stream);
            rocm_ffi_free(scratch);
        }
        scratch = nullptr;
        scratch_bytes = 0;
    }

    // `need` bytes for this call: the caller's, or the node's own, grown where that may be.
    NxrtStatus find_scratch(uint64_t need, void* ws, uint64_t ws_bytes, void** out)
    {
        *out = nullptr;
        if (need == 0) return ok();
        if (ws) {
            if (ws_bytes < need) return make_status(NXRT_INVALID_ARGUMENT, err("workspace of " + std::to_string(ws_bytes) + " bytes is smaller than the required " + std::to_string(need)));
            if (reinterpret_cast<uintptr_t>(ws) % 256 != 0) return make_status(NXRT_INVALID_ARGUMENT, err("workspace must be aligned to 256 bytes"));
            *out = ws;
            return ok();
        }
        if (scratch_bytes < need) {
            if (ep->capturing)
                return make_status(NXRT_INVALID_ARGUMENT, err("a call under graph capture needs a workspace, or one eager call of this height first (nothing is allocated while a capture is open)"));
            void* fresh = nullptr;
            const int e = rocm_ffi_malloc(&fresh, need);
            if (e != 0) return hip_status(e, "workspace hipMalloc");
            drop_scratch();
            scratch = fresh;
            scratch_bytes = need;
        }
        *out = scratch;
        return ok();
    }
    NxrtStatus launched(int rc) const { return hip_status(rc, (std::string(op()) + ": kernel launch").c_str()); }
};

namespace nxrt_rocm {

// A static [.., last] input's rows and last extent; false where a dimension is dynamic or the shape is missing.
inline bool static_matrix(const NxrtTensorDesc* in, uint32_t n, uint32_t i, int64_t* rows, int64_t* last)
{
    if (!in || i >= n || in[i].ndim < 1 || !in[i].dims) return false;
    *rows = 1;
    for (uint32_t d = 0; d < in[i].ndim; ++d) {
        if (in[i].dims[d] < 0 || in[i].dims[d] > (int64_t{1} << 31)) return false;
        if (d + 1 < in[i].ndim) *rows *= in[i].dims[d];
        if (*rows > (int64_t{1} << 31)) return false;
    }
    *last = in[i].dims[in[i].ndim - 1];
    return true;
}

inline int decline(const std::string& why, char* reason, size_t reason_len)
{
    if (reason && reason_len) {
        const size_t n = why.size() < reason_len - 1 ? why.size() : reason_len - 1;
        std::memcpy(reason, why.data(), n);
        reason[n] = 0;
    }
    return 0;
}

// What a shorter, older struct of the caller's lacks reads as absent.
template <typename A>
A read_attrs(const A* attrs)
{
    A a;
    std::memset(&a, 0, sizeof(a));
    std::memcpy(&a, attrs, attrs->struct_size < sizeof(A) ? attrs->struct_size : sizeof(A));
    return a;
}
#define NODE_ATTR_PRESENT(a, bit, member) ((a.present & (1u << (bit))) && a.struct_size >= offsetof(std::remove_reference_t<decltype(a)>, member) + sizeof(a.member))

template <typename Node, typename F>
NxrtStatus create_node(const char* op, NxrtRocmEp* ep, NxrtRocmNode** out, F settings)
{
    return fenced([&]() -> NxrtStatus {
        if (!out) return make_status(NXRT_INVALID_ARGUMENT, std::string(op) + ": null out_node");
        *out = nullptr;
        const auto s = settings();
        if (!s.problem.empty()) return make_status(NXRT_INVALID_ARGUMENT, std::string(op) + ": " + s.problem);
        if (!ep) return make_status(NXRT_INVALID_ARGUMENT, std::string(op) + ": null provider");
        *out = new Node(ep, s);
        return ok();
    });
}

template <typename F>
int supported(const char* op, char* reason, size_t reason_len, F&& problem) noexcept
{
    if (reason && reason_len) reason[0] = 0;
    try {
        const std::string why = problem();
        return why.empty() ? 1 : decline(std::string(op) + ": " + why, reason, reason_len);
    } catch (...) {
        return 0;
    }
}
inline std::string arity(uint32_t n, uint32_t least, uint32_t most)
{
    return n < least || n > most ? "expected " + std::to_string(least) + "..=" + std::to_string(most) + " inputs, got " + std::to_string(n) : std::string();
}

}  // namespace nxrt_rocm
