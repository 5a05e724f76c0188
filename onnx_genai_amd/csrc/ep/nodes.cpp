// The operators beside MatMulNBits (QMoE, MatMulInt8, GatedResidualNorm): attributes, input checks, scratch and the C entry points.
#include "nodes.h"

using namespace nxrt_rocm;

namespace {

// ---- GatedResidualNorm -----------------------------------------------------------------------------------------------

struct GatedNormSettings {
    float epsilon = 1e-5f, residual_scale = 1.f, block_scale = 1.f;
    int layer = 0;
    std::string problem;
};
GatedNormSettings settings_of(const NxrtRocmGatedResidualNormAttrs* attrs)
{
    GatedNormSettings s;
    if (!attrs) {
        s.problem = "null attributes";
        return s;
    }
    const auto a = read_attrs(attrs);
    if (NODE_ATTR_PRESENT(a, 0, epsilon)) s.epsilon = static_cast<float>(a.epsilon);
    if (NODE_ATTR_PRESENT(a, 1, residual_scale)) s.residual_scale = static_cast<float>(a.residual_scale);
    if (NODE_ATTR_PRESENT(a, 2, block_scale)) s.block_scale = static_cast<float>(a.block_scale);
    if (NODE_ATTR_PRESENT(a, 3, layer_norm)) {
        if (a.layer_norm != 0 && a.layer_norm != 1) s.problem = "layer_norm must be 0 or 1, got " + std::to_string(a.layer_norm);
        s.layer = a.layer_norm == 1;
    }
    if (!(s.epsilon >= 0.f) || !std::isfinite(s.epsilon)) s.problem = "epsilon must be finite and not negative";
    if (!std::isfinite(s.residual_scale) || !std::isfinite(s.block_scale)) s.problem = "residual_scale and block_scale must be finite";
    return s;
}

struct GatedNormNode final : NxrtRocmNode {
    GatedNormSettings s;
    GatedNormNode(NxrtRocmEp* provider, const GatedNormSettings& settings) : NxrtRocmNode(provider), s(settings) {}
    const char* op() const override { return "GatedResidualNorm"; }
    NxrtStatus workspace(const NxrtTensorDesc*, uint32_t, uint64_t* bytes) const override
    {
        *bytes = 0;
        return ok();
    }
    NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void*, uint64_t) override
    {
        Call c(op(), *ep, in, n_in, out, n_out);
        c.arity(1, 7, 3);
        if (!c.failed() && no_rows(in, n_in)) return ok();
        const auto* residual = c.required(c.input(0, "residual"), "residual");
        c.dtype(residual, "residual", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        uint64_t rows = 0, h = 0;
        c.matrix(residual, "residual", &rows, &h);
        if (!c.failed() && (h == 0 || h > ROCM_GATED_NORM_MAX_HIDDEN)) c.fail("the last dimension must be 1..=" + std::to_string(ROCM_GATED_NORM_MAX_HIDDEN) + ", got " + std::to_string(h));
        if (!c.failed() && rows > 0x7fffffff) c.fail("too many rows: " + std::to_string(rows));
        if (c.failed()) return c.status();
        const uint32_t dt = residual->dtype;
        RocmGatedNormArgs a{};
        const auto* block = c.input(1, "block");
        c.dtype(block, "block", {dt});
        c.shape_like(block, "block", residual, h);
        auto weight = [&](uint32_t i, const char* name, const void*& to, int& to_dtype) {
            const auto* v = c.input(i, name);
            if (dt == NXRT_DT_FLOAT32) c.dtype(v, name, {NXRT_DT_FLOAT32});
            else c.dtype(v, name, {dt, NXRT_DT_FLOAT32});
            to = v ? at(*v) : nullptr;
            to_dtype = v ? static_cast<int>(v->dtype) : ROCM_DT_F32;
            return v;
        };
        const auto* post = weight(2, "post_gamma", a.post_gamma, a.post_gamma_dtype);
        c.shape(post, "post_gamma", {h});
        const auto* gate = weight(3, "gate", a.gate, a.gate_dtype);
        c.shape(weight(4, "pre_gamma", a.pre_gamma, a.pre_gamma_dtype), "pre_gamma", {h});
        c.shape(weight(5, "pre_beta", a.pre_beta, a.pre_beta_dtype), "pre_beta", {h});
        const auto* post_beta = weight(6, "post_beta", a.post_beta, a.post_beta_dtype);
        c.shape(post_beta, "post_beta", {h});
        if (!c.failed() && !block && (post || gate || post_beta)) c.fail("post_gamma, gate and post_beta need a block");
        if (!c.failed() && post_beta && !post) c.fail("post_beta needs a post_gamma");
        uint64_t gates = 1;
        if (gate && !c.failed() && !is_shape(*gate, {h})) {
            if (gate->ndim != 2 || gate->shape[1] != h || gate->shape[0] == 0 || rows % gate->shape[0] != 0)
                c.fail("gate must have shape [" + std::to_string(h) + "] or [G, " + std::to_string(h) + "] with G dividing the " + std::to_string(rows) + " rows, got " + text(*gate));
            else gates = gate->shape[0];
        }
        const auto* z = c.output(0, "Z");
        c.dtype(z, "Z", {dt});
        c.shape_like(z, "Z", residual, h);
        const auto* n = c.output(1, "N");
        c.dtype(n, "N", {dt, NXRT_DT_INT8});
        c.shape_like(n, "N", residual, h);
        const auto* scale = c.output(2, "n_scale");
        c.dtype(scale, "n_scale", {NXRT_DT_FLOAT32});
        if (!c.failed() && !z && !n) c.fail("neither Z nor N is asked for");
        const bool codes = n && n->dtype == NXRT_DT_INT8;
        if (!c.failed() && codes != (scale != nullptr)) c.fail("n_scale goes with Int8 N, and only with it");
        c.one_per_row(scale, "n_scale", rows);
        // a thread reads its elements of a row before it writes any of them, and no other row's
        c.check_overlap([](uint32_t o, uint32_t i) { return o <= 1 && i <= 1; });
        if (c.failed()) return c.status();
        a.residual = at(*residual);
        a.block = block ? at(*block) : nullptr;
        a.z = z ? at(*z) : nullptr;
        a.n = n ? at(*n) : nullptr;
        a.n_scale = scale ? reinterpret_cast<float*>(at(*scale)) : nullptr;
        a.rows = static_cast<int64_t>(rows);
        a.hidden = static_cast<int64_t>(h);
        a.rows_per_gate = static_cast<int64_t>(rows / gates);
        a.dtype = static_cast<int>(dt);
        a.post = post != nullptr;
        a.layer = s.layer;
        a.epsilon = s.epsilon;
        a.residual_scale = s.residual_scale;
        a.block_scale = s.block_scale;
        variant = codes ? "gated_norm_codes" : "gated_norm";
        NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        ep->launches.fetch_add(1);
        return launched(rocm_launch_gated_norm(&a, ep->stream));
    }
};

// ---- MatMulInt8 --------------------------------------------------------------------------------------------------------

struct Int8Settings {
    int64_t k = 0, n = 0;
    std::string problem;
};
Int8Settings settings_of(const NxrtRocmMatMulInt8Attrs* attrs)
{
    Int8Settings s;
    if (!attrs) {
        s.problem = "null attributes";
        return s;
    }
    const auto a = read_attrs(attrs);
    if (!NODE_ATTR_PRESENT(a, 0, K)) s.problem = "missing required integer attribute 'K'";
    else if (!NODE_ATTR_PRESENT(a, 1, N)) s.problem = "missing required integer attribute 'N'";
    else if (a.K <= 0 || a.K >= ROCM_INT8_MAX_K) s.problem = "attribute 'K' must be 1..=" + std::to_string(ROCM_INT8_MAX_K - 1) + " (an int32 holds every sum then), got " + std::to_string(a.K);
    else if (a.N <= 0 || a.N > (int64_t{1} << 30)) s.problem = "attribute 'N' must be 1..=2^30, got " + std::to_string(a.N);
    s.k = a.K;
    s.n = a.N;
    return s;
}

struct Int8Node final : NxrtRocmNode {
    Int8Settings s;
    Int8Node(NxrtRocmEp* provider, const Int8Settings& settings) : NxrtRocmNode(provider), s(settings) {}
    const char* op() const override { return "MatMulInt8"; }
    int64_t kp() const { return (s.k + 127) / 128 * 128; }

    // What a call keeps while it runs: codes, their scales, B in padded rows, sums of slices of K.
    struct Layout {
        uint64_t codes = 0, scales = 0, b = 0, partial = 0, partial_bytes = 0, total = 0;
    };
    Layout layout(int64_t rows, uint32_t a_dtype, bool pads_codes) const
    {
        Layout l;
        auto part = [&](uint64_t bytes) {
            const uint64_t here = l.total;
            l.total += (bytes + 255) / 256 * 256;
            return here;
        };
        RocmInt8Args a{};
        a.m = rows;
        a.n = s.n;
        a.k = s.k;
        a.a_dtype = static_cast<int>(a_dtype);
        const bool makes_codes = a_dtype != NXRT_DT_INT8 && !rocm_int8_fuses_quantizer(&a);
        l.codes = part(makes_codes || pads_codes ? static_cast<uint64_t>(rows * kp()) : 0);
        l.scales = part(makes_codes ? static_cast<uint64_t>(rows) * 4 : 0);
        l.b = part(rocm_int8_pads_b(&a) ? static_cast<uint64_t>(s.n * kp()) : 0);
        l.partial_bytes = rocm_int8_scratch_bytes(&a);
        l.partial = part(l.partial_bytes);
        return l;
    }
    NxrtStatus workspace(const NxrtTensorDesc* in, uint32_t n, uint64_t* bytes) const override
    {
        int64_t rows = 0, last = 0;
        if (!static_matrix(in, n, 0, &rows, &last)) return make_status(NXRT_INVALID_ARGUMENT, err("workspace_requirement needs the shape of A"));
        const NxrtStatus st = ep->bind();          // (the plan goes by the GPU's CUs)
        if (st.code != NXRT_OK) return st;
        *bytes = rows ? layout(rows, in[0].dtype, in[0].dtype == NXRT_DT_INT8).total : 0;
        return ok();
    }
    NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void* ws, uint64_t ws_bytes) override
    {
        Call c(op(), *ep, in, n_in, out, n_out);
        c.arity(3, 5, 1);
        if (!c.failed() && no_rows(in, n_in)) return ok();
        const auto* a = c.required(c.input(0, "A"), "A");
        c.dtype(a, "A", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16, NXRT_DT_INT8});
        uint64_t rows = 0, last = 0;
        c.matrix(a, "A", &rows, &last);
        const uint64_t k = static_cast<uint64_t>(s.k), n = static_cast<uint64_t>(s.n);
        if (!c.failed() && last != k) c.fail("A must have last dimension K=" + std::to_string(k) + ", got " + text(*a));
        if (!c.failed() && (rows > 0x7fffffff || rows * n > kMaxExtent)) c.fail("too many rows: " + std::to_string(rows));
        const auto* b = c.required(c.input(1, "B"), "B");
        c.dtype(b, "B", {NXRT_DT_INT8});
        c.shape(b, "B", {n, k});
        if (!c.failed() && k % 16 == 0 && reinterpret_cast<uintptr_t>(at(*b)) % 16 != 0) c.fail("B must start at a multiple of 16 bytes where K is a multiple of 16");
        const auto* sb = c.required(c.input(2, "b_scale"), "b_scale");
        c.dtype(sb, "b_scale", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        c.shape(sb, "b_scale", {n});
        const auto* sa = c.input(3, "a_scale");
        c.dtype(sa, "a_scale", {NXRT_DT_FLOAT32});
        const bool codes = a && a->dtype == NXRT_DT_INT8;
        if (!c.failed() && codes != (sa != nullptr)) c.fail("a_scale goes with Int8 A, and only with it");
        c.one_per_row(sa, "a_scale", rows);
        const auto* bias = c.input(4, "bias");
        c.dtype(bias, "bias", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        const bool per_row = bias && !c.failed() && !is_shape(*bias, {n});
        if (per_row) c.shape_like(bias, "bias", a, n);
        const auto* y = c.required(c.output(0, "Y"), "Y");
        c.dtype(y, "Y", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        c.shape_like(y, "Y", a, n);
        c.check_overlap();
        if (c.failed()) return c.status();

        NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        const bool pads_codes = codes && (s.k % 128 != 0 || reinterpret_cast<uintptr_t>(at(*a)) % 16 != 0);
        const Layout l = layout(static_cast<int64_t>(rows), a->dtype, pads_codes);
        void* scratch_at = nullptr;
        st = find_scratch(l.total, ws, ws_bytes, &scratch_at);
        if (st.code != NXRT_OK) return st;
        uint8_t* const w = static_cast<uint8_t*>(scratch_at);

        RocmInt8Args args{};
        args.m = static_cast<int64_t>(rows);
        args.n = s.n;
        args.k = s.k;
        args.b = reinterpret_cast<const int8_t*>(at(*b));
        args.ldb = s.k;
        int rc = 0;
        if (rocm_int8_pads_b(&args)) {
            rc = rocm_launch_pad_codes(args.b, s.n, s.k, reinterpret_cast<int8_t*>(w + l.b), ep->stream);
            args.b = reinterpret_cast<const int8_t*>(w + l.b);
            args.ldb = kp();
        }
        args.lda = kp();
        args.a_dtype = static_cast<int>(a->dtype);
        if (codes) {
            args.a = reinterpret_cast<const int8_t*>(at(*a));
            args.a_scale = reinterpret_cast<const float*>(at(*sa));
            if (pads_codes) {
                if (rc == 0) rc = rocm_launch_pad_codes(args.a, args.m, s.k, reinterpret_cast<int8_t*>(w + l.codes), ep->stream);
                args.a = reinterpret_cast<const int8_t*>(w + l.codes);
            }
        } else if (rocm_int8_fuses_quantizer(&args)) {
            args.a_float = at(*a);
        } else {
            if (rc == 0) rc = rocm_launch_quantize_rows(at(*a), static_cast<int>(a->dtype), args.m, s.k, reinterpret_cast<int8_t*>(w + l.codes), reinterpret_cast<float*>(w + l.scales), ep->stream);
            args.a = reinterpret_cast<const int8_t*>(w + l.codes);
            args.a_scale = reinterpret_cast<const float*>(w + l.scales);
        }
        args.b_scale = at(*sb);
        args.b_scale_dtype = static_cast<int>(sb->dtype);
        args.bias = bias ? at(*bias) : nullptr;
        args.bias_dtype = bias ? static_cast<int>(bias->dtype) | (per_row ? ROCM_BIAS_PER_ROW : 0) : ROCM_DT_F32;
        args.y = at(*y);
        args.y_dtype = static_cast<int>(y->dtype);
        args.partial = l.partial_bytes ? reinterpret_cast<int32_t*>(w + l.partial) : nullptr;
        variant = rocm_int8_variant(&args);
        ep->launches.fetch_add(1);
        if (rc == 0) rc = rocm_launch_int8(&args, ep->stream);
        return launched(rc);
    }
};

// ---- QMoE --------------------------------------------------------------------------------------------------------------

struct MoeSettings {
    int64_t k = 1, block_size = 0, normalize = 0, fusion = 0;
    float alpha = 1.f, beta = 0.f, limit = std::numeric_limits<float>::infinity();
    std::string problem;
};
MoeSettings settings_of(const NxrtRocmQMoEAttrs* attrs)
{
    MoeSettings s;
    if (!attrs) {
        s.problem = "null attributes";
        return s;
    }
    const auto a = read_attrs(attrs);
    if (NODE_ATTR_PRESENT(a, 0, k)) s.k = a.k;
    if (NODE_ATTR_PRESENT(a, 1, block_size)) s.block_size = a.block_size;
    const int64_t bits = NODE_ATTR_PRESENT(a, 2, expert_weight_bits) ? a.expert_weight_bits : 4;
    if (NODE_ATTR_PRESENT(a, 3, normalize_routing_weights)) s.normalize = a.normalize_routing_weights;
    if (NODE_ATTR_PRESENT(a, 4, swiglu_fusion)) s.fusion = a.swiglu_fusion;
    if (NODE_ATTR_PRESENT(a, 5, activation_alpha)) s.alpha = static_cast<float>(a.activation_alpha);
    if (NODE_ATTR_PRESENT(a, 6, activation_beta)) s.beta = static_cast<float>(a.activation_beta);
    if (NODE_ATTR_PRESENT(a, 7, swiglu_limit)) s.limit = static_cast<float>(a.swiglu_limit);
    if (s.k < 1 || s.k > ROCM_MOE_MAX_CHOICES) s.problem = "attribute 'k' must be 1..=" + std::to_string(ROCM_MOE_MAX_CHOICES) + ", got " + std::to_string(s.k);
    else if (!NODE_ATTR_PRESENT(a, 1, block_size)) s.problem = "missing required integer attribute 'block_size'";
    else if (s.block_size < 32 || s.block_size > (int64_t{1} << 20) || (s.block_size & (s.block_size - 1)) != 0) s.problem = "block_size must be a power of two and at least 32, got " + std::to_string(s.block_size);
    else if (bits != 4) s.problem = "expert_weight_bits must be 4, got " + std::to_string(bits) + ". Why: only this packing has gfx950 kernels for experts. How to fix: export 4-bit experts";
    else if (s.normalize != 0 && s.normalize != 1) s.problem = "normalize_routing_weights must be 0 or 1, got " + std::to_string(s.normalize);
    else if (s.fusion < 0 || s.fusion > 2) s.problem = "swiglu_fusion must be 0, 1 or 2, got " + std::to_string(s.fusion);
    else if (!std::isfinite(s.alpha) || !std::isfinite(s.beta)) s.problem = "activation_alpha and activation_beta must be finite";
    else if (!(s.limit > 0.f)) s.problem = "swiglu_limit must be positive";
    return s;
}

struct MoeNode final : NxrtRocmNode {
    MoeSettings s;
    MoeNode(NxrtRocmEp* provider, const MoeSettings& settings) : NxrtRocmNode(provider), s(settings) {}
    const char* op() const override { return "QMoE"; }
    NxrtStatus workspace(const NxrtTensorDesc* in, uint32_t n, uint64_t* bytes) const override
    {
        int64_t rows = 0, hidden = 0, again = 0, experts = 0, outer = 0, depth = 0;
        if (!static_matrix(in, n, 0, &rows, &hidden) || !static_matrix(in, n, 1, &again, &experts) || n <= 2 || in[2].ndim < 3 || !in[2].dims || !static_matrix(in, n, 2, &outer, &depth))
            return make_status(NXRT_INVALID_ARGUMENT, err("workspace_requirement needs the shapes of input, router_probs and fc1_experts_weights"));
        RocmMoeArgs a{};
        a.rows = rows;
        a.hidden = hidden;
        a.inter = in[2].dims[1] / (s.fusion ? 2 : 1);
        a.experts = static_cast<int>(experts);
        a.k = static_cast<int>(s.k);
        a.block_size = static_cast<int>(s.block_size);
        if (hidden < 1 || hidden > (1 << 20) || a.inter < 1 || a.inter > (1 << 20) || experts < 1 || experts > ROCM_MOE_MAX_EXPERTS || rows * s.k >= (int64_t{1} << 24))
            return make_status(NXRT_INVALID_ARGUMENT, err("workspace_requirement got shapes that no call takes"));
        const NxrtStatus st = ep->bind();          // (the plan goes by the GPU's CUs)
        if (st.code != NXRT_OK) return st;
        *bytes = rows ? rocm_moe_workspace_bytes(&a) : 0;
        return ok();
    }
    NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void* ws, uint64_t ws_bytes) override
    {
        Call c(op(), *ep, in, n_in, out, n_out);
        c.arity(7, 14, 1);
        if (!c.failed() && no_rows(in, n_in)) return ok();
        const auto* x = c.required(c.input(0, "input"), "input");
        c.dtype(x, "input", {NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        uint64_t rows = 0, h = 0, logit_rows = 0, e = 0;
        c.matrix(x, "input", &rows, &h);
        const auto* logits = c.required(c.input(1, "router_probs"), "router_probs");
        c.dtype(logits, "router_probs", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        c.matrix(logits, "router_probs", &logit_rows, &e);
        if (!c.failed() && logit_rows != rows) c.fail("router_probs must have as many rows as input (" + std::to_string(rows) + "), got " + text(*logits));
        if (!c.failed() && (e < 1 || e > ROCM_MOE_MAX_EXPERTS)) c.fail("1..=" + std::to_string(ROCM_MOE_MAX_EXPERTS) + " experts are supported, got " + std::to_string(e));
        if (!c.failed() && e < static_cast<uint64_t>(s.k)) c.fail("k=" + std::to_string(s.k) + " is more than the " + std::to_string(e) + " experts");
        if (!c.failed() && (h < 1 || h > (1u << 20))) c.fail("the last dimension of input must be 1..=2^20, got " + std::to_string(h));
        if (!c.failed() && rows * static_cast<uint64_t>(s.k) >= (uint64_t{1} << 24)) c.fail("rows times k must be below 2^24, got " + std::to_string(rows) + " rows");
        const auto* w1 = c.required(c.input(2, "fc1_experts_weights"), "fc1_experts_weights");
        if (!c.failed() && w1->ndim != 3 && w1->ndim != 4) c.fail("fc1_experts_weights must have rank 3 or 4, got " + text(*w1));
        if (c.failed()) return c.status();
        const uint64_t f = w1->shape[1], i = s.fusion ? f / 2 : f;
        if (f < 1 || f > (1u << 20) || (s.fusion && f % 2 != 0)) c.fail("fc1_experts_weights must have 1..=2^20 rows an expert, an even number with swiglu_fusion, got " + text(*w1));
        const uint64_t bs = static_cast<uint64_t>(s.block_size), kb1 = (h + bs - 1) / bs, kb2 = (i + bs - 1) / bs;
        RocmMoeArgs a{};
        uint32_t scale_dtype = 0, bias_dtype = 0;
        struct Names {
            const char *weights, *scales, *bias, *zeros;
        };
        auto projection = [&](const Names& name, uint32_t first, uint32_t zp_at, uint64_t n, uint64_t kb, RocmMoeWeights& to) {
            const auto* w = c.required(c.input(first, name.weights), name.weights);
            c.dtype(w, name.weights, {NXRT_DT_UINT8});
            if (w && w->ndim == 3) c.shape(w, name.weights, {e, n, kb * bs / 2});
            else c.shape(w, name.weights, {e, n, kb, bs / 2});
            if (w && !c.failed() && reinterpret_cast<uintptr_t>(at(*w)) % 16 != 0) c.fail(std::string(name.weights) + " must start at a multiple of 16 bytes");
            const auto* sc = c.required(c.input(first + 1, name.scales), name.scales);
            c.dtype(sc, name.scales, {x->dtype, NXRT_DT_FLOAT32});
            c.shape(sc, name.scales, {e, n, kb});
            if (sc && !c.failed()) {
                if (scale_dtype && sc->dtype != scale_dtype) c.fail("all scales must have one dtype");
                scale_dtype = sc->dtype;
            }
            const auto* bi = c.input(first + 2, name.bias);
            c.dtype(bi, name.bias, {x->dtype, NXRT_DT_FLOAT32});
            c.shape(bi, name.bias, {e, n});
            if (bi && !c.failed()) {
                if (bias_dtype && bi->dtype != bias_dtype) c.fail("all biases must have one dtype");
                bias_dtype = bi->dtype;
            }
            const auto* z = c.input(zp_at, name.zeros);
            c.dtype(z, name.zeros, {NXRT_DT_UINT8});
            c.shape(z, name.zeros, {e, n, (kb + 1) / 2});
            if (c.failed()) return;
            to = RocmMoeWeights{at(*w), at(*sc), z ? at(*z) : nullptr, bi ? at(*bi) : nullptr};
        };
        projection({"fc1_experts_weights", "fc1_scales", "fc1_experts_bias", "fc1_zero_points"}, 2, 11, f, kb1, a.gate);
        projection({"fc2_experts_weights", "fc2_scales", "fc2_experts_bias", "fc2_zero_points"}, 5, 12, h, kb2, a.down);
        if (s.fusion == 0) {
            projection({"fc3_experts_weights", "fc3_scales", "fc3_experts_bias", "fc3_zero_points"}, 8, 13, f, kb1, a.up);
            if (!c.failed() && ((a.gate.bias == nullptr) != (a.up.bias == nullptr) || (a.gate.zp == nullptr) != (a.up.zp == nullptr)))
                c.fail("fc1 and fc3 must both have biases and zero points, or neither");
        } else {
            for (uint32_t extra : {8u, 9u, 10u, 13u})
                if (c.input(extra, "fc3")) c.fail("fc3 goes with swiglu_fusion=0 only");
        }
        const auto* y = c.required(c.output(0, "output"), "output");
        c.dtype(y, "output", {x->dtype});
        c.shape_like(y, "output", x, h);
        c.check_overlap();
        if (c.failed()) return c.status();

        a.x = at(*x);
        a.logits = at(*logits);
        a.y = at(*y);
        a.up_expert_step = static_cast<int64_t>(f);
        a.up_row_step = s.fusion == 1 ? 2 : 1;
        if (s.fusion != 0) {
            // up begins one row (alternating) or I rows (halves) behind gate
            const uint64_t skip = s.fusion == 1 ? 1 : i;
            a.up = a.gate;
            a.up.b += skip * kb1 * bs / 2;
            a.up.scales = static_cast<const uint8_t*>(a.up.scales) + skip * kb1 * item_size(scale_dtype);
            if (a.up.zp) a.up.zp += skip * ((kb1 + 1) / 2);
            if (a.up.bias) a.up.bias = static_cast<const uint8_t*>(a.up.bias) + skip * item_size(bias_dtype);
        }
        a.rows = static_cast<int64_t>(rows);
        a.hidden = static_cast<int64_t>(h);
        a.inter = static_cast<int64_t>(i);
        a.experts = static_cast<int>(e);
        a.k = static_cast<int>(s.k);
        a.block_size = static_cast<int>(s.block_size);
        a.normalize = static_cast<int>(s.normalize);
        a.dtype = static_cast<int>(x->dtype);
        a.logits_dtype = static_cast<int>(logits->dtype);
        a.scale_dtype = static_cast<int>(scale_dtype);
        a.bias_dtype = bias_dtype ? static_cast<int>(bias_dtype) : ROCM_DT_F32;
        a.alpha = s.alpha;
        a.beta = s.beta;
        a.limit = s.limit;
        NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        void* scratch_at = nullptr;
        st = find_scratch(rocm_moe_workspace_bytes(&a), ws, ws_bytes, &scratch_at);
        if (st.code != NXRT_OK) return st;
        variant = rocm_moe_variant(&a);
        ep->launches.fetch_add(1);
        return launched(rocm_launch_moe(&a, scratch_at, ep->stream));
    }
};

}  // namespace

extern "C" {

int nxrt_rocm_ep_supports_qmoe(const NxrtRocmEp*, const NxrtRocmQMoEAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len)
{
    return supported("QMoE", reason, reason_len, [&]() -> std::string {
        const MoeSettings s = settings_of(attrs);
        if (!s.problem.empty() || !inputs) return s.problem;
        std::string why = arity(n_inputs, 7, 14);
        if (!why.empty()) return why;
        if (inputs[0].dtype != NXRT_DT_FLOAT16 && inputs[0].dtype != NXRT_DT_BFLOAT16) return std::string("input must have dtype Float16 or BFloat16, got ") + dtype_name(inputs[0].dtype);
        if (!is_float(inputs[1].dtype)) return std::string("router_probs must have a float dtype, got ") + dtype_name(inputs[1].dtype);
        const bool fc3 = n_inputs > 8 && inputs[8].dtype != 0;
        if (fc3 != (s.fusion == 0)) return "fc3 goes with swiglu_fusion=0, and only with it";
        if (inputs[2].dtype != NXRT_DT_UINT8 || inputs[5].dtype != NXRT_DT_UINT8 || (fc3 && inputs[8].dtype != NXRT_DT_UINT8)) return "expert weights must have dtype Uint8";
        return {};
    });
}

int nxrt_rocm_ep_supports_matmul_int8(const NxrtRocmEp*, const NxrtRocmMatMulInt8Attrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len)
{
    return supported("MatMulInt8", reason, reason_len, [&]() -> std::string {
        const Int8Settings s = settings_of(attrs);
        if (!s.problem.empty() || !inputs) return s.problem;
        std::string why = arity(n_inputs, 3, 5);
        if (!why.empty()) return why;
        if (!is_float(inputs[0].dtype) && inputs[0].dtype != NXRT_DT_INT8) return std::string("A must have a float dtype or Int8, got ") + dtype_name(inputs[0].dtype);
        if (inputs[1].dtype != NXRT_DT_INT8) return std::string("B must have dtype Int8, got ") + dtype_name(inputs[1].dtype);
        if (!is_float(inputs[2].dtype)) return std::string("b_scale must have a float dtype, got ") + dtype_name(inputs[2].dtype);
        const bool scale = n_inputs > 3 && inputs[3].dtype != 0;
        if (scale != (inputs[0].dtype == NXRT_DT_INT8)) return "a_scale goes with Int8 A, and only with it";
        return {};
    });
}

int nxrt_rocm_ep_supports_gated_residual_norm(const NxrtRocmEp*, const NxrtRocmGatedResidualNormAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len)
{
    return supported("GatedResidualNorm", reason, reason_len, [&]() -> std::string {
        const GatedNormSettings s = settings_of(attrs);
        if (!s.problem.empty() || !inputs) return s.problem;
        std::string why = arity(n_inputs, 1, 7);
        if (!why.empty()) return why;
        if (!is_float(inputs[0].dtype)) return std::string("residual must have a float dtype, got ") + dtype_name(inputs[0].dtype);
        if (n_inputs > 1 && inputs[1].dtype != 0 && inputs[1].dtype != inputs[0].dtype) return "block must have the residual's dtype";
        return {};
    });
}

NxrtStatus nxrt_rocm_qmoe_create(NxrtRocmEp* ep, const NxrtRocmQMoEAttrs* attrs, NxrtRocmNode** out_node) { return create_node<MoeNode>("QMoE", ep, out_node, [&] { return settings_of(attrs); }); }
NxrtStatus nxrt_rocm_matmul_int8_create(NxrtRocmEp* ep, const NxrtRocmMatMulInt8Attrs* attrs, NxrtRocmNode** out_node) { return create_node<Int8Node>("MatMulInt8", ep, out_node, [&] { return settings_of(attrs); }); }
NxrtStatus nxrt_rocm_gated_residual_norm_create(NxrtRocmEp* ep, const NxrtRocmGatedResidualNormAttrs* attrs, NxrtRocmNode** out_node)
{
    return create_node<GatedNormNode>("GatedResidualNorm", ep, out_node, [&] { return settings_of(attrs); });
}

void nxrt_rocm_node_set_constant_inputs(NxrtRocmNode*, const uint8_t*, uint32_t) {}        // (no node copies its weights)

NxrtStatus nxrt_rocm_node_workspace_requirement(const NxrtRocmNode* node, const NxrtTensorDesc* inputs, uint32_t n_inputs, NxrtRocmWorkspaceRequirement* out)
{
    return fenced([&]() -> NxrtStatus {
        if (!node || !out) return make_status(NXRT_INVALID_ARGUMENT, "null pointer in workspace_requirement");
        out->alignment = 256;
        out->bytes = 0;
        return node->workspace(inputs, n_inputs, &out->bytes);
    });
}

NxrtStatus nxrt_rocm_node_execute(NxrtRocmNode* node, const NxrtRocmTensorView* inputs, uint32_t n_inputs, NxrtRocmTensorView* outputs, uint32_t n_outputs, void* workspace_device,
                                  uint64_t workspace_bytes)
{
    return fenced([&]() -> NxrtStatus {
        if (!node) return make_status(NXRT_INVALID_ARGUMENT, "null node in execute");
        std::lock_guard<std::mutex> lock(node->mu);
        return node->execute(inputs, n_inputs, outputs, n_outputs, workspace_device, workspace_bytes);
    });
}

const char* nxrt_rocm_node_last_variant(const NxrtRocmNode* node) { return node ? node->variant : ""; }
uint64_t nxrt_rocm_node_retired_buffers(const NxrtRocmNode* node) { return node ? node->retired.size() : 0; }
void nxrt_rocm_node_release(NxrtRocmNode* node)
{
    try {
        delete node;
    } catch (...) {
    }
}

}  // extern "C"
