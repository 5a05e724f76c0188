// The operators of a paged 8-bit cache (RotaryEmbedding, CacheAppend, CacheAttention, CachePages): attributes, input checks, scratch and the C entry points.
#include "nodes.h"

using namespace nxrt_rocm;

namespace {

// ---- RotaryEmbedding --------------------------------------------------------------------------------------------------

struct RotarySettings {
    int64_t head_size = 0, heads = 0, part = 0, interleaved = 0, scaling = 0;
    double magnitude = 1.0;
    std::vector<double> turns;          // whole turns a position, of each pair
    std::string problem;
};

RotarySettings settings_of(const NxrtRocmRotaryEmbeddingAttrs* attrs)
{
    RotarySettings s;
    if (!attrs) {
        s.problem = "null attributes";
        return s;
    }
    const auto a = read_attrs(attrs);
    if (!NODE_ATTR_PRESENT(a, 0, head_size)) {
        s.problem = "missing required integer attribute 'head_size'";
        return s;
    }
    s.head_size = a.head_size;
    if (NODE_ATTR_PRESENT(a, 1, num_heads)) s.heads = a.num_heads;
    s.part = NODE_ATTR_PRESENT(a, 2, rotary_embedding_dim) && a.rotary_embedding_dim ? a.rotary_embedding_dim : a.head_size;
    if (NODE_ATTR_PRESENT(a, 3, interleaved)) s.interleaved = a.interleaved;
    if (NODE_ATTR_PRESENT(a, 4, scaling)) s.scaling = a.scaling;
    const int64_t original = NODE_ATTR_PRESENT(a, 5, original_max_position) ? a.original_max_position : 8192;
    const double theta = NODE_ATTR_PRESENT(a, 6, rope_theta) ? a.rope_theta : 10000.0;
    const double factor = NODE_ATTR_PRESENT(a, 7, factor) ? a.factor : 1.0;
    const double low = NODE_ATTR_PRESENT(a, 8, low_freq_factor) ? a.low_freq_factor : 1.0, high = NODE_ATTR_PRESENT(a, 9, high_freq_factor) ? a.high_freq_factor : 4.0;
    const double fast = NODE_ATTR_PRESENT(a, 10, beta_fast) ? a.beta_fast : 32.0, slow = NODE_ATTR_PRESENT(a, 11, beta_slow) ? a.beta_slow : 1.0;
    s.magnitude = NODE_ATTR_PRESENT(a, 12, attention_factor) ? a.attention_factor : s.scaling == 3 && factor > 1.0 ? 0.1 * std::log(factor) + 1.0 : 1.0;
    if (s.head_size < 2 || s.head_size > (1 << 16)) s.problem = "head_size must be 2..=65536, got " + std::to_string(s.head_size);
    else if (s.heads < 0 || s.heads > (1 << 20)) s.problem = "num_heads must be 0..=2^20, got " + std::to_string(s.heads);
    else if (s.part < 2 || s.part > s.head_size || s.part % 2 != 0 || s.part > 2 * ROCM_ROTARY_MAX_PAIRS)
        s.problem = "rotary_embedding_dim must be even, 2..=" + std::to_string(2 * ROCM_ROTARY_MAX_PAIRS) + " and at most head_size, got " + std::to_string(s.part);
    else if (s.interleaved != 0 && s.interleaved != 1) s.problem = "interleaved must be 0 or 1, got " + std::to_string(s.interleaved);
    else if (s.scaling < 0 || s.scaling > 3) s.problem = "scaling must be 0 (none), 1 (linear), 2 (llama3) or 3 (yarn), got " + std::to_string(s.scaling);
    else if (!(theta > 1.0) || !std::isfinite(theta)) s.problem = "rope_theta must be finite and above 1";
    else if (!(factor > 0.0) || !std::isfinite(factor)) s.problem = "factor must be finite and positive";
    else if (original < 1) s.problem = "original_max_position must be positive, got " + std::to_string(original);
    else if (s.scaling == 2 && !(low < high && std::isfinite(low) && std::isfinite(high))) s.problem = "low_freq_factor must be below high_freq_factor";
    else if (s.scaling == 3 && !(slow > 0.0 && slow < fast && std::isfinite(fast))) s.problem = "beta_slow must be positive and below beta_fast";
    else if (!std::isfinite(s.magnitude)) s.problem = "attention_factor must be finite";
    if (!s.problem.empty()) return s;
    const double turn = 6.283185307179586476925, context = static_cast<double>(original);
    // yarn: the pair that makes so many turns within the first context (below 0: none does)
    auto pair = [&](double turns) { return static_cast<double>(s.part) * std::log(context / (turns * turn)) / (2.0 * std::log(theta)); };
    const double first = std::max(std::floor(pair(fast)), 0.0), last = std::min(std::ceil(pair(slow)), static_cast<double>(s.part - 1));
    for (int64_t i = 0; i < s.part / 2; ++i) {
        double f = std::pow(theta, -2.0 * static_cast<double>(i) / static_cast<double>(s.part));
        double kept = 1.0;                // of the frequency as it is, against the slower one
        if (s.scaling == 1) kept = 0.0;
        if (s.scaling == 2) kept = std::min(1.0, std::max(0.0, (context * f / turn - low) / (high - low)));
        if (s.scaling == 3) kept = last < 0.0 ? 0.0 : 1.0 - std::min(1.0, std::max(0.0, (static_cast<double>(i) - first) / std::max(last - first, 0.001)));
        f = f / factor * (1.0 - kept) + f * kept;
        s.turns.push_back(f / turn);
    }
    return s;
}

struct RotaryNode final : NxrtRocmNode {
    RotarySettings s;
    RotaryNode(NxrtRocmEp* provider, const RotarySettings& settings) : NxrtRocmNode(provider), s(settings) {}
    const char* op() const override { return "RotaryEmbedding"; }
    NxrtStatus workspace(const NxrtTensorDesc*, uint32_t, uint64_t* bytes) const override
    {
        *bytes = 0;
        return ok();
    }
    NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void*, uint64_t) override
    {
        Call c(op(), *ep, in, n_in, out, n_out);
        c.arity(2, 4, 1);
        if (!c.failed() && no_rows(in, n_in)) return ok();
        const auto* x = c.required(c.input(0, "input"), "input");
        c.dtype(x, "input", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        uint64_t rows = 0, last = 0;
        c.matrix(x, "input", &rows, &last);
        if (c.failed()) return c.status();
        const uint64_t d = static_cast<uint64_t>(s.head_size);
        RocmRotaryArgs a{};
        if (x->ndim == 4) {
            const uint64_t heads = x->shape[1], length = x->shape[2];
            if (last != d) c.fail("input of rank 4 must have last dimension head_size=" + std::to_string(d) + ", got " + text(*x));
            if (!c.failed() && s.heads && heads != static_cast<uint64_t>(s.heads)) c.fail("input must have num_heads=" + std::to_string(s.heads) + " heads, got " + text(*x));
            if (!c.failed() && heads > (1u << 20)) c.fail("input may have up to 2^20 heads, got " + text(*x));
            rows = x->shape[0] * length;
            a.inner = static_cast<int64_t>(length);
            a.outer_step = static_cast<int64_t>(heads * length * d);
            a.row_step = static_cast<int64_t>(d);
            a.head_step = static_cast<int64_t>(length * d);
            a.heads = static_cast<int>(heads);
        } else {
            if (s.heads == 0 && (last == 0 || last % d != 0)) c.fail("the last dimension of input must be a multiple of head_size=" + std::to_string(d) + ", got " + text(*x));
            if (!c.failed() && last < static_cast<uint64_t>(s.heads) * d) c.fail("the last dimension of input must hold num_heads=" + std::to_string(s.heads) + " heads of " + std::to_string(d) + ", got " + text(*x));
            const uint64_t heads = s.heads ? static_cast<uint64_t>(s.heads) : last / d;
            a.inner = static_cast<int64_t>(x->ndim >= 2 ? x->shape[x->ndim - 2] : 1);
            a.row_step = static_cast<int64_t>(last);
            a.outer_step = a.inner * a.row_step;
            a.head_step = static_cast<int64_t>(d);
            a.heads = static_cast<int>(heads);
            a.extra = static_cast<int64_t>(last - heads * d);
        }
        if (!c.failed() && rows > 0x7fffffff) c.fail("too many rows: " + std::to_string(rows));
        if (!c.failed() && last > (1u << 26)) c.fail("rows are too long: " + text(*x));
        const auto* positions = c.required(c.input(1, "position_ids"), "position_ids");
        c.dtype(positions, "position_ids", {NXRT_DT_INT64, NXRT_DT_INT32});
        uint64_t count = 0;
        if (positions && !c.failed()) {
            elements_of(*positions, positions->ndim, &count);
            if (count != rows && count != 1) c.fail("position_ids must have one element, or one for each of the " + std::to_string(rows) + " rows, got " + text(*positions));
        }
        const auto* cosines = c.input(2, "cos_cache");
        const auto* sines = c.input(3, "sin_cache");
        if (!c.failed() && (cosines == nullptr) != (sines == nullptr)) c.fail("cos_cache and sin_cache go together");
        if (cosines && !c.failed()) {
            c.dtype(cosines, "cos_cache", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
            if (cosines->ndim != 2 || cosines->shape[1] != static_cast<uint64_t>(s.part / 2)) c.fail("cos_cache must have shape [M, " + std::to_string(s.part / 2) + "], got " + text(*cosines));
            if (!c.failed()) c.dtype(sines, "sin_cache", {cosines->dtype});
            if (!c.failed()) c.shape(sines, "sin_cache", {cosines->shape[0], cosines->shape[1]});
        }
        const auto* y = c.required(c.output(0, "output"), "output");
        c.dtype(y, "output", {x->dtype});
        c.shape_like(y, "output", x, last);
        // a thread reads its pairs before it writes them, and no other row's
        c.check_overlap([](uint32_t, uint32_t i) { return i == 0; });
        if (c.failed()) return c.status();
        a.x = at(*x);
        a.y = at(*y);
        a.positions = at(*positions);
        a.positions_dtype = static_cast<int>(positions->dtype);
        a.one_position = count == 1;
        a.cos_cache = cosines ? at(*cosines) : nullptr;
        a.sin_cache = sines ? at(*sines) : nullptr;
        a.cache_dtype = cosines ? static_cast<int>(cosines->dtype) : ROCM_DT_F32;
        a.cache_rows = cosines ? static_cast<int64_t>(cosines->shape[0]) : 0;
        a.rows = static_cast<int64_t>(rows);
        a.head_size = static_cast<int>(d);
        a.part = static_cast<int>(s.part);
        a.interleaved = static_cast<int>(s.interleaved);
        a.dtype = static_cast<int>(x->dtype);
        a.magnitude = s.magnitude;
        std::copy(s.turns.begin(), s.turns.end(), a.turns);
        variant = cosines ? "rotary_cached" : "rotary";
        const NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        ep->launches.fetch_add(1);
        return launched(rocm_launch_rotary(&a, ep->stream));
    }
};

// ---- what the cache's nodes read alike -----------------------------------------------------------------------------------

// A call whose block table (input i) has no sequences has nothing to do, as one without rows, and none of its tensors needs memory behind it.
bool no_sequences(const NxrtRocmTensorView* in, uint32_t n_in, uint32_t i) { return i < n_in && in[i].ndim == 2 && in[i].shape && in[i].shape[0] == 0; }

// Inputs `first` (k_cache, v_cache, k_scale, v_scale, cumulative_lengths, past_lengths, block_table) of a call over `rows` new tokens.
struct CacheInputs {
    const NxrtRocmTensorView *k, *v, *k_scale, *v_scale, *ends, *past, *table;
    CacheInputs(Call& c, uint32_t first)
    {
        k = c.required(c.input(first, "k_cache"), "k_cache");
        v = c.required(c.input(first + 1, "v_cache"), "v_cache");
        k_scale = c.required(c.input(first + 2, "k_scale"), "k_scale");
        v_scale = c.required(c.input(first + 3, "v_scale"), "v_scale");
        ends = c.required(c.input(first + 4, "cumulative_lengths"), "cumulative_lengths");
        past = c.required(c.input(first + 5, "past_lengths"), "past_lengths");
        table = c.required(c.input(first + 6, "block_table"), "block_table");
    }
    void check(Call& c, uint64_t kv_heads, uint64_t d, RocmCache* to) const
    {
        c.dtype(k, "k_cache", {NXRT_DT_INT8, NXRT_DT_FLOAT8E4M3FN});
        if (c.failed()) return;
        if (k->ndim != 4 || k->shape[1] != kv_heads || k->shape[3] != d)
            return c.fail("k_cache must have shape [P, " + std::to_string(kv_heads) + ", B, " + std::to_string(d) + "], got " + text(*k));
        const uint64_t pages = k->shape[0], b = k->shape[2];
        if (b != 16 && b != 32 && b != 64 && b != 128) return c.fail("a page must have 16, 32, 64 or 128 tokens, got " + text(*k));
        if (pages < 1) return c.fail("k_cache has no pages");
        c.dtype(v, "v_cache", {k->dtype});
        c.shape(v, "v_cache", {pages, kv_heads, d, b});
        if (!c.failed() && (reinterpret_cast<uintptr_t>(at(*k)) % 16 != 0 || reinterpret_cast<uintptr_t>(at(*v)) % 16 != 0)) c.fail("k_cache and v_cache must start at multiples of 16 bytes");
        c.dtype(k_scale, "k_scale", {NXRT_DT_FLOAT32});
        c.shape(k_scale, "k_scale", {pages, kv_heads});
        c.dtype(v_scale, "v_scale", {NXRT_DT_FLOAT32});
        c.shape(v_scale, "v_scale", {pages, kv_heads});
        for (const auto* t : {ends, past, table}) c.dtype(t, t == ends ? "cumulative_lengths" : t == past ? "past_lengths" : "block_table", {NXRT_DT_INT32});
        if (c.failed()) return;
        if (table->ndim != 2 || table->shape[1] < 1) return c.fail("block_table must have shape [N, W] with W >= 1, got " + text(*table));
        const uint64_t n = table->shape[0], width = table->shape[1];
        if (width * b >= (uint64_t{1} << 30)) return c.fail("block_table must have fewer than 2^30 slots a sequence, got " + text(*table));
        if (n >= (1u << 20) || n * kv_heads >= (1u << 20)) return c.fail("block_table must have fewer than 2^20 sequences times key heads, got " + text(*table));
        c.shape(ends, "cumulative_lengths", {n + 1});
        c.shape(past, "past_lengths", {n});
        if (c.failed()) return;
        to->k = at(*k);
        to->v = at(*v);
        to->k_scale = reinterpret_cast<float*>(at(*k_scale));
        to->v_scale = reinterpret_cast<float*>(at(*v_scale));
        to->ends = reinterpret_cast<const int32_t*>(at(*ends));
        to->past = reinterpret_cast<const int32_t*>(at(*past));
        to->table = reinterpret_cast<const int32_t*>(at(*table));
        to->pages = static_cast<int64_t>(pages);
        to->sequences = static_cast<int>(n);
        to->width = static_cast<int>(width);
        to->page = static_cast<int>(b);
        to->kv_heads = static_cast<int>(kv_heads);
        to->head_size = static_cast<int>(d);
        to->code_dtype = static_cast<int>(k->dtype);
    }
};

// ---- CacheAppend ---------------------------------------------------------------------------------------------------------

struct AppendSettings {
    int64_t heads = 0, kv_heads = 0, head_size = 0;
    std::string problem;
};
AppendSettings settings_of(const NxrtRocmCacheAppendAttrs* attrs)
{
    AppendSettings s;
    if (!attrs) {
        s.problem = "null attributes";
        return s;
    }
    const auto a = read_attrs(attrs);
    if (NODE_ATTR_PRESENT(a, 0, num_heads)) s.heads = a.num_heads;
    if (!NODE_ATTR_PRESENT(a, 1, kv_num_heads)) s.problem = "missing required integer attribute 'kv_num_heads'";
    else if (!NODE_ATTR_PRESENT(a, 2, head_size)) s.problem = "missing required integer attribute 'head_size'";
    else if (s.heads < 0 || s.heads > 65535) s.problem = "num_heads must be 0..=65535, got " + std::to_string(s.heads);
    else if (a.kv_num_heads < 1 || a.kv_num_heads > 65535) s.problem = "kv_num_heads must be 1..=65535, got " + std::to_string(a.kv_num_heads);
    else if (a.head_size < 16 || a.head_size > ROCM_CACHE_MAX_HEAD || a.head_size % 16 != 0)
        s.problem = "head_size must be a multiple of 16 up to " + std::to_string(ROCM_CACHE_MAX_HEAD) + ", got " + std::to_string(a.head_size);
    s.kv_heads = a.kv_num_heads;
    s.head_size = a.head_size;
    return s;
}

struct AppendNode final : NxrtRocmNode {
    AppendSettings s;
    AppendNode(NxrtRocmEp* provider, const AppendSettings& settings) : NxrtRocmNode(provider), s(settings) {}
    const char* op() const override { return "CacheAppend"; }
    NxrtStatus workspace(const NxrtTensorDesc*, uint32_t, uint64_t* bytes) const override
    {
        *bytes = 0;
        return ok();
    }
    NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void*, uint64_t) override
    {
        Call c(op(), *ep, in, n_in, out, n_out);
        c.arity(9, 9, 4);
        if (!c.failed() && (no_rows(in, n_in) || no_sequences(in, n_in, 8))) return ok();
        const auto* key = c.required(c.input(0, "key"), "key");
        c.dtype(key, "key", {NXRT_DT_FLOAT32, NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        const auto* value = c.input(1, "value");
        if (c.failed()) return c.status();
        const uint64_t kv = static_cast<uint64_t>(s.kv_heads * s.head_size), packed = static_cast<uint64_t>(s.heads * s.head_size) + 2 * kv;
        if (key->ndim != 2 || key->shape[1] != (value ? kv : packed))
            c.fail(std::string(value ? "key" : "packed rows (no value)") + " must have shape [T, " + std::to_string(value ? kv : packed) + "], got " + text(*key));
        if (!c.failed() && key->shape[0] >= (1u << 26)) c.fail("too many rows: " + text(*key));
        c.dtype(value, "value", {key->dtype});
        if (value && !c.failed()) c.shape(value, "value", {key->shape[0], kv});
        const CacheInputs cache(c, 2);
        RocmCacheAppendArgs a{};
        if (!c.failed()) cache.check(c, static_cast<uint64_t>(s.kv_heads), static_cast<uint64_t>(s.head_size), &a.cache);
        const char* const names[] = {"k_cache", "v_cache", "k_scale", "v_scale"};
        const NxrtRocmTensorView* const state[] = {cache.k, cache.v, cache.k_scale, cache.v_scale};
        for (uint32_t i = 0; i < 4; ++i) c.in_place(state[i], c.required(c.output(i, names[i]), names[i]), names[i]);
        c.check_overlap([](uint32_t o, uint32_t i) { return i == o + 2; });
        if (c.failed()) return c.status();
        a.rows = static_cast<int64_t>(key->shape[0]);
        a.dtype = static_cast<int>(key->dtype);
        if (value) {
            a.k = at(*key);
            a.v = at(*value);
            a.k_step = a.v_step = static_cast<int64_t>(kv);
        } else {
            const uint64_t item = item_size(key->dtype);
            a.k = at(*key) + static_cast<uint64_t>(s.heads * s.head_size) * item;
            a.v = static_cast<const uint8_t*>(a.k) + kv * item;
            a.k_step = a.v_step = static_cast<int64_t>(packed);
        }
        variant = a.cache.code_dtype == ROCM_DT_E4M3 ? "cache_append_e4m3" : "cache_append_int8";
        const NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        ep->launches.fetch_add(1);
        return launched(rocm_launch_cache_append(&a, ep->stream));
    }
};

// ---- CacheAttention ------------------------------------------------------------------------------------------------------

struct AttentionSettings {
    int64_t heads = 0, kv_heads = 0, head_size = 0, window = -1;
    double scale = 0.0, softcap = 0.0;
    std::string problem;
};
AttentionSettings settings_of(const NxrtRocmCacheAttentionAttrs* attrs)
{
    AttentionSettings s;
    if (!attrs) {
        s.problem = "null attributes";
        return s;
    }
    const auto a = read_attrs(attrs);
    if (!NODE_ATTR_PRESENT(a, 0, num_heads)) s.problem = "missing required integer attribute 'num_heads'";
    else if (!NODE_ATTR_PRESENT(a, 1, kv_num_heads)) s.problem = "missing required integer attribute 'kv_num_heads'";
    else if (!NODE_ATTR_PRESENT(a, 2, head_size)) s.problem = "missing required integer attribute 'head_size'";
    s.heads = a.num_heads;
    s.kv_heads = a.kv_num_heads;
    s.head_size = a.head_size;
    if (NODE_ATTR_PRESENT(a, 3, local_window_size)) s.window = a.local_window_size;
    if (NODE_ATTR_PRESENT(a, 4, scale)) s.scale = a.scale;
    if (NODE_ATTR_PRESENT(a, 5, softcap)) s.softcap = a.softcap;
    if (!s.problem.empty()) return s;
    if (s.kv_heads < 1 || s.kv_heads > 4096) s.problem = "kv_num_heads must be 1..=4096, got " + std::to_string(s.kv_heads);
    else if (s.heads < s.kv_heads || s.heads > 65535 || s.heads % s.kv_heads != 0) s.problem = "num_heads must be a multiple of kv_num_heads up to 65535, got " + std::to_string(s.heads);
    else if (s.head_size != 64 && s.head_size != 80 && s.head_size != 96 && s.head_size != 128 && s.head_size != 256)
        s.problem = "head_size must be 64, 80, 96, 128 or 256, got " + std::to_string(s.head_size) + ". Why: only these have gfx950 kernels. How to fix: pad the heads with zeros";
    else if (s.window != -1 && (s.window < 1 || s.window > 0x7fffffff)) s.problem = "local_window_size must be -1 (none) or 1..=2^31 - 1, got " + std::to_string(s.window);
    else if (!(s.scale >= 0.0) || !std::isfinite(static_cast<float>(s.scale))) s.problem = "scale must be finite and not negative";
    else if (!(s.softcap >= 0.0) || !std::isfinite(static_cast<float>(s.softcap))) s.problem = "softcap must be finite and not negative";
    if (s.scale == 0.0 && s.problem.empty()) s.scale = 1.0 / std::sqrt(static_cast<double>(s.head_size));
    return s;
}

struct AttentionNode final : NxrtRocmNode {
    AttentionSettings s;
    AttentionNode(NxrtRocmEp* provider, const AttentionSettings& settings) : NxrtRocmNode(provider), s(settings) {}
    const char* op() const override { return "CacheAttention"; }
    RocmCacheAttentionArgs args() const
    {
        RocmCacheAttentionArgs a{};
        a.heads = static_cast<int>(s.heads);
        a.window = s.window > 0 && s.window < (1 << 30) ? static_cast<int>(s.window) : 0;          // (no sequence has 2^30 slots)
        a.scale = static_cast<float>(s.scale);
        // (a cap below f32's normal numbers makes scores alike, as the smallest of these does; 0 would be none)
        a.softcap = s.softcap > 0.0 ? std::max(static_cast<float>(s.softcap), std::numeric_limits<float>::min()) : 0.f;
        a.cache.kv_heads = static_cast<int>(s.kv_heads);
        a.cache.head_size = static_cast<int>(s.head_size);
        return a;
    }
    NxrtStatus workspace(const NxrtTensorDesc* in, uint32_t n, uint64_t* bytes) const override
    {
        int64_t rows = 0, last = 0, sequences = 0, width = 0, outer = 0;
        if (!static_matrix(in, n, 0, &rows, &last) || !static_matrix(in, n, 1, &outer, &last) || in[1].ndim != 4 || !static_matrix(in, n, 7, &sequences, &width))
            return make_status(NXRT_INVALID_ARGUMENT, err("workspace_requirement needs the shapes of query, k_cache and block_table"));
        RocmCacheAttentionArgs a = args();
        const int64_t page = in[1].dims[2];
        if (rows >= (1 << 29) || rows * s.heads >= (int64_t{1} << 29) || sequences >= (1 << 20) || sequences * s.kv_heads >= (1 << 20) || width < 1 || page < 1 || page > ROCM_CACHE_MAX_PAGE || width * page >= (int64_t{1} << 30))
            return make_status(NXRT_INVALID_ARGUMENT, err("workspace_requirement got shapes that no call takes"));
        a.rows = rows;
        a.cache.sequences = static_cast<int>(sequences);
        a.cache.width = static_cast<int>(width);
        a.cache.page = static_cast<int>(page);
        const NxrtStatus st = ep->bind();          // (the plan goes by the GPU's CUs)
        if (st.code != NXRT_OK) return st;
        *bytes = rows && sequences ? rocm_cache_attention_workspace_bytes(&a) : 0;
        return ok();
    }
    NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void* ws, uint64_t ws_bytes) override
    {
        Call c(op(), *ep, in, n_in, out, n_out);
        c.arity(8, 8, 1);
        if (!c.failed() && (no_rows(in, n_in) || no_sequences(in, n_in, 7))) return ok();
        const auto* q = c.required(c.input(0, "query"), "query");
        c.dtype(q, "query", {NXRT_DT_FLOAT16, NXRT_DT_BFLOAT16});
        if (c.failed()) return c.status();
        const uint64_t wide = static_cast<uint64_t>(s.heads * s.head_size), packed = wide + static_cast<uint64_t>(2 * s.kv_heads * s.head_size);
        if (q->ndim != 2 || (q->shape[1] != wide && q->shape[1] != packed))
            c.fail("query must have shape [T, " + std::to_string(wide) + "], or packed [T, " + std::to_string(packed) + "], got " + text(*q));
        if (!c.failed() && (q->shape[0] >= (1u << 29) || q->shape[0] * static_cast<uint64_t>(s.heads) >= (1u << 29))) c.fail("too many rows: " + text(*q));
        const CacheInputs cache(c, 1);
        RocmCacheAttentionArgs a = args();
        if (!c.failed()) cache.check(c, static_cast<uint64_t>(s.kv_heads), static_cast<uint64_t>(s.head_size), &a.cache);
        const auto* y = c.required(c.output(0, "output"), "output");
        if (!c.failed()) c.dtype(y, "output", {q->dtype});
        if (!c.failed()) c.shape(y, "output", {q->shape[0], wide});
        c.check_overlap();
        if (c.failed()) return c.status();
        a.q = at(*q);
        a.y = at(*y);
        a.rows = static_cast<int64_t>(q->shape[0]);
        a.q_step = static_cast<int64_t>(q->shape[1]);
        a.dtype = static_cast<int>(q->dtype);
        NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        void* scratch_at = nullptr;
        st = find_scratch(a.cache.sequences ? rocm_cache_attention_workspace_bytes(&a) : 0, ws, ws_bytes, &scratch_at);
        if (st.code != NXRT_OK) return st;
        variant = rocm_cache_attention_variant(&a);
        ep->launches.fetch_add(1);
        return launched(rocm_launch_cache_attention(&a, scratch_at, ep->stream));
    }
};

// ---- CachePages ----------------------------------------------------------------------------------------------------------

struct PagesSettings {
    int64_t page_size = 0, compact = 0;
    std::string problem;
};
PagesSettings settings_of(const NxrtRocmCachePagesAttrs* attrs)
{
    PagesSettings s;
    if (!attrs) {
        s.problem = "null attributes";
        return s;
    }
    const auto a = read_attrs(attrs);
    if (!NODE_ATTR_PRESENT(a, 0, page_size)) s.problem = "missing required integer attribute 'page_size'";
    else if (a.page_size < 1 || a.page_size > (1 << 20)) s.problem = "page_size must be 1..=2^20, got " + std::to_string(a.page_size);
    s.page_size = a.page_size;
    if (NODE_ATTR_PRESENT(a, 1, compact)) s.compact = a.compact;
    if (s.problem.empty() && s.compact != 0 && s.compact != 1) s.problem = "compact must be 0 or 1, got " + std::to_string(s.compact);
    return s;
}

struct PagesNode final : NxrtRocmNode {
    PagesSettings s;
    PagesNode(NxrtRocmEp* provider, const PagesSettings& settings) : NxrtRocmNode(provider), s(settings) {}
    const char* op() const override { return "CachePages"; }
    NxrtStatus workspace(const NxrtTensorDesc* in, uint32_t n, uint64_t* bytes) const override
    {
        if (!in || n < 5 || in[4].ndim < 2 || !in[4].dims || in[4].dims[1] < 1 || in[4].dims[1] > ROCM_PAGES_MAX_PAGES)
            return make_status(NXRT_INVALID_ARGUMENT, err("workspace_requirement needs the shape of a pool, [L, P, ..] with P up to " + std::to_string(ROCM_PAGES_MAX_PAGES)));
        RocmCachePagesArgs a{};
        a.pages = in[4].dims[1];
        *bytes = rocm_cache_pages_workspace_bytes(&a);
        return ok();
    }
    // No page is in use and none moves; whoever asks for counts and moves has to find that. None of the other tensors needs memory behind it.
    NxrtStatus without_slots(Call& c)
    {
        const auto* moves = s.compact ? c.output(2, "moves") : nullptr;
        const auto* counts = c.output(3, "counts");
        c.dtype(counts, "counts", {NXRT_DT_INT32});
        c.shape(counts, "counts", {2});
        c.dtype(moves, "moves", {NXRT_DT_INT32});
        if (moves && !c.failed() && (moves->ndim != 2 || moves->shape[0] > ROCM_PAGES_MAX_PAGES / 2)) c.fail("moves must have shape [P / 2, 2], got " + text(*moves));
        if (moves && !c.failed()) c.shape(moves, "moves", {moves->shape[0], 2});
        c.check_overlap();
        if (c.failed()) return c.status();
        if (!counts && !moves) return ok();
        RocmCachePagesArgs a{};
        a.compact = static_cast<int>(s.compact);
        a.counts = counts ? reinterpret_cast<int32_t*>(at(*counts)) : nullptr;
        a.moves = moves ? reinterpret_cast<int32_t*>(at(*moves)) : nullptr;
        a.pages = moves ? static_cast<int64_t>(2 * moves->shape[0]) : 0;
        const NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        ep->launches.fetch_add(1);
        return launched(rocm_launch_cache_pages(&a, nullptr, ep->stream));
    }
    NxrtStatus execute(const NxrtRocmTensorView* in, uint32_t n_in, NxrtRocmTensorView* out, uint32_t n_out, void* ws, uint64_t ws_bytes) override
    {
        Call c(op(), *ep, in, n_in, out, n_out);
        c.arity(5, 4 + ROCM_PAGES_MAX_POOLS, 4 + ROCM_PAGES_MAX_POOLS);
        if (!c.failed() && no_rows(in, n_in)) return without_slots(c);
        const auto* table = c.required(c.input(0, "block_table"), "block_table");
        c.dtype(table, "block_table", {NXRT_DT_INT32});
        if (!c.failed() && (table->ndim != 2 || table->shape[1] < 1)) c.fail("block_table must have shape [S, W] with W >= 1, got " + text(*table));
        if (c.failed()) return c.status();
        const uint64_t slots = table->shape[0], width = table->shape[1];
        if (slots > ROCM_PAGES_MAX_SLOTS) c.fail("block_table may have up to " + std::to_string(ROCM_PAGES_MAX_SLOTS) + " sequences, got " + text(*table));
        if (!c.failed() && width * static_cast<uint64_t>(s.page_size) >= (uint64_t{1} << 30)) c.fail("block_table must have fewer than 2^30 tokens a sequence, got " + text(*table));
        if (!c.failed() && slots * width > 0x7fffffff) c.fail("block_table must have fewer than 2^31 entries, got " + text(*table));
        RocmCachePagesArgs a{};
        auto whole = [&](uint32_t i, const char* name, bool needed) -> const int32_t* {
            const auto* v = c.input(i, name);
            if (needed) c.required(v, name);
            c.dtype(v, name, {NXRT_DT_INT32});
            c.shape(v, name, {slots});
            return v ? reinterpret_cast<const int32_t*>(at(*v)) : nullptr;
        };
        a.lengths = whole(1, "lengths", true);
        a.parents = whole(2, "parents", false);
        a.grow = whole(3, "new_tokens", false);
        if (!c.failed() && s.compact && (a.parents || a.grow)) c.fail("parents and new_tokens do not go with compact=1");
        uint64_t pages = 0;
        for (uint32_t i = 4; i < n_in && !c.failed(); ++i) {
            const auto* pool = c.required(c.input(i, "pool"), "pool");
            if (!pool) break;
            if (pool->ndim < 2) return c.fail("a pool must have shape [L, P, ..], got " + text(*pool)), c.status();
            if (i == 4) pages = pool->shape[1];
            if (pool->shape[1] != pages) c.fail("all pools must have P=" + std::to_string(pages) + " pages, got " + text(*pool));
            if (!c.failed() && (pages < 1 || pages > ROCM_PAGES_MAX_PAGES)) c.fail("a pool may have 1..=" + std::to_string(ROCM_PAGES_MAX_PAGES) + " pages, got " + text(*pool));
            if (c.failed()) break;
            if (pool->dtype != NXRT_DT_FLOAT32 && pool->dtype != NXRT_DT_INT8 && pool->dtype != NXRT_DT_UINT8 && pool->dtype != NXRT_DT_INT32 && pool->dtype != NXRT_DT_FLOAT16 &&
                pool->dtype != NXRT_DT_BFLOAT16 && pool->dtype != NXRT_DT_FLOAT8E4M3FN && pool->dtype != NXRT_DT_INT64)
                c.fail("pool has an element type that this provider does not know");
            uint64_t bytes = item_size(pool->dtype);
            for (uint32_t d = 2; d < pool->ndim; ++d) bytes *= pool->shape[d];
            RocmPool& to = a.pool[a.pools++];
            to = RocmPool{at(*pool), static_cast<int64_t>(pool->shape[0]), static_cast<int64_t>(bytes)};
            if (to.layers * ((to.page_bytes + 8191) / 8192) >= (1 << 16)) c.fail("a pool's pages are too large: " + text(*pool));
            c.in_place(pool, c.required(c.output(i, "pool"), "pool"), "pool");
        }
        if (!c.failed() && n_out != n_in) c.fail("expected as many outputs as inputs, got " + std::to_string(n_out));
        auto written = [&](uint32_t i, const char* name, std::initializer_list<uint64_t> shape) -> int32_t* {
            const auto* v = c.required(c.output(i, name), name);
            c.dtype(v, name, {NXRT_DT_INT32});
            c.shape(v, name, shape);
            return v ? reinterpret_cast<int32_t*>(at(*v)) : nullptr;
        };
        a.next = written(0, "next_table", {slots, width});
        a.next_lengths = written(1, "next_lengths", {slots});
        if (s.compact && pages < 2) a.moves = nullptr;                      // (nothing can move: the output has no elements)
        else a.moves = written(2, "moves", {s.compact ? pages / 2 : slots, 2});
        a.counts = written(3, "counts", {2});
        c.check_overlap([](uint32_t o, uint32_t i) { return o >= 4 && i == o; });
        if (c.failed()) return c.status();
        a.table = reinterpret_cast<const int32_t*>(at(*table));
        a.pages = static_cast<int64_t>(pages);
        a.slots = static_cast<int>(slots);
        a.width = static_cast<int>(width);
        a.page = static_cast<int>(s.page_size);
        a.compact = static_cast<int>(s.compact);
        NxrtStatus st = ep->bind();
        if (st.code != NXRT_OK) return st;
        void* scratch_at = nullptr;
        st = find_scratch(rocm_cache_pages_workspace_bytes(&a), ws, ws_bytes, &scratch_at);
        if (st.code != NXRT_OK) return st;
        variant = s.compact ? "cache_pages_compact" : "cache_pages_step";
        ep->launches.fetch_add(1);
        return launched(rocm_launch_cache_pages(&a, scratch_at, ep->stream));
    }
};

}  // namespace

extern "C" {

int nxrt_rocm_ep_supports_rotary_embedding(const NxrtRocmEp*, const NxrtRocmRotaryEmbeddingAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len)
{
    return supported("RotaryEmbedding", reason, reason_len, [&]() -> std::string {
        const RotarySettings s = settings_of(attrs);
        if (!s.problem.empty() || !inputs) return s.problem;
        std::string why = arity(n_inputs, 2, 4);
        if (!why.empty()) return why;
        if (!is_float(inputs[0].dtype)) return std::string("input must have a float dtype, got ") + dtype_name(inputs[0].dtype);
        if (inputs[1].dtype != NXRT_DT_INT64 && inputs[1].dtype != NXRT_DT_INT32) return std::string("position_ids must have dtype Int64 or Int32, got ") + dtype_name(inputs[1].dtype);
        if ((n_inputs > 2 && inputs[2].dtype != 0) != (n_inputs > 3 && inputs[3].dtype != 0)) return "cos_cache and sin_cache go together";
        return {};
    });
}

int nxrt_rocm_ep_supports_cache_append(const NxrtRocmEp*, const NxrtRocmCacheAppendAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len)
{
    return supported("CacheAppend", reason, reason_len, [&]() -> std::string {
        const AppendSettings s = settings_of(attrs);
        if (!s.problem.empty() || !inputs) return s.problem;
        std::string why = arity(n_inputs, 9, 9);
        if (!why.empty()) return why;
        if (!is_float(inputs[0].dtype)) return std::string("key must have a float dtype, got ") + dtype_name(inputs[0].dtype);
        if (inputs[2].dtype != NXRT_DT_INT8 && inputs[2].dtype != NXRT_DT_FLOAT8E4M3FN) return std::string("k_cache must have dtype Int8 or Float8E4M3FN, got ") + dtype_name(inputs[2].dtype);
        return {};
    });
}

int nxrt_rocm_ep_supports_cache_attention(const NxrtRocmEp*, const NxrtRocmCacheAttentionAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len)
{
    return supported("CacheAttention", reason, reason_len, [&]() -> std::string {
        const AttentionSettings s = settings_of(attrs);
        if (!s.problem.empty() || !inputs) return s.problem;
        std::string why = arity(n_inputs, 8, 8);
        if (!why.empty()) return why;
        if (inputs[0].dtype != NXRT_DT_FLOAT16 && inputs[0].dtype != NXRT_DT_BFLOAT16) return std::string("query must have dtype Float16 or BFloat16, got ") + dtype_name(inputs[0].dtype);
        if (inputs[1].dtype != NXRT_DT_INT8 && inputs[1].dtype != NXRT_DT_FLOAT8E4M3FN) return std::string("k_cache must have dtype Int8 or Float8E4M3FN, got ") + dtype_name(inputs[1].dtype);
        return {};
    });
}

int nxrt_rocm_ep_supports_cache_pages(const NxrtRocmEp*, const NxrtRocmCachePagesAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len)
{
    return supported("CachePages", reason, reason_len, [&]() -> std::string {
        const PagesSettings s = settings_of(attrs);
        if (!s.problem.empty() || !inputs) return s.problem;
        std::string why = arity(n_inputs, 5, 4 + ROCM_PAGES_MAX_POOLS);
        if (!why.empty()) return why;
        if (inputs[0].dtype != NXRT_DT_INT32) return std::string("block_table must have dtype Int32, got ") + dtype_name(inputs[0].dtype);
        return {};
    });
}

NxrtStatus nxrt_rocm_rotary_embedding_create(NxrtRocmEp* ep, const NxrtRocmRotaryEmbeddingAttrs* attrs, NxrtRocmNode** out_node)
{
    return create_node<RotaryNode>("RotaryEmbedding", ep, out_node, [&] { return settings_of(attrs); });
}
NxrtStatus nxrt_rocm_cache_append_create(NxrtRocmEp* ep, const NxrtRocmCacheAppendAttrs* attrs, NxrtRocmNode** out_node)
{
    return create_node<AppendNode>("CacheAppend", ep, out_node, [&] { return settings_of(attrs); });
}
NxrtStatus nxrt_rocm_cache_attention_create(NxrtRocmEp* ep, const NxrtRocmCacheAttentionAttrs* attrs, NxrtRocmNode** out_node)
{
    return create_node<AttentionNode>("CacheAttention", ep, out_node, [&] { return settings_of(attrs); });
}
NxrtStatus nxrt_rocm_cache_pages_create(NxrtRocmEp* ep, const NxrtRocmCachePagesAttrs* attrs, NxrtRocmNode** out_node)
{
    return create_node<PagesNode>("CachePages", ep, out_node, [&] { return settings_of(attrs); });
}

}  // extern "C"
