#include "spec.hpp"

#include <cmath>
#include <cstring>

namespace jade {
namespace {

using json::Value;

constexpr uint64_t kIntMax = 2147483647ull;  // i32::MAX, the reference's index bound
// HIP grid limits of the attention launches. Heads: grid.y of the batched
// P.V launch and grid.z of the score launches may not exceed 65535 (the
// online kernel puts heads on grid.x, but all attention ops share the cap).
// Sequence: the online kernel's query blocks (at least 128 queries each) sit
// on grid.y, so seq may not exceed 65535 * 128.
constexpr uint32_t kHipMaxHeads = 65535;
constexpr uint32_t kHipMaxOnlineSeq = 65535u * 128u;

struct OpName {
    const char *tag;
    Op op;
};
constexpr OpName kOps[] = {
    {"elementwise", Op::Elementwise},
    {"axpy", Op::Axpy},
    {"add", Op::Add},
    {"gemm", Op::Gemm},
    {"gemm_simd", Op::GemmSimd},
    {"gemm_mps", Op::GemmMps},
    {"attention_scores", Op::AttentionScores},
    {"attention_apply", Op::AttentionApply},
    {"attention_online", Op::AttentionOnline},
    {"rms_norm", Op::RmsNorm},
    {"swi_glu", Op::SwiGlu},
    {"softmax", Op::Softmax},
    {"rotary", Op::Rotary},
    {"qk_norm_rotary", Op::QkNormRotary},
    {"attention_tree", Op::AttentionTree},
    {"cache_append", Op::CacheAppend},
    {"attention_cross", Op::AttentionCross},
};

const char *tag_of(Op op) {
    for (const auto &o : kOps)
        if (o.op == op) return o.tag;
    return "?";
}

bool get_u32(const Value &obj, const char *key, uint32_t &out, std::string &error) {
    const Value *v = obj.find(key);
    if (!v) { error = std::string("missing field `") + key + "`"; return false; }
    if (!json::as_u32(*v, out)) { error = std::string("field `") + key + "` must be a u32"; return false; }
    return true;
}
bool get_bool(const Value &obj, const char *key, bool &out, std::string &error) {
    const Value *v = obj.find(key);
    if (!v) { error = std::string("missing field `") + key + "`"; return false; }
    if (v->kind != Value::Kind::Bool) { error = std::string("field `") + key + "` must be a boolean"; return false; }
    out = v->boolean;
    return true;
}
bool get_f32(const Value &obj, const char *key, float &out, std::string &error) {
    const Value *v = obj.find(key);
    if (!v) { error = std::string("missing field `") + key + "`"; return false; }
    if (!json::as_f32(*v, out)) { error = std::string("field `") + key + "` must be a number"; return false; }
    return true;
}

// A field that may be left out: `out` keeps its default then.
bool maybe_f32(const Value &obj, const char *key, float &out, std::string &error) {
    return !obj.find(key) || get_f32(obj, key, out, error);
}
bool get_rotation(const Value &obj, KernelSpec &s, std::string &error) {
    return get_u32(obj, "batch", s.batch, error) && get_u32(obj, "seq", s.seq, error) &&
           get_u32(obj, "heads", s.heads, error) && get_u32(obj, "dim", s.dim, error) &&
           get_u32(obj, "rotary_dim", s.rotary_dim, error) && get_bool(obj, "interleaved", s.interleaved, error) &&
           get_bool(obj, "token_major", s.token_major, error) &&
           get_bool(obj, "out_token_major", s.out_token_major, error) && get_f32(obj, "base", s.base, error) &&
           maybe_f32(obj, "factor", s.factor, error) && maybe_f32(obj, "context", s.context, error) &&
           maybe_f32(obj, "low_turns", s.low_turns, error) && maybe_f32(obj, "high_turns", s.high_turns, error) &&
           maybe_f32(obj, "magnitude", s.magnitude, error);
}

bool parse_expr(const Value &v, Expr &out, std::string &error, int depth) {
    // Structural guard only; the reference's depth/node limits apply in validate.
    if (depth > 64) { error = "expression nesting exceeds parser limit"; return false; }
    if (v.kind != Value::Kind::Object) { error = "expression must be an object"; return false; }
    const Value *kind = v.find("kind");
    if (!kind || kind->kind != Value::Kind::String) { error = "expression missing string tag `kind`"; return false; }
    const std::string &k = kind->text;
    auto child = [&](const char *key, std::unique_ptr<Expr> &slot) -> bool {
        const Value *c = v.find(key);
        if (!c) { error = std::string("missing field `") + key + "`"; return false; }
        slot.reset(new Expr);
        return parse_expr(*c, *slot, error, depth + 1);
    };
    if (k == "input") {
        out.kind = Expr::Kind::Input;
        return get_u32(v, "binding", out.binding, error);
    }
    if (k == "constant") {
        out.kind = Expr::Kind::Constant;
        return get_f32(v, "value", out.value, error);
    }
    if (k == "add" || k == "multiply" || k == "maximum") {
        out.kind = k == "add" ? Expr::Kind::Add : k == "multiply" ? Expr::Kind::Multiply : Expr::Kind::Maximum;
        return child("left", out.left) && child("right", out.right);
    }
    if (k == "negate" || k == "exp") {
        out.kind = k == "negate" ? Expr::Kind::Negate : Expr::Kind::Exp;
        return child("value", out.left);
    }
    error = "unknown expression kind `" + k + "`";
    return false;
}

bool expr_validate(const Expr &e, uint32_t inputs, uint32_t depth, uint32_t &nodes, std::string &error) {
    nodes += 1;
    if (!(depth <= kMaxExprDepth && nodes <= kMaxExprNodes)) {
        error = "expression exceeds compiler complexity limit";
        return false;
    }
    switch (e.kind) {
        case Expr::Kind::Input:
            if (!(e.binding < inputs)) { error = "expression input binding out of range"; return false; }
            return true;
        case Expr::Kind::Constant:
            if (!std::isfinite(e.value)) { error = "expression constant must be finite"; return false; }
            return true;
        case Expr::Kind::Add:
        case Expr::Kind::Multiply:
        case Expr::Kind::Maximum:
            return expr_validate(*e.left, inputs, depth + 1, nodes, error) &&
                   expr_validate(*e.right, inputs, depth + 1, nodes, error);
        case Expr::Kind::Negate:
        case Expr::Kind::Exp:
            return expr_validate(*e.left, inputs, depth + 1, nodes, error);
    }
    return false;
}

bool dim_ok(uint64_t v, std::string &error) {
    if (!(v > 0 && v <= kIntMax)) { error = "dimension must be in 1..=INT_MAX"; return false; }
    return true;
}
bool matrix_ok(uint64_t x, uint64_t y, std::string &error) {
    if (!dim_ok(x, error) || !dim_ok(y, error)) return false;
    if (x * y > kIntMax) { error = "tensor exceeds checked 31-bit indexing"; return false; }
    return true;
}

// batch x heads x rows x dim, each at least 1, at most `most` elements.
bool heads_ok(uint64_t batch, uint64_t heads, uint64_t rows, uint64_t dim, uint64_t most, std::string &error) {
    // No factor reaches 2^32, so the checks before each product keep it in 64 bits.
    if (!(batch >= 1 && batch <= kHipMaxHeads)) { error = "batch must be 1..=65535"; return false; }
    if (!(heads >= 1 && heads <= kHipMaxHeads)) { error = "heads and kv_heads must be 1..=65535"; return false; }
    if (!(rows >= 1 && rows <= kIntMax)) { error = "dimension must be in 1..=INT_MAX"; return false; }
    const uint64_t bh = batch * heads;
    if (bh > most / rows || bh * rows > most / dim) {
        error = most == kIntMax ? "tensor exceeds checked 31-bit indexing" : "cache exceeds 2^40 elements";
        return false;
    }
    return true;
}
bool rotation_ok(const KernelSpec &s, std::string &error) {
    if (!(s.dim >= 2 && s.dim <= kMaxRotaryDim)) { error = "rotary head dimension must be 2..=512"; return false; }
    if (!(s.rotary_dim >= 2 && s.rotary_dim <= s.dim && s.rotary_dim % 2 == 0)) {
        error = "rotary_dim must be even and in 2..=dim";
        return false;
    }
    if (!(std::isfinite(s.base) && s.base > 0.0f)) { error = "base must be finite and positive"; return false; }
    if (!(std::isfinite(s.factor) && s.factor > 0.0f)) { error = "factor must be finite and positive"; return false; }
    if (!(std::isfinite(s.magnitude) && s.magnitude > 0.0f)) {
        error = "magnitude must be finite and positive";
        return false;
    }
    if (!(std::isfinite(s.context) && s.context >= 0.0f)) {
        error = "context must be finite and not negative";
        return false;
    }
    if (s.context == 0.0f ? s.low_turns != 0.0f || s.high_turns != 0.0f
                          : !(std::isfinite(s.high_turns) && s.low_turns >= 0.0f && s.low_turns < s.high_turns)) {
        error = "low_turns and high_turns come with a context, and 0 <= low_turns < high_turns";
        return false;
    }
    return true;
}
bool grouped_ok(const KernelSpec &s, std::string &error) {
    if (!(s.dim >= 1 && s.dim <= 128)) { error = "attention head dimension must be 1..=128"; return false; }
    if (!(s.kv_heads >= 1 && s.heads % s.kv_heads == 0)) {
        error = "heads must be a multiple of kv_heads";
        return false;
    }
    return true;
}
bool whole_ok(uint32_t v, const char *name, std::string &error) {
    if (!(v >= 1 && v <= kMaxWhole)) { error = std::string(name) + " must be 1..=16777216"; return false; }
    return true;
}

void expr_json(const Expr &e, std::string &out) {
    switch (e.kind) {
        case Expr::Kind::Input:
            out += "{\"kind\":\"input\",\"binding\":" + std::to_string(e.binding) + "}";
            return;
        case Expr::Kind::Constant:
            out += "{\"kind\":\"constant\",\"value\":" + json::format_f32(e.value) + "}";
            return;
        case Expr::Kind::Add:
        case Expr::Kind::Multiply:
        case Expr::Kind::Maximum:
            out += std::string("{\"kind\":\"") +
                   (e.kind == Expr::Kind::Add ? "add" : e.kind == Expr::Kind::Multiply ? "multiply" : "maximum") +
                   "\",\"left\":";
            expr_json(*e.left, out);
            out += ",\"right\":";
            expr_json(*e.right, out);
            out += "}";
            return;
        case Expr::Kind::Negate:
        case Expr::Kind::Exp:
            out += std::string("{\"kind\":\"") + (e.kind == Expr::Kind::Negate ? "negate" : "exp") + "\",\"value\":";
            expr_json(*e.left, out);
            out += "}";
            return;
    }
}

void lower(const Expr &e, std::vector<Instr> &code) {
    switch (e.kind) {
        case Expr::Kind::Input:
            code.push_back({uint32_t(Opcode::Input), e.binding});
            return;
        case Expr::Kind::Constant: {
            uint32_t bits;
            std::memcpy(&bits, &e.value, sizeof bits);
            code.push_back({uint32_t(Opcode::Constant), bits});
            return;
        }
        case Expr::Kind::Add:
        case Expr::Kind::Multiply:
        case Expr::Kind::Maximum:
            lower(*e.left, code);
            lower(*e.right, code);
            code.push_back({uint32_t(e.kind == Expr::Kind::Add ? Opcode::Add
                                     : e.kind == Expr::Kind::Multiply ? Opcode::Multiply
                                                                      : Opcode::Maximum),
                            0});
            return;
        case Expr::Kind::Negate:
        case Expr::Kind::Exp:
            lower(*e.left, code);
            code.push_back({uint32_t(e.kind == Expr::Kind::Negate ? Opcode::Negate : Opcode::Exp), 0});
            return;
    }
}

}  // namespace

bool parse_spec(const std::string &text, KernelSpec &out, std::string &error) {
    if (text.size() > 65536) { error = "kernel JSON exceeds 64 KiB"; return false; }
    Value root;
    if (!json::parse(text, root, error)) return false;
    if (root.kind != Value::Kind::Object) { error = "kernel spec must be a JSON object"; return false; }
    const Value *tag = root.find("op");
    if (!tag || tag->kind != Value::Kind::String) { error = "missing string tag `op`"; return false; }
    bool known = false;
    for (const auto &o : kOps)
        if (tag->text == o.tag) { out.op = o.op; known = true; }
    if (!known) { error = "unknown variant `" + tag->text + "`"; return false; }
    switch (out.op) {
        case Op::Elementwise: {
            if (!get_u32(root, "len", out.len, error) || !get_u32(root, "inputs", out.inputs, error)) return false;
            const Value *e = root.find("expression");
            if (!e) { error = "missing field `expression`"; return false; }
            auto expr = std::make_shared<Expr>();
            if (!parse_expr(*e, *expr, error, 0)) return false;
            out.expression = expr;
            return true;
        }
        case Op::Axpy:
            return get_u32(root, "len", out.len, error) && get_f32(root, "alpha", out.alpha, error);
        case Op::Add:
        case Op::SwiGlu:
            return get_u32(root, "len", out.len, error);
        case Op::Gemm:
            return get_u32(root, "m", out.m, error) && get_u32(root, "n", out.n, error) &&
                   get_u32(root, "k", out.k, error) && get_bool(root, "tiled", out.tiled, error);
        case Op::GemmSimd:
        case Op::GemmMps:
            return get_u32(root, "m", out.m, error) && get_u32(root, "n", out.n, error) &&
                   get_u32(root, "k", out.k, error);
        case Op::AttentionScores:
        case Op::AttentionOnline:
            return get_u32(root, "heads", out.heads, error) && get_u32(root, "seq", out.seq, error) &&
                   get_u32(root, "dim", out.dim, error) && get_bool(root, "causal", out.causal, error);
        case Op::AttentionApply:
            return get_u32(root, "heads", out.heads, error) && get_u32(root, "seq", out.seq, error) &&
                   get_u32(root, "dim", out.dim, error);
        case Op::RmsNorm:
            return get_u32(root, "rows", out.rows, error) && get_u32(root, "cols", out.cols, error) &&
                   get_f32(root, "epsilon", out.epsilon, error);
        case Op::Softmax:
            return get_u32(root, "rows", out.rows, error) && get_u32(root, "cols", out.cols, error);
        case Op::Rotary:
            return get_rotation(root, out, error) && get_bool(root, "inverse", out.inverse, error);
        case Op::QkNormRotary:
            return get_rotation(root, out, error) && get_u32(root, "kv_heads", out.kv_heads, error) &&
                   get_f32(root, "epsilon", out.epsilon, error);
        case Op::AttentionTree:
            return get_u32(root, "batch", out.batch, error) && get_u32(root, "heads", out.heads, error) &&
                   get_u32(root, "kv_heads", out.kv_heads, error) && get_u32(root, "nodes", out.nodes, error) &&
                   get_u32(root, "capacity", out.capacity, error) && get_u32(root, "dim", out.dim, error) &&
                   get_bool(root, "token_major", out.token_major, error);
        case Op::CacheAppend:
            return get_u32(root, "batch", out.batch, error) && get_u32(root, "kv_heads", out.kv_heads, error) &&
                   get_u32(root, "rows", out.rows, error) && get_u32(root, "picks", out.picks, error) &&
                   get_u32(root, "capacity", out.capacity, error) && get_u32(root, "dim", out.dim, error) &&
                   get_bool(root, "token_major", out.token_major, error);
        case Op::AttentionCross:
            return get_u32(root, "batch", out.batch, error) && get_u32(root, "heads", out.heads, error) &&
                   get_u32(root, "kv_heads", out.kv_heads, error) && get_u32(root, "queries", out.queries, error) &&
                   get_u32(root, "keys", out.keys, error) && get_u32(root, "dim", out.dim, error) &&
                   get_bool(root, "token_major", out.token_major, error);
    }
    return false;
}

const char *spec_name(const KernelSpec &spec) {
    switch (spec.op) {
        case Op::Elementwise: return "elementwise";
        case Op::Axpy: return "axpy";
        case Op::Add: return "add";
        case Op::Gemm: return spec.tiled ? "gemm_register32" : "gemm_naive";
        case Op::GemmSimd: return "gemm_simdgroup_fp32";
        case Op::GemmMps: return "gemm_mps_fp32";
        case Op::AttentionScores: return "attention_scores";
        case Op::AttentionApply: return "attention_apply";
        case Op::AttentionOnline: return "attention_online";
        case Op::RmsNorm: return "rms_norm";
        case Op::SwiGlu: return "swi_glu";
        case Op::Softmax: return "softmax";
        case Op::Rotary: return "rotary";
        case Op::QkNormRotary: return "qk_norm_rotary";
        case Op::AttentionTree: return "attention_tree";
        case Op::CacheAppend: return "cache_append";
        case Op::AttentionCross: return "attention_cross";
    }
    return "?";
}

bool validate(const KernelSpec &s, Rules rules, std::string &error) {
    if (rules == Rules::Reference && s.op >= Op::Rotary) {
        error = std::string(tag_of(s.op)) + " is not an operation of the reference";
        return false;
    }
    switch (s.op) {
        case Op::Elementwise: {
            if (!dim_ok(s.len, error)) return false;
            if (!(s.inputs > 0 && s.inputs <= kMaxElementwiseInputs)) {
                error = "elementwise input count must be 1..8";
                return false;
            }
            if (!s.expression) { error = "missing expression"; return false; }
            uint32_t nodes = 0;
            return expr_validate(*s.expression, s.inputs, 0, nodes, error);
        }
        case Op::Axpy:
            if (!dim_ok(s.len, error)) return false;
            if (!std::isfinite(s.alpha)) { error = "alpha must be finite"; return false; }
            return true;
        case Op::Add:
        case Op::SwiGlu:
            return dim_ok(s.len, error);
        case Op::Gemm:
        case Op::GemmSimd:
        case Op::GemmMps:
            return matrix_ok(s.m, s.k, error) && matrix_ok(s.k, s.n, error) && matrix_ok(s.m, s.n, error);
        case Op::AttentionScores:
        case Op::AttentionApply:
        case Op::AttentionOnline: {
            if (rules == Rules::Reference) {
                if (!(s.heads >= 1 && s.heads <= 32)) { error = "attention heads must be 1..=32"; return false; }
                if (!(s.seq >= 1 && s.seq <= 2048)) { error = "attention sequence must be 1..=2048"; return false; }
                if (!(s.dim >= 1 && s.dim <= 128)) { error = "attention head dimension must be 1..=128"; return false; }
                const uint64_t hs = uint64_t(s.heads) * s.seq;  // cannot exceed u32 under the caps
                return matrix_ok(hs, s.dim, error) && matrix_ok(hs, s.seq, error);
            }
            if (!(s.heads >= 1 && s.heads <= kHipMaxHeads)) { error = "attention heads must be 1..=65535"; return false; }
            if (!(s.seq >= 1)) { error = "attention sequence must be positive"; return false; }
            if (!(s.dim >= 1 && s.dim <= 128)) { error = "attention head dimension must be 1..=128"; return false; }
            const uint64_t hs = uint64_t(s.heads) * s.seq;
            if (!matrix_ok(hs, s.dim, error)) return false;
            if (s.op != Op::AttentionOnline) return matrix_ok(hs, s.seq, error);
            if (s.seq > kHipMaxOnlineSeq) {
                error = "online attention sequence must be at most 8388480 (65535 query blocks of 128)";
                return false;
            }
            return true;
        }
        case Op::RmsNorm:
            if (!matrix_ok(s.rows, s.cols, error)) return false;
            if (!(std::isfinite(s.epsilon) && s.epsilon > 0.0f)) {
                error = "epsilon must be finite and positive";
                return false;
            }
            return true;
        case Op::Softmax:
            return matrix_ok(s.rows, s.cols, error);
        case Op::Rotary:
            return rotation_ok(s, error) && heads_ok(s.batch, s.heads, s.seq, s.dim, kIntMax, error);
        case Op::QkNormRotary:
            if (!rotation_ok(s, error) || !heads_ok(s.batch, s.heads, s.seq, s.dim, kIntMax, error) ||
                !heads_ok(s.batch, s.kv_heads, s.seq, s.dim, kIntMax, error))
                return false;
            if (!(std::isfinite(s.epsilon) && s.epsilon > 0.0f)) {
                error = "epsilon must be finite and positive";
                return false;
            }
            return true;
        case Op::AttentionTree:
            if (!(s.nodes >= 1 && s.nodes <= kMaxTreeNodes)) { error = "nodes must be 1..=256"; return false; }
            return grouped_ok(s, error) && whole_ok(s.capacity, "capacity", error) &&
                   heads_ok(s.batch, s.heads, s.nodes, s.dim, kIntMax, error) &&
                   heads_ok(s.batch, s.kv_heads, s.capacity, s.dim, kMaxCacheElements, error);
        case Op::CacheAppend:
            if (!(s.dim >= 1 && s.dim <= kMaxRotaryDim)) { error = "head dimension must be 1..=512"; return false; }
            return whole_ok(s.rows, "rows", error) && whole_ok(s.picks, "picks", error) &&
                   whole_ok(s.capacity, "capacity", error) && matrix_ok(s.batch, s.picks, error) &&
                   heads_ok(s.batch, s.kv_heads, s.rows, s.dim, kIntMax, error) &&
                   heads_ok(s.batch, s.kv_heads, s.capacity, s.dim, kMaxCacheElements, error);
        case Op::AttentionCross:
            return grouped_ok(s, error) && whole_ok(s.keys, "keys", error) &&
                   heads_ok(s.batch, s.heads, s.queries, s.dim, kIntMax, error) &&
                   heads_ok(s.batch, s.kv_heads, s.keys, s.dim, kMaxCacheElements, error);
    }
    error = "unknown op";
    return false;
}

bool hip_supported(const KernelSpec &spec, std::string &error) {
    if (spec.op == Op::GemmMps) {
        error = "gemm_mps is an Apple MPS library operation; use gemm or gemm_simd on the HIP backend";
        return false;
    }
    return true;
}

std::vector<Binding> bindings(const KernelSpec &s) {
    static const char *kInputNames[] = {"input0", "input1", "input2", "input3",
                                        "input4", "input5", "input6", "input7"};
    const uint64_t hsd = uint64_t(s.heads) * s.seq * s.dim;
    const uint64_t hss = uint64_t(s.heads) * s.seq * s.seq;
    const uint64_t b = s.batch, d = s.dim, kv = b * s.kv_heads * d;
    switch (s.op) {
        case Op::Elementwise: {
            std::vector<Binding> out;
            for (uint32_t i = 0; i < s.inputs && i < kMaxElementwiseInputs; ++i)
                out.push_back({kInputNames[i], s.len, false});
            out.push_back({"out", s.len, true});
            return out;
        }
        case Op::Axpy:
        case Op::Add:
            return {{"a", s.len, false}, {"b", s.len, false}, {"out", s.len, true}};
        case Op::SwiGlu:
            return {{"gate", s.len, false}, {"up", s.len, false}, {"out", s.len, true}};
        case Op::Gemm:
        case Op::GemmSimd:
        case Op::GemmMps:
            return {{"a", uint64_t(s.m) * s.k, false},
                    {"b", uint64_t(s.k) * s.n, false},
                    {"out", uint64_t(s.m) * s.n, true}};
        case Op::AttentionScores:
            return {{"q", hsd, false}, {"k", hsd, false}, {"scores", hss, true}};
        case Op::AttentionApply:
            return {{"probabilities", hss, false}, {"v", hsd, false}, {"out", hsd, true}};
        case Op::AttentionOnline:
            return {{"q", hsd, false}, {"k", hsd, false}, {"v", hsd, false}, {"out", hsd, true}};
        case Op::RmsNorm:
            return {{"x", uint64_t(s.rows) * s.cols, false},
                    {"weight", s.cols, false},
                    {"out", uint64_t(s.rows) * s.cols, true}};
        case Op::Softmax:
            return {{"x", uint64_t(s.rows) * s.cols, false}, {"out", uint64_t(s.rows) * s.cols, true}};
        case Op::Rotary:
            return {{"x", b * s.seq * s.heads * d, false}, {"positions", b * s.seq, false},
                    {"out", b * s.seq * s.heads * d, true}};
        case Op::QkNormRotary:
            return {{"q", b * s.seq * s.heads * d, false}, {"k", kv * s.seq, false}, {"q_weight", d, false},
                    {"k_weight", d, false}, {"positions", b * s.seq, false},
                    {"q_out", b * s.seq * s.heads * d, true}, {"k_out", kv * s.seq, true}};
        case Op::AttentionTree:
            return {{"q", b * s.heads * s.nodes * d, false}, {"k_cache", kv * s.capacity, false},
                    {"v_cache", kv * s.capacity, false}, {"lengths", b, false}, {"k_draft", kv * s.nodes, false},
                    {"v_draft", kv * s.nodes, false}, {"parents", b * s.nodes, false},
                    {"out", b * s.heads * s.nodes * d, true}};
        case Op::CacheAppend:
            return {{"k", kv * s.rows, false}, {"v", kv * s.rows, false}, {"picks", b * s.picks, false},
                    {"lengths", b, false}, {"k_cache", kv * s.capacity, true}, {"v_cache", kv * s.capacity, true},
                    {"new_lengths", b, true}};
        case Op::AttentionCross:
            return {{"q", b * s.heads * s.queries * d, false}, {"k", kv * s.keys, false}, {"v", kv * s.keys, false},
                    {"lengths", b, false}, {"out", b * s.heads * s.queries * d, true}};
    }
    return {};
}

bool validate_bindings(const KernelSpec &spec, const uint64_t *lengths, const uint64_t *ids, size_t count,
                       std::string &error) {
    const auto expected = bindings(spec);
    if (count != expected.size()) {
        error = std::string(spec_name(spec)) + " expects " + std::to_string(expected.size()) + " bindings";
        return false;
    }
    for (size_t i = 0; i < expected.size(); ++i) {
        if (lengths[i] != expected[i].elements) {
            error = std::string(spec_name(spec)) + " binding " + expected[i].name + " expected " +
                    std::to_string(expected[i].elements) + " floats, got " + std::to_string(lengths[i]);
            return false;
        }
        if (expected[i].write) {
            for (size_t j = 0; j < count; ++j) {
                if (i != j && ids[i] == ids[j]) {
                    error = "output binding must not alias another binding";
                    return false;
                }
            }
        }
    }
    return true;
}

std::string canonical_json(const KernelSpec &s) {
    std::string out = std::string("{\"op\":\"") + tag_of(s.op) + "\"";
    auto u = [&](const char *k, uint32_t v) { out += std::string(",\"") + k + "\":" + std::to_string(v); };
    auto b = [&](const char *k, bool v) { out += std::string(",\"") + k + "\":" + (v ? "true" : "false"); };
    auto f = [&](const char *k, float v) { out += std::string(",\"") + k + "\":" + json::format_f32(v); };
    switch (s.op) {
        case Op::Elementwise:
            u("len", s.len);
            u("inputs", s.inputs);
            out += ",\"expression\":";
            if (s.expression) expr_json(*s.expression, out);
            else out += "null";
            break;
        case Op::Axpy: u("len", s.len); f("alpha", s.alpha); break;
        case Op::Add:
        case Op::SwiGlu: u("len", s.len); break;
        case Op::Gemm: u("m", s.m); u("n", s.n); u("k", s.k); b("tiled", s.tiled); break;
        case Op::GemmSimd:
        case Op::GemmMps: u("m", s.m); u("n", s.n); u("k", s.k); break;
        case Op::AttentionScores:
        case Op::AttentionOnline: u("heads", s.heads); u("seq", s.seq); u("dim", s.dim); b("causal", s.causal); break;
        case Op::AttentionApply: u("heads", s.heads); u("seq", s.seq); u("dim", s.dim); break;
        case Op::RmsNorm: u("rows", s.rows); u("cols", s.cols); f("epsilon", s.epsilon); break;
        case Op::Softmax: u("rows", s.rows); u("cols", s.cols); break;
        case Op::Rotary:
        case Op::QkNormRotary:
            u("batch", s.batch); u("seq", s.seq); u("heads", s.heads);
            if (s.op == Op::QkNormRotary) u("kv_heads", s.kv_heads);
            u("dim", s.dim); u("rotary_dim", s.rotary_dim); b("interleaved", s.interleaved);
            if (s.op == Op::Rotary) b("inverse", s.inverse);
            b("token_major", s.token_major); b("out_token_major", s.out_token_major);
            if (s.op == Op::QkNormRotary) f("epsilon", s.epsilon);
            f("base", s.base); f("factor", s.factor); f("context", s.context); f("low_turns", s.low_turns);
            f("high_turns", s.high_turns); f("magnitude", s.magnitude);
            break;
        case Op::AttentionTree:
            u("batch", s.batch); u("heads", s.heads); u("kv_heads", s.kv_heads); u("nodes", s.nodes);
            u("capacity", s.capacity); u("dim", s.dim); b("token_major", s.token_major);
            break;
        case Op::CacheAppend:
            u("batch", s.batch); u("kv_heads", s.kv_heads); u("rows", s.rows); u("picks", s.picks);
            u("capacity", s.capacity); u("dim", s.dim); b("token_major", s.token_major);
            break;
        case Op::AttentionCross:
            u("batch", s.batch); u("heads", s.heads); u("kv_heads", s.kv_heads); u("queries", s.queries);
            u("keys", s.keys); u("dim", s.dim); b("token_major", s.token_major);
            break;
    }
    return out + "}";
}

std::vector<double> rotary_rates(const KernelSpec &s) {
    constexpr double kTau = 6.283185307179586476925286766559;
    std::vector<double> rates;
    for (uint32_t i = 0; i < s.rotary_dim / 2; ++i) {
        const double plain = std::pow(double(s.base), -2.0 * i / s.rotary_dim) / kTau;
        double keep = 0.0;
        if (s.context > 0.0f) {
            keep = (s.context * plain - s.low_turns) / (double(s.high_turns) - s.low_turns);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        }
        rates.push_back(plain * (keep + (1.0 - keep) / s.factor));
    }
    return rates;
}

std::vector<Instr> compile_expression(const Expr &expr) {
    std::vector<Instr> code;
    lower(expr, code);
    return code;
}

}  // namespace jade
