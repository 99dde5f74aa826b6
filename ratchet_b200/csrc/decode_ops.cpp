// Checks of the operators around the Linears: everything a launch relies on, worked out from the description alone.
#include "decode_ops.hpp"

#include <cmath>
#include <initializer_list>

namespace rt {

namespace {

bool activation_dtype(rt_dtype dt) { return dt == RT_F32 || dt == RT_F16 || dt == RT_BF16; }
bool aligned_to(const void *p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

// [rows][d] values of `size` bytes whose rows start `ld` values apart
struct Rows {
    const void *p;
    int64_t rows, d, ld;
    size_t size;
    bool same(const Rows &o) const { return p == o.p && ld == o.ld; }
};

// Whether two operands have a byte in common.  Windows of one wider matrix (equal ld) interleave without touching.
bool overlap(const Rows &a, const Rows &b) {
    if (!a.p || !b.p || a.rows == 0 || b.rows == 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
    const uint64_t an = ((uint64_t)(a.rows - 1) * (uint64_t)a.ld + (uint64_t)a.d) * a.size;
    const uint64_t bn = ((uint64_t)(b.rows - 1) * (uint64_t)b.ld + (uint64_t)b.d) * b.size;
    if (a0 + an <= b0 || b0 + bn <= a0) return false;
    if (a.rows > 1 && b.rows > 1 && a.ld == b.ld && a.size == b.size) {
        const uint64_t pitch = (uint64_t)a.ld * a.size, ad = (uint64_t)a.d * a.size, bd = (uint64_t)b.d * b.size;
        const uint64_t off = b0 >= a0 ? (b0 - a0) % pitch : (pitch - (a0 - b0) % pitch) % pitch; // of b inside a's rows
        if (off >= ad && off + bd <= pitch) return false;
    }
    return true;
}

Status arg(const std::string &m) { return Status::Err(RT_ERR_ARG, m); }

Status check_norm(const rt_norm &n, rt_dtype dt, const char *which) {
    auto name = [&]() { return std::string("rt_residual_norm: ") + which; };
    if (n.kind == RT_NORM_NONE) return Status::Ok();
    if (n.kind != RT_NORM_RMS && n.kind != RT_NORM_LAYER) return arg(name() + ": invalid norm kind");
    if (!(n.eps >= 0.f) || std::isinf(n.eps)) return arg(name() + ": eps must be finite and not negative");
    if (n.weight || n.bias) {
        if (n.dt != RT_F32 && n.dt != dt)
            return Status::Err(RT_ERR_DTYPE, name() + ": weight and bias are F32 or of the activations' type, not " + (dtype_valid(n.dt) ? dtype_name(n.dt) : "?"));
        if (!aligned_to(n.weight, dtype_size(n.dt)) || !aligned_to(n.bias, dtype_size(n.dt))) return arg(name() + ": misaligned weight or bias");
    }
    if (n.bias && n.kind != RT_NORM_LAYER) return arg(name() + ": only a layer norm takes a bias");
    return Status::Ok();
}

} // namespace

Status check_residual_norm(const rt_residual_norm &op) {
    if (!dtype_valid(op.dt)) return arg("rt_residual_norm: invalid dtype enum");
    if (!activation_dtype(op.dt)) return Status::Err(RT_ERR_DTYPE, std::string("rt_residual_norm: no norm of ") + dtype_name(op.dt) + " rows");
    if (op.rows < 0 || op.rows >= (int64_t(1) << 31) || op.d < 1) return Status::Err(RT_ERR_SHAPE, "rt_residual_norm: rows or d out of range");
    if (op.d > RT_NORM_MAX_D)
        return Status::Err(RT_ERR_UNSUPPORTED, "rt_residual_norm: rows of more than " + std::to_string(RT_NORM_MAX_D) + " values");
    for (auto &n : {std::make_pair(&op.post, "post"), std::make_pair(&op.pre, "pre")})
        if (Status st = check_norm(*n.first, op.dt, n.second); !st.ok()) return st;
    if (!op.residual && !op.block) return arg("rt_residual_norm: neither residual nor block");
    if (!op.block && (op.post.kind != RT_NORM_NONE || op.gate)) return arg("rt_residual_norm: a post norm or a gate needs a block");
    if (!op.h && !op.x) return arg("rt_residual_norm: neither h nor x");
    if ((op.x != nullptr) != (op.pre.kind != RT_NORM_NONE)) return arg("rt_residual_norm: x goes with a pre norm");
    const size_t size = dtype_size(op.dt);
    const Rows r{op.residual, op.rows, op.d, op.residual_ld, size}, y{op.block, op.rows, op.d, op.block_ld, size};
    const Rows h{op.h, op.rows, op.d, op.h_ld, size}, x{op.x, op.rows, op.d, op.x_ld, size};
    for (const Rows *v : {&r, &y, &h, &x}) {
        if (!v->p) continue;
        if (v->ld < op.d || v->ld > (int64_t(1) << 40)) return Status::Err(RT_ERR_SHAPE, "rt_residual_norm: rows overlap (ld < d)");
        if (!aligned_to(v->p, size)) return arg("rt_residual_norm: misaligned operand");
    }
    if (op.gate) {
        if (op.gate_rows < 1 || op.rows % op.gate_rows != 0) return Status::Err(RT_ERR_SHAPE, "rt_residual_norm: gate_rows must divide rows");
        if (!aligned_to(op.gate, size)) return arg("rt_residual_norm: misaligned gate");
    }
    if (overlap(h, x)) return Status::Err(RT_ERR_INVARIANT, "rt_residual_norm: h and x overlap");
    const Rows gate{op.gate, op.gate ? op.gate_rows : 0, op.d, op.d, size};
    const Rows constants[] = {gate,
                              {op.post.kind ? op.post.weight : nullptr, 1, op.d, op.d, dtype_valid(op.post.dt) ? dtype_size(op.post.dt) : 0},
                              {op.post.kind ? op.post.bias : nullptr, 1, op.d, op.d, dtype_valid(op.post.dt) ? dtype_size(op.post.dt) : 0},
                              {op.pre.kind ? op.pre.weight : nullptr, 1, op.d, op.d, dtype_valid(op.pre.dt) ? dtype_size(op.pre.dt) : 0},
                              {op.pre.kind ? op.pre.bias : nullptr, 1, op.d, op.d, dtype_valid(op.pre.dt) ? dtype_size(op.pre.dt) : 0}};
    for (const Rows *o : {&h, &x}) {
        for (const Rows *in : {&r, &y})
            if (!o->same(*in) && overlap(*o, *in)) return Status::Err(RT_ERR_INVARIANT, "rt_residual_norm: an output overlaps an input without being it");
        for (const Rows &c : constants)
            if (overlap(*o, c)) return Status::Err(RT_ERR_INVARIANT, "rt_residual_norm: an output overlaps a gate or a weight");
    }
    return Status::Ok();
}

Status check_log_probs(const rt_log_probs &op) {
    if (!dtype_valid(op.dt)) return arg("rt_log_probs: invalid dtype enum");
    if (!activation_dtype(op.dt)) return Status::Err(RT_ERR_DTYPE, std::string("rt_log_probs: no logits of ") + dtype_name(op.dt));
    if (op.rows < 0 || op.rows >= (int64_t(1) << 31) || op.vocab < 1 || op.vocab >= (int64_t(1) << 31))
        return Status::Err(RT_ERR_SHAPE, "rt_log_probs: rows or vocab out of range");
    if (op.ld < op.vocab || op.ld > (int64_t(1) << 40)) return Status::Err(RT_ERR_SHAPE, "rt_log_probs: rows overlap (ld < vocab)");
    if (op.top < 0 || op.top > op.vocab) return Status::Err(RT_ERR_SHAPE, "rt_log_probs: top must lie in 0 .. vocab");
    if (op.top > RT_LOG_PROBS_MAX_TOP)
        return Status::Err(RT_ERR_UNSUPPORTED, "rt_log_probs: more than " + std::to_string(RT_LOG_PROBS_MAX_TOP) + " alternatives");
    if (!op.logits) return arg("rt_log_probs: null logits");
    if ((op.tokens != nullptr) != (op.log_prob != nullptr)) return arg("rt_log_probs: log_prob goes with tokens");
    if ((op.top > 0) != (op.top_ids != nullptr) || (op.top > 0) != (op.top_log_prob != nullptr))
        return arg("rt_log_probs: top_ids and top_log_prob go with top > 0");
    if (!op.log_prob && !op.entropy && op.top == 0) return arg("rt_log_probs: no output");
    if (!aligned_to(op.logits, dtype_size(op.dt))) return arg("rt_log_probs: misaligned logits");
    const Rows outs[] = {{op.log_prob, op.rows, 1, 1, 4}, {op.entropy, op.rows, 1, 1, 4}, {op.top_ids, op.rows, op.top, op.top, 4},
                         {op.top_log_prob, op.rows, op.top, op.top, 4}};
    const Rows logits{op.logits, op.rows, op.vocab, op.ld, dtype_size(op.dt)}, tokens{op.tokens, op.rows, 1, 1, 4};
    if (!aligned_to(op.tokens, 4)) return arg("rt_log_probs: misaligned tokens");
    for (int i = 0; i < 4; i++) {
        if (!aligned_to(outs[i].p, 4)) return arg("rt_log_probs: misaligned output");
        bool bad = overlap(outs[i], logits) || overlap(outs[i], tokens);
        for (int j = 0; j < i; j++) bad = bad || overlap(outs[i], outs[j]);
        if (bad) return Status::Err(RT_ERR_INVARIANT, "rt_log_probs: an output overlaps another operand");
    }
    return Status::Ok();
}

} // namespace rt
