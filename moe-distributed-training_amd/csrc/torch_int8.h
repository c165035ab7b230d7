// Part of torch_layer.cpp: the expert products over 8-bit weights as autograd functions.  The weights are frozen; gradients of the input and of the gate
// weights go straight through the rounding to codes.

constexpr int64_t MAX_SUM = 1 << 17;   // products of codes in one sum of 32 bits, fewer than

inline int64_t code_pitch(int64_t cols) { return (cols + 127) / 128 * 128; }

// Rows that are summed per token stay fp32 until then (sums: whether they are).
inline at::ScalarType rows_type(at::ScalarType dt, bool sums) { return sums ? at::kFloat : dt; }

Tensor combine_rows(const Tensor& y, const Tensor& gates, int64_t k, int64_t T, at::ScalarType dt)
{
    Tensor out = at::empty({T, y.size(1)}, y.options().dtype(dt));
    check(moe_combine_f32((const float*)ptr(y), y.stride(0), ptr(out), out.stride(0), dtype_code(out), ptr(gates), gates.defined() ? dtype_code(gates) : 0, (int)k, T,
                          y.size(1), stream_of(y)), "moe_combine_f32");
    return out;
}

Tensor combine_rows_dgates(const Tensor& y, const Tensor& dout, int64_t k, at::ScalarType dt)
{
    Tensor dg = at::empty({dout.size(0), k}, y.options().dtype(dt));
    check(moe_combine_f32_dgates((const float*)ptr(y), y.stride(0), ptr(dout), dout.stride(0), dtype_code(dout), ptr(dg), dtype_code(dg), (int)k, dout.size(0), y.size(1),
                                 stream_of(y)), "moe_combine_f32_dgates");
    return dg;
}

// (codes (rows, cols), scale (rows)); the codes are a view of whole 128-column pieces
variable_list quantize_rows(const Tensor& x_)
{
    require_gpu({&x_});
    TORCH_CHECK(x_.dim() == 2, "quantize_rows takes (rows, columns), got ", x_.sizes());
    dtype_code(x_);
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = unit_inner(x_.detach());
    const int64_t pitch = code_pitch(x.size(1));   // (0 for rows of no columns: the codes' own stride says 1)
    Tensor q = at::empty({x.size(0), pitch}, x.options().dtype(at::kChar)), scale = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
    check(moe_quantize_rows(ptr(x), x.stride(0), dtype_code(x), (int8_t*)ptr(q), pitch, (float*)ptr(scale), x.size(0), x.size(1), stream_of(x)), "moe_quantize_rows");
    return {q.narrow(1, 0, x.size(1)), scale};
}

// (E, K, N) -> codes (E, K, N) in w's orientation, rows padded to 16 bytes, and scale (E, N)
variable_list quantize_weights(const Tensor& w_)
{
    require_gpu({&w_});
    TORCH_CHECK(w_.dim() == 3, "quantize_expert_weights takes (experts, inputs, outputs), got ", w_.sizes());
    const Tensor w = w_.detach();
    const int64_t E = w.size(0), K = w.size(1), N = w.size(2);
    const int dt = dtype_code(w);
    const c10::DeviceGuard guard(w.device());
    const bool along_k = w.stride(1) < w.stride(2);
    const int64_t inner = along_k ? K : N, pitch = (inner + 15) / 16 * 16;
    Tensor q = at::empty({E, along_k ? N : K, pitch}, w.options().dtype(at::kChar)).narrow(2, 0, inner);
    if (along_k) q = q.transpose(1, 2);
    Tensor scale = at::empty({E, N}, w.options().dtype(at::kFloat));
    if (w.numel() == 0) return {q, scale.zero_()};
    Tensor ws = bytes_on(w, moe_quantize_weights_workspace_bytes((int)E, N));
    check(moe_quantize_weights(ptr(w), w.stride(0), w.stride(1), w.stride(2), dt, (int)E, K, N, (int8_t*)ptr(q), q.stride(0), q.stride(1), q.stride(2),
                               (float*)ptr(scale), ptr(ws), (size_t)ws.numel(), stream_of(w)), "moe_quantize_weights");
    return {q, scale};
}

// codes of weights with the scale of every expert's output columns
void check_codes(const Tensor& q, const Tensor& scale, int64_t E, int64_t N)
{
    TORCH_CHECK_TYPE(q.scalar_type() == at::kChar, "weight codes are int8, got ", q.scalar_type());
    TORCH_CHECK_TYPE(scale.scalar_type() == at::kFloat, "weight scales are float32, got ", scale.scalar_type());
    TORCH_CHECK(!(at::GradMode::is_enabled() && scale.requires_grad()), "weights in 8 bits are frozen: their scales take no gradient");
    TORCH_CHECK(scale.dim() == 2 && scale.size(0) == E && scale.size(1) == N, "weight scales of ", scale.sizes(), " are not one for each of ", E, " experts' ",
                N, " output columns");
}

Tensor linear_int8_rows(const Tensor& x, const Tensor& W, const Tensor& scale, const Tensor& ssi, const Tensor& eo, const LinearCfg& c, bool sums)
{
    const int64_t R = ssi.size(0), E = W.size(0), K = W.size(1), N = W.size(2);
    Tensor y = at::empty({R, N}, x.options().dtype(rows_type(x.scalar_type(), sums)));
    if (R == 0 || N == 0) return y;
    const int8_t* w = (const int8_t*)ptr(W);
    Tensor ws = bytes_on(x, moe_linear_int8_workspace_bytes(w, W.stride(0), W.stride(1), W.stride(2), x.size(0), R, (int)E, K, N));
    check(moe_linear_int8_fwd(ptr(x), x.stride(0), x.size(0), dtype_code(x), w, W.stride(0), W.stride(1), W.stride(2), (const float*)ptr(scale), ptr(y), y.stride(0), dtype_code(y),
                              ptr(ssi), is64(ssi), ptr(eo), is64(eo), (int)E, R, K, N, (int)c.k, c.grouped_in, c.grouped_out, ptr(ws), (size_t)ws.numel(), stream_of(x)),
          "moe_linear_int8_fwd");
    return y;
}

// rows of dx, at their flat positions or grouped
Tensor linear_int8_dx_rows(const Tensor& dout, const Tensor& gates, int64_t gate_fan, const Tensor& W, const Tensor& scale, const Tensor& ssi, const Tensor& eo,
                           bool dy_grouped, bool dx_grouped, bool sums)
{
    const int64_t R = ssi.size(0), E = W.size(0), K = W.size(1), N = W.size(2);
    Tensor dx = at::empty({R, K}, dout.options().dtype(rows_type(dout.scalar_type(), sums)));
    if (R == 0) return dx;
    if (N == 0) return dx.zero_();
    const int8_t* w = (const int8_t*)ptr(W);
    Tensor ws = bytes_on(dout, moe_linear_int8_workspace_bytes(w, W.stride(0), W.stride(2), W.stride(1), R, R, (int)E, N, K));
    check(moe_linear_int8_bwd(ptr(dout), dout.stride(0), dtype_code(dout), dy_grouped, (int)gate_fan, ptr(gates), gates.defined() ? dtype_code(gates) : 0, w,
                              W.stride(0), W.stride(1), W.stride(2), (const float*)ptr(scale), ptr(dx), dx.stride(0), dtype_code(dx), dx_grouped, ptr(ssi), is64(ssi), ptr(eo), is64(eo),
                              (int)E, R, K, N, ptr(ws), (size_t)ws.numel(), stream_of(dout)), "moe_linear_int8_bwd");
    return dx;
}

struct LinearI8Fn : Function<LinearI8Fn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& gates_, const Tensor& W, const Tensor& scale, const Tensor& ssi, const Tensor& eo,
                          const LinearCfg& c)
    {
        const Tensor gates = val(gates_);
        Tensor y = linear_int8_rows(x, W, scale, ssi, eo, c, gates.defined()), y_rows;
        if (gates.defined()) {
            y_rows = y;
            y = combine_rows(y_rows, gates, gates.size(1), gates.size(0), x.scalar_type());
        }
        ctx->save_for_backward({W, scale, gates, ssi, eo, gates.defined() && gates.requires_grad() ? y_rows : Tensor()});
        ctx->saved_data["k"] = c.k;
        ctx->saved_data["flags"] = (int64_t)(c.grouped_in | (c.grouped_out << 1));
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g)
    {
        const auto sv = ctx->get_saved_variables();
        const Tensor &W = sv[0], &gates = sv[2];
        const c10::DeviceGuard guard(W.device());
        const Tensor scale = sv[1].contiguous(), ssi = sv[3].contiguous(), eo = sv[4].contiguous();   // (a saved-tensor hook may hand back other strides)
        const int64_t k = ctx->saved_data["k"].toInt(), flags = ctx->saved_data["flags"].toInt();
        const bool grouped_in = flags & 1, grouped_out = flags & 2;
        const Tensor dout = g[0].contiguous();
        Tensor dx, d_gates;
        int64_t gate_fan = 1;
        if (gates.defined()) {
            gate_fan = gates.size(1);
            if (ctx->needs_input_grad(1)) d_gates = combine_rows_dgates(sv[5].contiguous(), dout, gate_fan, gates.scalar_type());
        }
        if (ctx->needs_input_grad(0)) {
            dx = linear_int8_dx_rows(dout, flat_gates(gates), gate_fan, W, scale, ssi, eo, grouped_out, grouped_in, k != 1);
            if (k != 1) dx = combine_rows(dx, Tensor(), k, dx.size(0) / k, dout.scalar_type());
        }
        return {dx, d_gates, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor linear_int8(const Tensor& x_, const Tensor& W, const Tensor& scale_, int64_t k, const Tensor& sei, const Tensor& ssi_, const OptTensor& eo_in,
                   const OptTensor& gates_in, bool grouped_in, bool grouped_out)
{
    const Tensor eo_ = val(eo_in), gates_ = val(gates_in);
    require_gpu({&x_, &W, &scale_, &sei, &ssi_, &eo_, &gates_});
    MOE_ASSERT(x_.dim() == 2 && W.dim() == 3 && x_.size(1) == W.size(1), "X and W have inconsistent inner dims.");
    MOE_ASSERT(ssi_.dim() == 1 && sei.dim() == 1 && ssi_.size(0) == sei.size(0), "sorted_scattered_idxs and sorted_expert_idxs differ in length");
    MOE_ASSERT(k >= 1 && ssi_.size(0) == x_.size(0) * k, "the number of assignments is not rows of X times k");
    MOE_ASSERT(!grouped_in || k == 1, "grouped rows of X are one for each assignment: k is 1 with them");
    MOE_ASSERT(!grouped_out || !gates_.defined(), "gates combine rows in token order: not with a grouped output");
    check_codes(W, scale_, W.size(0), W.size(2));
    TORCH_CHECK(W.size(0) >= 1 && W.size(1) >= 1, "expert weights of ", W.sizes(), " hold nothing to multiply by");
    dtype_code(x_);
    is64(ssi_);
    is64(sei);
    if (eo_.defined()) { check_offsets(eo_, W.size(0)); is64(eo_); }
    check_gates(gates_, ssi_.size(0));
    if (gates_.defined()) dtype_code(gates_);
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = unit_inner(x_), scale = scale_.contiguous(), ssi = ssi_.contiguous(), eo = eo_.defined() ? eo_.contiguous() : offsets_from_sorted(sei, W.size(0));
    const Tensor gates = gates_.defined() ? gates_.contiguous() : Tensor();
    const LinearCfg c{0.0, 0.0, k, grouped_in, grouped_out};
    TORCH_CHECK(!needs_node({&x}) || W.size(2) < MAX_SUM, "the gradient of X is a sum over the ", W.size(2), " output columns: exact for fewer than ", MAX_SUM);
    if (needs_node({&x, &gates})) return LinearI8Fn::apply(x, opt(gates), W, scale, ssi, eo, c);
    Tensor y = linear_int8_rows(x, W, scale, ssi, eo, c, gates.defined());
    return gates.defined() ? combine_rows(y, gates, gates.size(1), gates.size(0), x.scalar_type()) : y;
}

// ---- expert MLP: codes (E, f, d) and scales in the order w1, w2, w3
struct I8Mlp { Tensor w[3], s[3]; };

Tensor mlp_int8_rows(const Tensor& x, const I8Mlp& m, const MlpCfg& c, const Tensor& ssi, const Tensor& offsets, Tensor* saved, bool sums)
{
    const int64_t E = m.w[0].size(0), f = m.w[0].size(1), d = m.w[0].size(2), R = ssi.numel();
    Tensor y = at::empty({R, d}, x.options().dtype(rows_type(x.scalar_type(), sums)));
    if (R == 0) return y;
    if (saved) *saved = bytes_on(x, moe_mlp_int8_saved_bytes(R, f));
    Tensor ws = bytes_on(x, moe_mlp_int8_workspace_bytes(R, x.size(0), (int)E, d, f, 0));
    auto q = [&](int i) { return (const int8_t*)ptr(m.w[i]); };
    auto s = [&](int i) { return (const float*)ptr(m.s[i]); };
    check(moe_mlp_int8_fwd(ptr(x), x.stride(0), x.size(0), dtype_code(x), q(0), s(0), q(2), s(2), q(1), s(1), ptr(y), y.stride(0), dtype_code(y), ptr(ssi), is64(ssi),
                           ptr(offsets), is64(offsets), (int)E, R, d, f, (int)c.fan_out, c.y_grouped, saved ? ptr(*saved) : nullptr,
                           saved ? (size_t)saved->numel() : 0, ptr(ws), (size_t)ws.numel(), stream_of(x)), "moe_mlp_int8_fwd");
    return y;
}

struct MlpI8Fn : Function<MlpI8Fn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& gates_, const I8Mlp& m, const Tensor& ssi, const Tensor& offsets, const MlpCfg& c)
    {
        const Tensor gates = val(gates_);
        Tensor saved, y = mlp_int8_rows(x, m, c, ssi, offsets, x.requires_grad() ? &saved : nullptr, gates.defined());   // (only dx reads gate and up again)
        Tensor out = gates.defined() ? combine_rows(y, gates, gates.size(1), gates.size(0), x.scalar_type()) : y;
        ctx->save_for_backward({m.w[0], m.w[1], m.w[2], m.s[0], m.s[1], m.s[2], gates, ssi, offsets, saved, gates.defined() && gates.requires_grad() ? y : Tensor()});
        ctx->saved_data["fan_out"] = c.fan_out;
        ctx->saved_data["y_grouped"] = c.y_grouped;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g)
    {
        const auto sv = ctx->get_saved_variables();
        const Tensor& gates = sv[6];
        const c10::DeviceGuard guard(sv[0].device());
        Tensor m[6];   // (a saved-tensor hook may hand back other strides)
        for (int i = 0; i < 6; ++i) m[i] = sv[i].contiguous();
        const Tensor ssi = sv[7].contiguous(), offsets = sv[8].contiguous(), saved = sv[9].defined() ? sv[9].contiguous() : Tensor();
        const int64_t fan_out = ctx->saved_data["fan_out"].toInt(), E = sv[0].size(0), f = sv[0].size(1), d = sv[0].size(2), R = ssi.numel();
        const Tensor dout = g[0].contiguous();
        Tensor dx, d_gates;
        int64_t dy_fan = 1;
        if (gates.defined()) {
            dy_fan = gates.size(1);
            if (ctx->needs_input_grad(1)) d_gates = combine_rows_dgates(sv[10].contiguous(), dout, dy_fan, gates.scalar_type());
        }
        if (ctx->needs_input_grad(0)) {
            Tensor rows = at::empty({R, d}, dout.options().dtype(rows_type(dout.scalar_type(), fan_out != 1)));
            const Tensor coeff = flat_gates(gates);
            Tensor ws = bytes_on(dout, moe_mlp_int8_workspace_bytes(R, R, (int)E, d, f, 1));
            auto q = [&](int i) { return (const int8_t*)ptr(m[i]); };
            auto s = [&](int i) { return (const float*)ptr(m[3 + i]); };
            check(moe_mlp_int8_bwd(ptr(dout), dout.stride(0), dtype_code(dout), ctx->saved_data["y_grouped"].toBool(), (int)dy_fan, ptr(coeff),
                                   gates.defined() ? dtype_code(gates) : 0, q(0), s(0), q(2), s(2), q(1), s(1), ptr(saved), saved.defined() ? (size_t)saved.numel() : 0, ptr(rows), rows.stride(0), dtype_code(rows),
                                   ptr(ssi), is64(ssi), ptr(offsets), is64(offsets), (int)E, R, d, f, ptr(ws), (size_t)ws.numel(), stream_of(dout)),
                  "moe_mlp_int8_bwd");
            dx = fan_out == 1 ? rows : combine_rows(rows, Tensor(), fan_out, R / fan_out, dout.scalar_type());
        }
        return {dx, d_gates, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

I8Mlp take_mlp_int8(const Tensor& w1, const Tensor& s1, const Tensor& w2, const Tensor& s2, const Tensor& w3, const Tensor& s3)
{
    TORCH_CHECK(w1.dim() == 3, "expert codes are (experts, ffn size, hidden size), got ", w1.sizes());
    const int64_t E = w1.size(0), f = w1.size(1), d = w1.size(2);
    for (const Tensor* w : {&w2, &w3}) { TORCH_CHECK(w->dim() == 3, "expert codes are (experts, ffn size, hidden size), got ", w->sizes()); check_expert_weight(*w, E, f, d); }
    check_codes(w1, s1, E, f);
    check_codes(w2, s2, E, d);
    check_codes(w3, s3, E, f);
    TORCH_CHECK(E >= 1 && d >= 64 && f >= 64 && d % 64 == 0 && f % 64 == 0 && w1.is_contiguous() && w2.is_contiguous() && w3.is_contiguous(),
                "the expert MLP over 8-bit weights needs contiguous (E,f,d) codes, d and f multiples of 64; use parallel_linear_int8 for other cases");
    return {{w1, w2, w3}, {s1.contiguous(), s2.contiguous(), s3.contiguous()}};
}

Tensor expert_mlp_int8(const Tensor& x_, const Tensor& w1, const Tensor& s1, const Tensor& w2, const Tensor& s2, const Tensor& w3, const Tensor& s3,
                       int64_t fan_out, const Tensor& ssi_, const Tensor& offsets_, const OptTensor& gates_in, bool grouped_out)
{
    const Tensor gates_ = val(gates_in);
    require_gpu({&x_, &w1, &s1, &w2, &s2, &w3, &s3, &ssi_, &offsets_, &gates_});
    const c10::DeviceGuard guard(x_.device());
    const I8Mlp m = take_mlp_int8(w1, s1, w2, s2, w3, s3);
    check_gates(gates_, ssi_.numel());
    if (gates_.defined()) dtype_code(gates_);
    check_offsets(offsets_, w1.size(0));
    is64(ssi_);
    is64(offsets_);
    TORCH_CHECK(x_.dim() == 2 && x_.size(1) == w1.size(2), "rows of ", x_.sizes(), " do not fit expert weights of ", w1.sizes());
    TORCH_CHECK_TYPE(x_.scalar_type() == at::kBFloat16 || x_.scalar_type() == at::kHalf, "fused_expert_mlp_int8 takes bf16 or fp16 rows, got ", x_.scalar_type(),
                     "; use parallel_linear_int8 for others");
    const bool grouped = grouped_out && !gates_.defined();
    TORCH_CHECK(fan_out >= 1 && (grouped || ssi_.numel() <= x_.size(0) * fan_out), "positions of ", ssi_.sizes(), " do not fit ", x_.size(0),
                " rows with a fan-out of ", fan_out);
    const Tensor x = unit_inner(x_), ssi = ssi_.contiguous(), offsets = offsets_.contiguous(), gates = gates_.defined() ? gates_.contiguous() : Tensor();
    const MlpCfg c{0.0, fan_out, grouped};
    if (needs_node({&x, &gates})) {
        // rows of dx lie at their positions: each is written once only where the positions are a permutation of all of x's assignments
        TORCH_CHECK(ssi.numel() == x.size(0) * fan_out, "gradients need one position for each of the ", x.size(0) * fan_out, " assignments, got ", ssi.numel());
        TORCH_CHECK(!needs_node({&x}) || 2 * w1.size(1) < MAX_SUM, "the gradient of x is a sum over twice the ", w1.size(1), " ffn columns: exact for fewer than ", MAX_SUM);
        return MlpI8Fn::apply(x, opt(gates), m, ssi, offsets, c);
    }
    Tensor y = mlp_int8_rows(x, m, c, ssi, offsets, nullptr, gates.defined());
    return gates.defined() ? combine_rows(y, gates, gates.size(1), gates.size(0), x.scalar_type()) : y;
}

// router -> sort -> expert MLP over 8-bit weights -> weighted combine; returns as layer()
variable_list layer_int8(const Tensor& x, const Tensor& wg, const Tensor& w1, const Tensor& s1, const Tensor& w2, const Tensor& s2, const Tensor& w3, const Tensor& s3,
                         int64_t k, bool normalize)
{
    require_gpu({&x, &wg, &w1, &s1, &w2, &s2, &w3, &s3});
    TORCH_CHECK(x.dim() == 2, "the layer takes (tokens, hidden size), got ", x.sizes());
    const int64_t E = w1.dim() ? w1.size(0) : 0;
    TORCH_CHECK(wg.dim() == 2 && wg.size(0) == E && wg.size(1) == x.size(1), "router weight of ", wg.sizes(), " does not fit ", E, " experts of rows of ", x.sizes());
    MOE_ASSERT(wg.scalar_type() == x.scalar_type(), "router weight and X must share a dtype");
    const c10::DeviceGuard guard(x.device());
    RouterOut rt;
    Sorted so;
    if (needs_node({&x, &wg})) {
        const variable_list r = router(x, wg, k, normalize);
        rt = {r[0], r[1], r[2]};
        so = sort_assignments(rt.indices, E);
    } else {
        const Tensor xi = unit_inner(x);
        router_and_sort(xi, unit_inner(wg), k, normalize, rt, so);
    }
    const Tensor out = expert_mlp_int8(x, w1, s1, w2, s2, w3, s3, k, so.ints.narrow(0, so.R, so.R), so.ints.narrow(0, 3 * so.R, E), opt(rt.weights), false);
    return {out, rt.weights, rt.indices};
}
