// Part of torch_layer.cpp: the expert products over 4-bit weights and the SwiGLU that keeps its inputs in 8 bits as autograd functions.

constexpr int64_t FP4_GROUP = 32, FP4_GROUP_BYTES = 16;
inline int64_t fp4_groups(int64_t K) { return (K + FP4_GROUP - 1) / FP4_GROUP; }

// (E, K, N) weights -> codes (E, N, groups * 16) and scales (E, N, groups), both uint8
variable_list quantize_weights_fp4(const Tensor& w_)
{
    require_gpu({&w_});
    TORCH_CHECK(w_.dim() == 3, "quantize_expert_weights_fp4 takes (experts, inputs, outputs), got ", w_.sizes());
    const Tensor w = w_.detach();
    const int64_t E = w.size(0), K = w.size(1), N = w.size(2), G = fp4_groups(K);
    const int dt = dtype_code(w);
    const c10::DeviceGuard guard(w.device());
    Tensor codes = at::empty({E, N, G * FP4_GROUP_BYTES}, w.options().dtype(at::kByte)), scales = at::empty({E, N, G}, w.options().dtype(at::kByte));
    if (w.numel() == 0) return {codes, scales};
    check(moe_fp4_quantize_weights(ptr(w), w.stride(0), w.stride(1), w.stride(2), dt, (int)E, K, N, (uint8_t*)ptr(codes), codes.stride(0), codes.stride(1), (uint8_t*)ptr(scales),
                                   scales.stride(0), scales.stride(1), stream_of(w)), "moe_fp4_quantize_weights");
    return {codes, scales};
}

// codes and scales of (E, N, K) weights
struct Fp4W {
    Tensor codes, scales;
    const uint8_t* c() const { return (const uint8_t*)ptr(codes); }
    const uint8_t* s() const { return (const uint8_t*)ptr(scales); }
};

void check_fp4(const Tensor& codes, const Tensor& scales, int64_t K)
{
    TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte, "4-bit weight codes are uint8, two to a byte, got ", codes.scalar_type());
    TORCH_CHECK_TYPE(scales.scalar_type() == at::kByte, "scales of 4-bit weights are uint8 exponents, got ", scales.scalar_type());
    TORCH_CHECK(codes.dim() == 3 && scales.dim() == 3, "4-bit weights are (experts, outputs, bytes) with scales (experts, outputs, groups), got ", codes.sizes(), " and ", scales.sizes());
    TORCH_CHECK(scales.size(0) == codes.size(0) && scales.size(1) == codes.size(1) && scales.size(2) == fp4_groups(K) && codes.size(2) == scales.size(2) * FP4_GROUP_BYTES,
                "codes of ", codes.sizes(), " with scales of ", scales.sizes(), " are not 4-bit weights of ", K, " inputs");
}

// as the kernels read them: rows of codes in 16-byte pieces, a row's scales one after the other
Fp4W take_fp4(const Tensor& codes, const Tensor& scales)
{
    const bool ok = codes.stride(2) == 1 && codes.stride(0) % 16 == 0 && codes.stride(1) % 16 == 0 && (uintptr_t)codes.data_ptr() % 16 == 0;
    // (a copy also where contiguous() would see nothing to do: an odd address, or an odd pitch of a single row)
    return {ok ? codes : codes.clone(at::MemoryFormat::Contiguous), scales.stride(2) == 1 ? scales : scales.contiguous()};
}

Tensor linear_fp4_rows(const Tensor& x, const Fp4W& w, const Tensor& ssi, const Tensor& eo, const LinearCfg& c, bool sums)
{
    const int64_t R = ssi.size(0), E = w.codes.size(0), K = x.size(1), N = w.codes.size(1);
    Tensor y = at::empty({R, N}, x.options().dtype(rows_type(x.scalar_type(), sums)));
    if (R == 0 || N == 0) return y;
    Tensor ws = bytes_on(x, moe_linear_fp4_workspace_bytes(ptr(x), x.stride(0), x.size(0), c.grouped_in, dtype_code(x), w.s(), w.scales.stride(0), w.scales.stride(1), R, (int)E, K, N));
    check(moe_linear_fp4_fwd(ptr(x), x.stride(0), x.size(0), dtype_code(x), w.c(), w.codes.stride(0), w.codes.stride(1), w.s(), w.scales.stride(0), w.scales.stride(1), ptr(y), y.stride(0),
                             dtype_code(y), ptr(ssi), is64(ssi), ptr(eo), is64(eo), (int)E, R, K, N, (int)c.k, c.grouped_in, c.grouped_out, ptr(ws), (size_t)ws.numel(), stream_of(x)),
          "moe_linear_fp4_fwd");
    return y;
}

struct LinearFp4Fn : Function<LinearFp4Fn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& gates_, const Tensor& codes, const Tensor& scales, const Tensor& ssi, const Tensor& eo, const LinearCfg& c)
    {
        const Tensor gates = val(gates_);
        Tensor y = linear_fp4_rows(x, take_fp4(codes, scales), ssi, eo, c, gates.defined()), y_rows;
        if (gates.defined()) {
            y_rows = y;
            y = combine_rows(y_rows, gates, gates.size(1), gates.size(0), x.scalar_type());
        }
        ctx->save_for_backward({codes, scales, gates, ssi, eo, gates.defined() && gates.requires_grad() ? y_rows : Tensor()});
        ctx->saved_data["K"] = x.size(1);
        ctx->saved_data["k"] = c.k;
        ctx->saved_data["flags"] = (int64_t)(c.grouped_in | (c.grouped_out << 1));
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g)
    {
        const auto sv = ctx->get_saved_variables();
        const Tensor& gates = sv[2];
        const c10::DeviceGuard guard(sv[0].device());
        const Fp4W w = take_fp4(sv[0], sv[1]);
        const Tensor ssi = sv[3].contiguous(), eo = sv[4].contiguous();   // (a saved-tensor hook may hand back other strides)
        const int64_t k = ctx->saved_data["k"].toInt(), flags = ctx->saved_data["flags"].toInt(), K = ctx->saved_data["K"].toInt(), E = w.codes.size(0), N = w.codes.size(1), R = ssi.size(0);
        const bool grouped_in = flags & 1, grouped_out = flags & 2;
        const Tensor dout = g[0].contiguous();
        Tensor dx, d_gates;
        int64_t gate_fan = 1;
        if (gates.defined()) {
            gate_fan = gates.size(1);
            if (ctx->needs_input_grad(1)) d_gates = combine_rows_dgates(sv[5].contiguous(), dout, gate_fan, gates.scalar_type());
        }
        if (ctx->needs_input_grad(0)) {
            dx = at::empty({R, K}, dout.options().dtype(rows_type(dout.scalar_type(), k != 1)));
            if (R > 0 && N > 0) {
                const Tensor coeff = flat_gates(gates);
                Tensor ws = bytes_on(dout, moe_linear_fp4_bwd_workspace_bytes(ptr(dout), dout.stride(0), dout.size(0), grouped_out, dtype_code(dout), w.s(),
                                                                              w.scales.stride(0), w.scales.stride(1), R, (int)E, K, N));
                check(moe_linear_fp4_bwd(ptr(dout), dout.stride(0), dout.size(0), dtype_code(dout), grouped_out, (int)gate_fan, ptr(coeff), coeff.defined() ? dtype_code(coeff) : 0, w.c(),
                                         w.codes.stride(0), w.codes.stride(1), w.s(), w.scales.stride(0), w.scales.stride(1), ptr(dx), dx.stride(0), dtype_code(dx), grouped_in, ptr(ssi),
                                         is64(ssi), ptr(eo), is64(eo), (int)E, R, K, N, ptr(ws), (size_t)ws.numel(), stream_of(dout)), "moe_linear_fp4_bwd");
            } else dx.zero_();
            if (k != 1) dx = combine_rows(dx, Tensor(), k, R / k, dout.scalar_type());
        }
        return {dx, d_gates, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor linear_fp4(const Tensor& x_, const Tensor& codes, const Tensor& scales, int64_t k, const Tensor& sei, const Tensor& ssi_, const OptTensor& eo_in, const OptTensor& gates_in,
                  bool grouped_in, bool grouped_out)
{
    const Tensor eo_ = val(eo_in), gates_ = val(gates_in);
    require_gpu({&x_, &codes, &scales, &sei, &ssi_, &eo_, &gates_});
    MOE_ASSERT(x_.dim() == 2, "X has to be (rows, inputs).");
    TORCH_CHECK(x_.size(1) >= 1, "rows of ", x_.sizes(), " hold nothing to multiply");
    check_fp4(codes, scales, x_.size(1));
    TORCH_CHECK(codes.size(0) >= 1, "expert weights of ", codes.sizes(), " hold nothing to multiply by");
    MOE_ASSERT(ssi_.dim() == 1 && sei.dim() == 1 && ssi_.size(0) == sei.size(0), "sorted_scattered_idxs and sorted_expert_idxs differ in length");
    MOE_ASSERT(k >= 1 && ssi_.size(0) == x_.size(0) * k, "the number of assignments is not rows of X times k");
    MOE_ASSERT(!grouped_in || k == 1, "grouped rows of X are one for each assignment: k is 1 with them");
    MOE_ASSERT(!grouped_out || !gates_.defined(), "gates combine rows in token order: not with a grouped output");
    dtype_code(x_);
    is64(ssi_);
    is64(sei);
    if (eo_.defined()) { check_offsets(eo_, codes.size(0)); is64(eo_); }
    check_gates(gates_, ssi_.size(0));
    if (gates_.defined()) dtype_code(gates_);
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = unit_inner(x_), ssi = ssi_.contiguous(), eo = eo_.defined() ? eo_.contiguous() : offsets_from_sorted(sei, codes.size(0));
    const Tensor gates = gates_.defined() ? gates_.contiguous() : Tensor();
    const LinearCfg c{0.0, 0.0, k, grouped_in, grouped_out};
    if (needs_node({&x, &gates})) return LinearFp4Fn::apply(x, opt(gates), codes, scales, ssi, eo, c);
    Tensor y = linear_fp4_rows(x, take_fp4(codes, scales), ssi, eo, c, gates.defined());
    return gates.defined() ? combine_rows(y, gates, gates.size(1), gates.size(0), x.scalar_type()) : y;
}

// ---- SwiGLU with its inputs kept in 8 bits
Tensor swiglu8_forward(const Tensor& gate, const Tensor& up, at::IntArrayRef sizes, Tensor* kept)
{
    const int64_t rows = gate.size(0), cols = gate.size(1);
    Tensor h = at::empty(sizes, gate.options());
    if (kept) *kept = bytes_on(gate, moe_swiglu8_kept_bytes(rows, cols));
    check(moe_swiglu8_fwd(ptr(gate), gate.stride(0), ptr(up), up.stride(0), ptr(h), cols, kept ? ptr(*kept) : nullptr, kept ? (size_t)kept->numel() : 0, rows, cols, dtype_code(gate),
                          stream_of(gate)), "moe_swiglu8_fwd");
    return h;
}

// rows of any pitch whose columns lie one after the other
Tensor as_rows(const Tensor& t) { return unit_inner(t.dim() == 2 ? t : t.reshape({t.numel() / (t.size(-1) ? t.size(-1) : 1), t.size(-1)})); }

struct Swiglu8Fn : Function<Swiglu8Fn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up)
    {
        Tensor kept, h = swiglu8_forward(as_rows(gate), as_rows(up), gate.sizes(), &kept);
        ctx->save_for_backward({kept});
        ctx->saved_data["sizes"] = gate.sizes().vec();
        return h;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g)
    {
        const Tensor kept = ctx->get_saved_variables()[0].contiguous();
        const c10::DeviceGuard guard(kept.device());
        const auto sizes = ctx->saved_data["sizes"].toIntVector();
        const Tensor dh = as_rows(g[0]);
        const int64_t rows = dh.size(0), cols = dh.size(1);
        Tensor dg = at::empty(sizes, dh.options()), du = at::empty(sizes, dh.options());
        check(moe_swiglu8_bwd(ptr(kept), (size_t)kept.numel(), ptr(dh), dh.stride(0), ptr(dg), cols, ptr(du), cols, rows, cols, dtype_code(dh), stream_of(dh)), "moe_swiglu8_bwd");
        return {dg, du};
    }
};

Tensor swiglu_8bit(const Tensor& gate, const Tensor& up)
{
    require_gpu({&gate, &up});
    TORCH_CHECK(gate.dim() >= 1 && gate.sizes() == up.sizes(), "gate of ", gate.sizes(), " and up of ", up.sizes(), " differ in shape");
    MOE_ASSERT(gate.scalar_type() == up.scalar_type(), "gate and up must share a dtype");
    dtype_code(gate);
    const c10::DeviceGuard guard(gate.device());
    return needs_node({&gate, &up}) ? Swiglu8Fn::apply(gate, up) : swiglu8_forward(as_rows(gate), as_rows(up), gate.sizes(), nullptr);
}

// ---- expert MLP and layer: codes and scales in the order w1, w2, w3; w1 and w3 (E, f, d), w2 (E, d, f)
struct Fp4Mlp { Tensor w[3], s[3]; int64_t E, d, f; };

Fp4Mlp take_mlp_fp4(const Tensor& w1, const Tensor& s1, const Tensor& w2, const Tensor& s2, const Tensor& w3, const Tensor& s3, int64_t d)
{
    check_fp4(w1, s1, d);
    const int64_t E = w1.size(0), f = w1.size(1);
    check_fp4(w3, s3, d);
    check_fp4(w2, s2, f);
    TORCH_CHECK(w3.size(0) == E && w3.size(1) == f && w2.size(0) == E && w2.size(1) == d, "4-bit expert weights of ", w1.sizes(), ", ", w2.sizes(), " and ", w3.sizes(), " do not fit ", E,
                " experts of ", f, " x ", d);
    TORCH_CHECK(E >= 1 && f >= 1, "expert weights of ", w1.sizes(), " hold nothing to multiply by");
    return {{w1, w2, w3}, {s1, s2, s3}, E, d, f};
}

struct DecodeOut { Tensor out, weights, indices; };
DecodeOut decode_outputs(const Tensor& x, int64_t k)
{
    const int64_t T = x.size(0);
    return {at::empty({T, x.size(1)}, x.options()), at::empty({T, k}, x.options().dtype(at::kFloat)), at::empty({T, k}, x.options().dtype(at::kInt))};
}

// rows at multiples of 16 bytes, within 32-bit offsets
Tensor aligned_rows(const Tensor& t)
{
    const Tensor u = unit_inner(t);
    const bool ok = (uintptr_t)u.data_ptr() % 16 == 0 && u.stride(0) % 8 == 0 && u.size(0) * u.stride(0) + u.size(1) < (int64_t)1 << 30;
    return ok ? u : u.clone(at::MemoryFormat::Contiguous);
}

// all of it in order, from a multiple of 16 bytes on
Tensor whole(const Tensor& t) { return t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous); }

// what the two launches for a few tokens take
bool decode_takes(int64_t T, int64_t E, int64_t d, int64_t f, int64_t k)
{
    return T <= 16 && E <= 256 && k <= 16 && d % 64 == 0 && f % 64 == 0 && d <= (1 << 20) && f <= (1 << 20) && d * f < (int64_t)1 << 30;
}

void check_layer_input(const Tensor& x, const Tensor& wg, int64_t E, int64_t k)
{
    TORCH_CHECK(x.dim() == 2, "the layer takes (tokens, hidden size), got ", x.sizes());
    TORCH_CHECK(wg.dim() == 2 && wg.size(0) == E && wg.size(1) == x.size(1), "router weight of ", wg.sizes(), " does not fit ", E, " experts of rows of ", x.sizes());
    MOE_ASSERT(wg.scalar_type() == x.scalar_type(), "router weight and X must share a dtype");
    MOE_ASSERT(k >= 1 && k <= E, "top_k must be between 1 and the number of experts");
}

variable_list layer_decode(const Tensor& x_, const Tensor& wg_, const Tensor& w1_, const Tensor& w2_, const Tensor& w3_, int64_t k, bool normalize)
{
    require_gpu({&x_, &wg_, &w1_, &w2_, &w3_});
    TORCH_CHECK(w1_.dim() == 3, "expert weights are (experts, ffn size, hidden size), got ", w1_.sizes());
    const int64_t E = w1_.size(0), f = w1_.size(1), d = w1_.size(2), T = x_.dim() ? x_.size(0) : 0;
    check_layer_input(x_, wg_, E, k);
    for (const Tensor* w : {&w1_, &w2_, &w3_}) {
        TORCH_CHECK(w->dim() == 3, "expert weights are (experts, ffn size, hidden size), got ", w->sizes());
        check_expert_weight(*w, E, f, d);
        MOE_ASSERT(w->scalar_type() == x_.scalar_type(), "X and W must share a dtype");
    }
    TORCH_CHECK_TYPE(x_.scalar_type() == at::kBFloat16 || x_.scalar_type() == at::kHalf, "moe_layer_decode takes bf16 or fp16, got ", x_.scalar_type(), "; use moe_layer_forward for others");
    TORCH_CHECK(!needs_node({&x_, &wg_, &w1_, &w2_, &w3_}), "moe_layer_decode takes no gradients: call it under torch.no_grad(), or use moe_layer_forward");
    TORCH_CHECK(d >= 64 && f >= 64 && decode_takes(T, E, d, f, k), "moe_layer_decode takes up to 16 tokens, 256 experts and 16 experts per token, hidden and ffn sizes that are multiples of 64, and matrices below 2 GiB; got ", T,
                " tokens, ", E, " experts of ", f, " x ", d, ", top ", k, "; use moe_layer_forward for others");
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = aligned_rows(x_), wg = aligned_rows(wg_);
    const Tensor w1 = whole(w1_), w2 = whole(w2_), w3 = whole(w3_);
    DecodeOut o = decode_outputs(x, k);
    if (T == 0) return {o.out, o.weights, o.indices};
    Tensor ws = bytes_on(x, moe_decode_layer_workspace_bytes(T, (int)E, d, f, (int)k, 16));
    check(moe_decode_layer(ptr(x), x.stride(0), ptr(wg), wg.stride(0), dtype_code(x), ptr(w1), ptr(w3), ptr(w2), ptr(o.out), o.out.stride(0), (float*)ptr(o.weights),
                           (int32_t*)ptr(o.indices), T, (int)E, d, f, (int)k, normalize, ptr(ws), (size_t)ws.numel(), stream_of(x)), "moe_decode_layer");
    return {o.out, o.weights, o.indices};
}

// Few tokens without gradients: two launches.
DecodeOut layer_decode_fp4(const Tensor& x_, const Tensor& wg_, const Fp4Mlp& m, int64_t k, bool normalize)
{
    const Tensor x = aligned_rows(x_), wg = aligned_rows(wg_);
    const int64_t T = x.size(0);
    DecodeOut o = decode_outputs(x, k);
    Tensor w[3], s[3];
    for (int i = 0; i < 3; ++i) { w[i] = whole(m.w[i]); s[i] = whole(m.s[i]); }
    auto b = [](const Tensor& t) { return (const uint8_t*)ptr(t); };
    Tensor ws = bytes_on(x, moe_decode_layer_workspace_bytes(T, (int)m.E, m.d, m.f, (int)k, 4));
    check(moe_decode_layer_fp4(ptr(x), x.stride(0), ptr(wg), wg.stride(0), dtype_code(x), b(w[0]), b(s[0]), b(w[2]), b(s[2]), b(w[1]), b(s[1]), ptr(o.out), o.out.stride(0),
                               (float*)ptr(o.weights), (int32_t*)ptr(o.indices), T, (int)m.E, m.d, m.f, (int)k, normalize, ptr(ws), (size_t)ws.numel(), stream_of(x)),
          "moe_decode_layer_fp4");
    return o;
}

// the three projections as autograd nodes of their own; keep8: gate and up are kept in 8 bits
Tensor mlp_fp4(const Tensor& x, const Fp4Mlp& m, int64_t fan_out, const Tensor& ssi, const Tensor& offsets, const Tensor& gates, bool grouped_out, bool keep8)
{
    auto proj = [&](const Tensor& in, int i, const Tensor& g, int64_t k, bool gin, bool gout) {
        const LinearCfg c{0.0, 0.0, k, gin, gout};
        const Tensor xr = unit_inner(in);
        if (needs_node({&xr, &g})) return LinearFp4Fn::apply(xr, opt(g), m.w[i], m.s[i], ssi, offsets, c);
        Tensor y = linear_fp4_rows(xr, take_fp4(m.w[i], m.s[i]), ssi, offsets, c, g.defined());
        return g.defined() ? combine_rows(y, g, g.size(1), g.size(0), xr.scalar_type()) : y;
    };
    const Tensor gate = proj(x, 0, Tensor(), fan_out, false, true), up = proj(x, 2, Tensor(), fan_out, false, true);
    return proj(keep8 ? swiglu_8bit(gate, up) : swiglu(gate, up), 1, gates, 1, true, grouped_out);
}

Tensor expert_mlp_fp4(const Tensor& x, const Tensor& w1, const Tensor& s1, const Tensor& w2, const Tensor& s2, const Tensor& w3, const Tensor& s3, int64_t fan_out, const Tensor& ssi_,
                      const Tensor& offsets_, const OptTensor& gates_in, bool grouped_out, bool keep8)
{
    const Tensor gates_ = val(gates_in);
    require_gpu({&x, &w1, &s1, &w2, &s2, &w3, &s3, &ssi_, &offsets_, &gates_});
    TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1, "the expert MLP takes (rows, hidden size), got ", x.sizes());
    const c10::DeviceGuard guard(x.device());
    const Fp4Mlp m = take_mlp_fp4(w1, s1, w2, s2, w3, s3, x.size(1));
    dtype_code(x);
    check_gates(gates_, ssi_.numel());
    if (gates_.defined()) dtype_code(gates_);
    check_offsets(offsets_, m.E);
    is64(ssi_);
    is64(offsets_);
    TORCH_CHECK(fan_out >= 1 && ssi_.numel() == x.size(0) * fan_out, "positions of ", ssi_.sizes(), " do not fit ", x.size(0), " rows with a fan-out of ", fan_out);
    const Tensor ssi = ssi_.contiguous(), offsets = offsets_.contiguous(), gates = gates_.defined() ? gates_.contiguous() : Tensor();
    return mlp_fp4(x, m, fan_out, ssi, offsets, gates, grouped_out && !gates.defined(), keep8);
}

// router -> experts over 4-bit weights -> weighted sum; returns as layer()
variable_list layer_fp4(const Tensor& x, const Tensor& wg, const Tensor& w1, const Tensor& s1, const Tensor& w2, const Tensor& s2, const Tensor& w3, const Tensor& s3, int64_t k,
                        bool normalize, bool keep8)
{
    require_gpu({&x, &wg, &w1, &s1, &w2, &s2, &w3, &s3});
    TORCH_CHECK(x.dim() == 2 && x.size(1) >= 1, "the layer takes (tokens, hidden size), got ", x.sizes());
    const Fp4Mlp m = take_mlp_fp4(w1, s1, w2, s2, w3, s3, x.size(1));
    check_layer_input(x, wg, m.E, k);
    dtype_code(x);
    const c10::DeviceGuard guard(x.device());
    const bool node = needs_node({&x, &wg});
    if (!node && x.size(0) > 0 && x.scalar_type() != at::kFloat && decode_takes(x.size(0), m.E, m.d, m.f, k)) {
        const DecodeOut o = layer_decode_fp4(x, wg, m, k, normalize);
        return {o.out, o.weights, o.indices};
    }
    RouterOut rt;
    Sorted so;
    if (node) {
        const variable_list r = router(x, wg, k, normalize);
        rt = {r[0], r[1], r[2]};
        so = sort_assignments(rt.indices, m.E);
    } else router_and_sort(unit_inner(x), unit_inner(wg), k, normalize, rt, so);
    const Tensor out = mlp_fp4(x, m, k, so.ints.narrow(0, so.R, so.R), so.ints.narrow(0, 3 * so.R, m.E), rt.weights, false, keep8);
    return {out, rt.weights, rt.indices};
}
