// The host path of qk_norm_rotary and cross_attention (part of host.cpp): as for the layer, from Python's call to the kernels' launches, and one
// autograd node for a training forward.  A step of single tokens is a launch or two of a few microseconds; through the operator dispatcher, a
// foreign-function call and an autograd function of Python's a call took 25 us and a training step 150 to 200.  None for anything that is not
// of a kind the kernels take as it is: the Python functions then check it, with their own errors.

// What a graph through the operators' gradients (create_graph) ends in.
struct NoSecondGradient : public torch::autograd::Node {
    std::string name() const override { return "NoSecondGradient"; }
    variable_list apply(variable_list &&) override {
        TORCH_CHECK(false, "lookupffn_amd: the gradients of qk_norm_rotary and cross_attention cannot be differentiated (a graph through them was "
                           "asked for with create_graph)");
    }
};

// Gradients that a graph is recorded through end in one that raises.
void end_graph(torch::autograd::Node &node, const variable_list &grads, variable_list &out) {
    auto end = std::shared_ptr<NoSecondGradient>(new NoSecondGradient(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges = node.next_edges();
    for (const Tensor &g : grads)
        if (g.defined())
            for (auto &e : torch::autograd::collect_next_edges(g)) edges.push_back(std::move(e));
    end->set_next_edges(std::move(edges));
    for (Tensor &t : out)
        if (t.defined()) torch::autograd::set_history(t, end);
}

int32_t format_of(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: return -1;
    }
}

bool aligned(const Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

Tensor aligned_contiguous(const Tensor &t) {
    const Tensor c = t.contiguous();
    return aligned(c) ? c : c.clone();
}

// [B, L, heads, columns] as the kernels read it, a copy where it has to be; near, if not 0: 128 tokens of so many neighbouring heads within 32 bits.
Tensor head_rows(const Tensor &t, int64_t near = 0) {
    if (near && ((t.size(1) > 1 && t.stride(1) * t.element_size() >= int64_t(1) << 25) ||
                 (near > 1 && t.stride(2) * near * t.element_size() >= int64_t(1) << 30)))
        return aligned_contiguous(t);
    bool as_it_is = (t.stride(3) == 1 || t.size(3) == 1) && aligned(t);
    for (int d = 0; d < 3; ++d) as_it_is = as_it_is && (t.size(d) <= 1 || t.stride(d) * t.element_size() % 16 == 0);
    return as_it_is ? t : aligned_contiguous(t);
}

// What hooks on saved tensors gave back has the type and shape of what was saved: the kernels' reads go by one array's.
constexpr const char *OTHER = "lookupffn_amd: a hook on saved tensors gave back one of another type or shape";
bool alike(const Tensor &a, const Tensor &b) { return a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes() && a.device() == b.device(); }
bool heads_of(const Tensor &t, const Tensor &q) {
    return t.dim() == 4 && t.scalar_type() == q.scalar_type() && t.size(0) == q.size(0) && t.size(3) == q.size(3) && t.numel() > 0 && t.device() == q.device();
}

Tensor neighbours_together(const Tensor &t) {
    return !t.defined() || t.size(t.dim() - 1) <= 1 || t.stride(t.dim() - 1) == 1 ? t : t.contiguous();
}

void head_strides(const Tensor &t, int64_t (&s)[3]) {
    for (int d = 0; d < 3; ++d) s[d] = t.size(d) <= 1 ? 0 : t.stride(d);
}

// An argument that may be None; false where it is neither that nor an ordinary tensor on the device.
bool optional_tensor(PyObject *o, const at::Device &dev, Tensor &t) {
    if (o == Py_None) return true;
    if (!plain(o)) return false;
    t = THPVariable_Unpack(o);
    return t.device() == dev;
}

bool any_tangent(std::initializer_list<const Tensor *> tensors) {
    if (!forward_mode()) return false;
    for (const Tensor *t : tensors)
        if (has_tangent(*t)) return true;
    return false;
}

bool any_gradient(std::initializer_list<const Tensor *> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// A backward that is captured must not meet a leaf whose gradient accumulates on another stream, as it does while a graph from before the capture holds it: the
// engine then has the captured stream wait for that one, and the process ends in its thread.  Refused here, where it can be raised.
void refuse_foreign_leaves(std::initializer_list<const Tensor *> tensors, const at::Device &dev) {
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(static_cast<hipStream_t>(stream_on(dev)), &capture) != hipSuccess || capture == hipStreamCaptureStatusNone) return;
    const c10::Stream now = c10::impl::VirtualGuardImpl(dev.type()).getStream(dev);
    for (const Tensor *t : tensors) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        TORCH_CHECK(!node || !node->stream() || *node->stream() == now,
                    "lookupffn_amd: this forward is captured, but a graph from before the capture still holds one of its leaves: drop that graph's results first");
    }
}

// refuse_foreign_leaves(tensors or None ...): the same in front of Python's autograd functions
PyObject *refuse_foreign_leaves(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    for (Py_ssize_t i = 0; i < n; ++i) {
        if (!THPVariable_Check(args[i])) continue;
        const Tensor &t = THPVariable_Unpack(args[i]);
        if (ordinary(t)) refuse_foreign_leaves({&t}, t.device());
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// Queries or keys: four dimensions, a format, not empty.
bool heads_tensor(PyObject *o, Tensor &t) {
    if (!plain(o)) return false;
    t = THPVariable_Unpack(o);
    return t.dim() == 4 && t.numel() > 0 && format_of(t) >= 0;
}

// ---------------------------------------------------------------- norms and rotation

struct NormInputs {
    Tensor q, k, q_weight, k_weight, table, q_positions, k_positions;
    double eps = 0;
    bool interleaved = false;

    // as the kernels read them; q and k stay what they are for the graph
    void lay_out() {
        q = head_rows(q);
        if (k.defined()) k = head_rows(k);
        for (Tensor *t : {&q_weight, &k_weight, &table})
            if (t->defined()) *t = aligned_contiguous(*t);
        q_positions = neighbours_together(q_positions);
        k_positions = neighbours_together(k_positions);
    }

    lffn_qk_norm_rotary arguments() const {
        lffn_qk_norm_rotary a{};
        a.q = q.data_ptr();
        a.q_weight = f32(q_weight);
        a.B = q.size(0); a.q_len = q.size(1); a.q_heads = q.size(2); a.columns = q.size(3);
        head_strides(q, a.q_strides);
        a.eps = (float)eps;
        a.format = format_of(q);
        a.interleaved = interleaved;
        if (k.defined()) {
            a.k = k.data_ptr();
            a.k_weight = f32(k_weight);
            a.k_len = k.size(1); a.k_heads = k.size(2);
            head_strides(k, a.k_strides);
        }
        if (table.defined()) {
            a.table = f32(table);
            a.table_rows = table.size(0); a.rotary = table.size(1);
            auto place = [&](const Tensor &p, const void *&at, int64_t &stride) {
                if (!p.defined()) return;
                at = p.data_ptr();
                stride = p.dim() == 2 && p.size(0) > 1 ? p.stride(0) : 0;
                a.positions_64 = p.scalar_type() == at::kLong;
            };
            place(q_positions, a.q_positions, a.q_positions_stride);
            place(k_positions, a.k_positions, a.k_positions_stride);
        }
        return a;
    }
};

bool norm_weight(const Tensor &w, const Tensor &t) {
    return !w.defined() || (w.dim() == 1 && w.size(0) == t.size(3) && w.scalar_type() == at::kFloat);
}

bool norm_positions(const Tensor &p, const Tensor &t) {
    if (!p.defined()) return true;
    if (p.scalar_type() != at::kLong && p.scalar_type() != at::kInt) return false;
    return p.dim() == 1 ? p.size(0) == t.size(1) : p.dim() == 2 && p.size(0) == t.size(0) && p.size(1) == t.size(1);
}

struct QkNormRotaryBackward : public torch::autograd::Node {
    SavedVariable q, k, q_weight, k_weight, table, q_positions, k_positions;
    double eps = 0;
    bool interleaved = false;

    std::string name() const override { return "QkNormRotaryBackward"; }

    void release_variables() override {
        for (SavedVariable *v : {&q, &k, &q_weight, &k_weight, &table, &q_positions, &k_positions}) v->reset_data();
    }

    variable_list apply(variable_list &&grads) override {
        const bool graph = at::GradMode::is_enabled();
        variable_list out = gradients(grads);
        if (graph) end_graph(*this, grads, out);
        return out;
    }

    static void fit(const NormInputs &in, const variable_list &grads) {
        TORCH_CHECK(heads_of(in.q, in.q) && (!in.k.defined() || heads_of(in.k, in.q)) && (!grads[0].defined() || alike(in.q, grads[0])) &&
                        (!grads[1].defined() || (in.k.defined() && alike(in.k, grads[1]))) && norm_weight(in.q_weight, in.q) && norm_weight(in.k_weight, in.q) &&
                        (!in.table.defined() || (in.table.dim() == 2 && in.table.scalar_type() == at::kFloat)) && norm_positions(in.q_positions, in.q) &&
                        (!in.k_positions.defined() || (in.k.defined() && norm_positions(in.k_positions, in.k))) &&
                        (!in.q_positions.defined() || !in.k_positions.defined() || in.q_positions.scalar_type() == in.k_positions.scalar_type()), OTHER);
    }

    variable_list gradients(const variable_list &grads) {
        variable_list out(4);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        at::AutoGradMode no_grad(false);
        const auto self = shared_from_this();
        NormInputs in{q.unpack(self), k.unpack(self), q_weight.unpack(self), k_weight.unpack(self), table.unpack(self), q_positions.unpack(self),
                      k_positions.unpack(self), eps, interleaved};
        const at::Device dev = in.q.device();
        const c10::DeviceGuard guard(dev);
        void *st = stream_on(dev);
        fit(in, grads);
        in.lay_out();
        const lffn_qk_norm_rotary a = in.arguments();
        const Tensor g_q = grads[0].defined() ? aligned_contiguous(grads[0]) : at::zeros(in.q.sizes(), in.q.options());
        Tensor g_k;
        out[0] = at::empty(in.q.sizes(), in.q.options());
        if (in.k.defined()) {
            g_k = grads[1].defined() ? aligned_contiguous(grads[1]) : at::zeros(in.k.sizes(), in.k.options());
            out[1] = at::empty(in.k.sizes(), in.k.options());
        }
        if (in.q_weight.defined() && task_should_compute_output(2)) out[2] = empty_f32({a.columns}, dev);
        if (in.k_weight.defined() && task_should_compute_output(3)) out[3] = empty_f32({a.columns}, dev);
        int64_t bytes = 0;
        CALL(lffn_qk_norm_rotary_bwd_workspace_bytes, &a, &bytes);
        const Tensor ws = empty_bytes(bytes, dev);
        CALL(lffn_qk_norm_rotary_bwd, &a, g_q.data_ptr(), g_k.defined() ? g_k.data_ptr() : nullptr, out[0].data_ptr(),
             out[1].defined() ? out[1].data_ptr() : nullptr, f32(out[2]), f32(out[3]), ws.data_ptr(), bytes, st);
        return out;
    }
};

// qk_norm_rotary(q, k, q_weight, k_weight, table, q_positions, k_positions, eps, interleaved) -> (q, k or None), or None: not for this path
PyObject *qk_norm_rotary(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 9, "qk_norm_rotary: 9 arguments");
    NormInputs in;
    if (watched_over() || !heads_tensor(args[0], in.q)) Py_RETURN_NONE;
    const at::Device dev = in.q.device();
    if (c10::hip::current_device() != dev.index()) Py_RETURN_NONE;
    Tensor *const rest[] = {&in.k, &in.q_weight, &in.k_weight, &in.table, &in.q_positions, &in.k_positions};
    for (int i = 0; i < 6; ++i)
        if (!optional_tensor(args[1 + i], dev, *rest[i])) Py_RETURN_NONE;
    const int interleaved = PyObject_IsTrue(args[8]);
    if (interleaved < 0) return nullptr;
    in.interleaved = interleaved;
    if (!number(args[7], in.eps) || !(in.eps >= 0)) Py_RETURN_NONE;
    const int64_t columns = in.q.size(3);
    if (columns % 8 != 0 || columns > 256 || !norm_weight(in.q_weight, in.q) || !norm_positions(in.q_positions, in.q)) Py_RETURN_NONE;
    if (in.k.defined()) {
        if (in.k.dim() != 4 || in.k.numel() == 0 || in.k.scalar_type() != in.q.scalar_type() || in.k.size(0) != in.q.size(0) ||
            in.k.size(3) != columns || !norm_weight(in.k_weight, in.k) || !norm_positions(in.k_positions, in.k))
            Py_RETURN_NONE;
        if (in.q_positions.defined() && in.k_positions.defined() && in.q_positions.scalar_type() != in.k_positions.scalar_type()) Py_RETURN_NONE;
    } else {
        in.k_weight.reset();
        in.k_positions.reset();
    }
    if (in.table.defined() && (in.table.dim() != 2 || in.table.scalar_type() != at::kFloat || in.table.size(0) < 1 || in.table.size(1) < 16 ||
                               in.table.size(1) % 16 != 0 || in.table.size(1) > columns || in.table.requires_grad()))
        Py_RETURN_NONE;
    if (any_tangent({&in.q, &in.k, &in.q_weight, &in.k_weight, &in.table})) Py_RETURN_NONE;
    const bool grads = any_gradient({&in.q, &in.k, &in.q_weight, &in.k_weight});
    if (grads) refuse_foreign_leaves({&in.q, &in.k, &in.q_weight, &in.k_weight}, dev);
    Tensor q_out, k_out;
    {
        const WithoutInterpreter unlocked;
        at::AutoGradMode no_grad(false);
        NormInputs laid = in;
        laid.lay_out();
        const lffn_qk_norm_rotary a = laid.arguments();
        q_out = at::empty(in.q.sizes(), in.q.options());
        if (in.k.defined()) k_out = at::empty(in.k.sizes(), in.k.options());
        CALL(lffn_qk_norm_rotary_fwd, &a, q_out.data_ptr(), k_out.defined() ? k_out.data_ptr() : nullptr, stream_on(dev));
        if (grads) {
            auto node = std::shared_ptr<QkNormRotaryBackward>(new QkNormRotaryBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(in.q, in.k, in.q_weight, in.k_weight));
            node->eps = in.eps;
            node->interleaved = in.interleaved;
            node->q = SavedVariable(in.q, false);
            node->k = SavedVariable(in.k, false);
            node->q_weight = SavedVariable(in.q_weight, false);
            node->k_weight = SavedVariable(in.k_weight, false);
            node->table = SavedVariable(in.table, false);
            node->q_positions = SavedVariable(in.q_positions, false);
            node->k_positions = SavedVariable(in.k_positions, false);
            torch::autograd::set_history(q_out, node);
            if (k_out.defined()) torch::autograd::set_history(k_out, node);
            else node->add_input_metadata(torch::autograd::Node::undefined_input());
        }
    }
    PyObject *const q_object = THPVariable_Wrap(std::move(q_out));
    if (!q_object) return nullptr;
    PyObject *k_object = Py_None;
    if (k_out.defined()) k_object = THPVariable_Wrap(std::move(k_out));
    else Py_INCREF(Py_None);
    if (!k_object) {
        Py_DECREF(q_object);
        return nullptr;
    }
    PyObject *const both = PyTuple_New(2);
    if (!both) {
        Py_DECREF(q_object);
        Py_DECREF(k_object);
        return nullptr;
    }
    PyTuple_SET_ITEM(both, 0, q_object);
    PyTuple_SET_ITEM(both, 1, k_object);
    return both;
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- attention

struct AttentionInputs {
    Tensor q, k, v, mask;
    double scale = 0;

    void lay_out() {
        q = head_rows(q, q.size(2) / k.size(2));          // (the heads that share a key head)
        k = head_rows(k, 1);
        v = head_rows(v, 1);
        mask = neighbours_together(mask);
    }

    lffn_cross_attention arguments() const {
        lffn_cross_attention a{};
        a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
        a.B = q.size(0); a.q_len = q.size(1); a.heads = q.size(2); a.columns = q.size(3);
        a.k_len = k.size(1); a.key_heads = k.size(2);
        head_strides(q, a.q_strides);
        head_strides(k, a.k_strides);
        head_strides(v, a.v_strides);
        if (mask.defined()) {
            a.key_mask = static_cast<const uint8_t *>(mask.data_ptr());
            a.mask_stride = mask.size(0) <= 1 ? 0 : mask.stride(0);
        }
        a.scale = (float)scale;
        a.format = format_of(q);
        return a;
    }
};

struct CrossAttentionBackward : public torch::autograd::Node {
    SavedVariable q, k, v, mask, result, kept;
    double scale = 0;

    std::string name() const override { return "CrossAttentionBackward"; }

    void release_variables() override {
        for (SavedVariable *s : {&q, &k, &v, &mask, &result, &kept}) s->reset_data();
    }

    variable_list apply(variable_list &&grads) override {
        const bool graph = at::GradMode::is_enabled();
        variable_list out = gradients(grads);
        if (graph) end_graph(*this, grads, out);
        return out;
    }

    variable_list gradients(const variable_list &grads) {
        variable_list out(3);
        if (!grads[0].defined()) return out;
        at::AutoGradMode no_grad(false);
        const auto self = shared_from_this();
        AttentionInputs in{q.unpack(self), k.unpack(self), v.unpack(self), mask.unpack(self), scale};
        // (hooks on saved tensors may have laid out anew what the forward left contiguous)
        const Tensor result_ = aligned_contiguous(result.unpack(self)), kept_ = aligned_contiguous(kept.unpack(self)), g = aligned_contiguous(grads[0]);
        const at::Device dev = in.q.device();
        const c10::DeviceGuard guard(dev);
        void *st = stream_on(dev);
        TORCH_CHECK(alike(in.q, g) && heads_of(in.q, in.q) && heads_of(in.k, in.q) && alike(in.v, in.k) && in.q.size(2) % in.k.size(2) == 0 && alike(result_, in.q) &&
                        kept_.scalar_type() == at::kByte && kept_.dim() == 1 && kept_.device() == dev &&
                        (!in.mask.defined() || (in.mask.scalar_type() == at::kBool && in.mask.sizes() == in.k.sizes().slice(0, 2))), OTHER);
        in.lay_out();
        const lffn_cross_attention a = in.arguments();
        const bool of_keys = task_should_compute_output(1) || task_should_compute_output(2);
        if (task_should_compute_output(0)) out[0] = at::empty(in.q.sizes(), in.q.options());
        if (of_keys) {
            out[1] = at::empty(in.k.sizes(), in.k.options());
            out[2] = at::empty(in.v.sizes(), in.v.options());
        }
        int64_t bytes = 0;
        CALL(lffn_cross_attention_kept_bytes, &a, &bytes);
        TORCH_CHECK(kept_.numel() == bytes, OTHER);
        CALL(lffn_cross_attention_bwd_workspace_bytes, &a, &bytes);
        const Tensor ws = empty_bytes(bytes, dev);
        CALL(lffn_cross_attention_bwd, &a, result_.data_ptr(), kept_.data_ptr(), g.data_ptr(), out[0].defined() ? out[0].data_ptr() : nullptr,
             of_keys ? out[1].data_ptr() : nullptr, of_keys ? out[2].data_ptr() : nullptr, ws.data_ptr(), bytes, st);
        return out;
    }
};

// cross_attention(q, k, v, key_mask, scale or None) -> a tensor, or None: not for this path
PyObject *cross_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 5, "cross_attention: 5 arguments");
    AttentionInputs in;
    if (watched_over() || !heads_tensor(args[0], in.q) || !heads_tensor(args[1], in.k) || !heads_tensor(args[2], in.v)) Py_RETURN_NONE;
    const at::Device dev = in.q.device();
    if (c10::hip::current_device() != dev.index() || in.k.device() != dev || in.v.device() != dev || !optional_tensor(args[3], dev, in.mask))
        Py_RETURN_NONE;
    const int64_t columns = in.q.size(3);
    if (args[4] == Py_None) in.scale = 1.0 / std::sqrt((double)columns);
    else if (!number(args[4], in.scale)) Py_RETURN_NONE;
    const auto type = in.q.scalar_type();
    if (!((float)in.scale > 0.f && (float)in.scale <= 3.4e38f) || in.k.scalar_type() != type || in.v.scalar_type() != type ||
        in.k.size(0) != in.q.size(0) || in.k.size(3) != columns || in.v.sizes() != in.k.sizes() || columns % 8 != 0 || columns > 128 ||
        in.q.size(2) % in.k.size(2) != 0)
        Py_RETURN_NONE;
    if (in.mask.defined() && (in.mask.scalar_type() != at::kBool || in.mask.dim() != 2 || in.mask.size(0) != in.k.size(0) ||
                              in.mask.size(1) != in.k.size(1)))
        Py_RETURN_NONE;
    if (any_tangent({&in.q, &in.k, &in.v})) Py_RETURN_NONE;
    const bool grads = any_gradient({&in.q, &in.k, &in.v});
    if (grads) refuse_foreign_leaves({&in.q, &in.k, &in.v}, dev);
    Tensor out;
    {
        const WithoutInterpreter unlocked;
        at::AutoGradMode no_grad(false);
        AttentionInputs laid = in;
        laid.lay_out();
        const lffn_cross_attention a = laid.arguments();
        out = at::empty(in.q.sizes(), in.q.options());
        Tensor kept, ws;
        int64_t bytes = 0;
        if (grads) {
            CALL(lffn_cross_attention_kept_bytes, &a, &bytes);
            kept = empty_bytes(bytes, dev);
        }
        CALL(lffn_cross_attention_workspace_bytes, &a, &bytes);
        if (bytes > 0) ws = empty_bytes(bytes, dev);
        CALL(lffn_cross_attention_fwd, &a, out.data_ptr(), grads ? kept.data_ptr() : nullptr, bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_on(dev));
        if (grads) {
            auto node = std::shared_ptr<CrossAttentionBackward>(new CrossAttentionBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(in.q, in.k, in.v));
            node->scale = in.scale;
            node->q = SavedVariable(in.q, false);
            node->k = SavedVariable(in.k, false);
            node->v = SavedVariable(in.v, false);
            node->mask = SavedVariable(in.mask, false);
            node->kept = SavedVariable(kept, false);
            torch::autograd::set_history(out, node);
            node->result = SavedVariable(out, true);
        }
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}
