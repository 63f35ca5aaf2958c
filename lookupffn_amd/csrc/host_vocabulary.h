// The host path of embedding, layer_norm and linear_cross_entropy (part of host.cpp): as host_attention.h's, from Python's call to the kernels' launches, and one autograd node
// for a training forward.  Through the dispatcher, a foreign-function call and an autograd function of Python's a call of a few tokens took 18 to 24 us and a training step 140 to 180.
// None for anything that is not of a kind the kernels take: the Python functions then check it, with their own errors.

// [..., columns] as rows of one stride, a copy where they are not; wide: addresses and strides of 16 bytes, as the products read them.
struct TokenRows {
    Tensor t;
    int64_t rows, columns, stride;

    TokenRows(const Tensor &from, bool wide) : t(from), columns(from.size(from.dim() - 1)) {
        rows = t.numel() / columns;
        stride = columns;
        bool as_it_is = true;
        if (!t.is_contiguous()) {
            t = t.reshape({-1, columns});
            as_it_is = (columns <= 1 || t.stride(1) == 1) && (rows <= 1 || t.stride(0) >= columns);
            if (rows > 1) stride = t.stride(0);
        }
        if (wide) as_it_is = as_it_is && aligned(t) && stride * t.element_size() % 16 == 0 && stride < int64_t(1) << 22;
        if (!as_it_is) {
            t = wide ? aligned_contiguous(t) : t.contiguous();
            stride = columns;
        }
    }
};

bool token_numbers(const Tensor &t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

// What a tensor was when it was saved.
struct Saved {
    at::ScalarType type{};
    std::vector<int64_t> sizes;
    Saved() = default;
    explicit Saved(const Tensor &t) : type(t.scalar_type()), sizes(t.sizes().vec()) {}
    bool operator==(const Tensor &t) const { return t.scalar_type() == type && t.sizes().equals(sizes); }
};

// ---------------------------------------------------------------- rows of a table

lffn_embedding embedding_arguments(const Tensor &ids, int64_t rows, int64_t columns, int32_t format, double scale, int64_t padding) {
    lffn_embedding a{};
    a.ids = ids.data_ptr();
    a.tokens = ids.numel(); a.rows = rows; a.columns = columns; a.padding = padding;
    a.scale = (float)scale;
    a.format = format;
    a.ids_64 = ids.scalar_type() == at::kLong;
    return a;
}

struct EmbeddingBackward : public torch::autograd::Node {
    SavedVariable ids;
    Saved ids_were;
    int64_t rows = 0, columns = 0, padding = -1;
    double scale = 1;
    at::ScalarType type{};

    std::string name() const override { return "EmbeddingBackward"; }

    void release_variables() override { ids.reset_data(); }

    variable_list apply(variable_list &&grads) override {
        const bool graph = at::GradMode::is_enabled();
        variable_list out = gradients(grads);
        if (graph) end_graph(*this, grads, out);
        return out;
    }

    variable_list gradients(const variable_list &grads) {
        variable_list out(1);
        if (!grads[0].defined()) return out;
        at::AutoGradMode no_grad(false);
        const Tensor ids_ = ids.unpack(shared_from_this()), g = grads[0].contiguous();
        const at::Device dev = g.device();
        const c10::DeviceGuard guard(dev);
        TORCH_CHECK(ids_were == ids_ && ids_.device() == dev && g.scalar_type() == type && g.numel() == ids_.numel() * columns, OTHER);
        const Tensor laid = ids_.contiguous();
        const lffn_embedding a = embedding_arguments(laid, rows, columns, format_of(g), scale, padding);
        out[0] = at::empty({rows, columns}, g.options());
        int64_t bytes = 0;
        CALL(lffn_embedding_bwd_workspace_bytes, &a, &bytes);
        const Tensor ws = empty_bytes(bytes, dev);
        CALL(lffn_embedding_bwd, &a, g.data_ptr(), out[0].data_ptr(), ws.data_ptr(), bytes, stream_on(dev));
        return out;
    }
};

// embedding(ids, weight, scale, padding_idx or None) -> a tensor, or None: not for this path
PyObject *embedding(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 4, "embedding: 4 arguments");
    if (watched_over() || !plain(args[0]) || !plain(args[1])) Py_RETURN_NONE;
    const Tensor ids = THPVariable_Unpack(args[0]), weight = THPVariable_Unpack(args[1]);
    const at::Device dev = weight.device();
    double scale = 1;
    int64_t padding = -1;
    if (c10::hip::current_device() != dev.index() || ids.device() != dev || !token_numbers(ids) || ids.numel() == 0 || ids.numel() >= int64_t(1) << 31 || weight.dim() != 2 ||
        weight.numel() == 0 || format_of(weight) < 0 || weight.size(0) > (int64_t(1) << 31) - 2 || weight.size(1) > 1 << 20 || !number(args[2], scale) || !std::isfinite(scale))
        Py_RETURN_NONE;
    const int64_t rows = weight.size(0), columns = weight.size(1);
    if (args[3] != Py_None) {
        if (!whole(args[3], padding) || padding < -rows || padding >= rows) Py_RETURN_NONE;
        if (padding < 0) padding += rows;
    }
    if (any_tangent({&weight})) Py_RETURN_NONE;
    const bool grads = any_gradient({&weight});
    if (grads) refuse_foreign_leaves({&weight}, dev);
    Tensor out;
    {
        const WithoutInterpreter unlocked;
        at::AutoGradMode no_grad(false);
        const Tensor laid = ids.contiguous();
        const TokenRows table(weight, false);
        lffn_embedding a = embedding_arguments(laid, rows, columns, format_of(weight), scale, padding);
        a.weight = table.t.data_ptr();
        a.stride = table.stride;
        std::vector<int64_t> sizes = ids.sizes().vec();
        sizes.push_back(columns);
        out = at::empty(sizes, weight.options());
        CALL(lffn_embedding_fwd, &a, out.data_ptr(), stream_on(dev));
        if (grads) {
            auto node = std::shared_ptr<EmbeddingBackward>(new EmbeddingBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(weight));
            node->ids = SavedVariable(ids, false);
            node->ids_were = Saved(ids);
            node->rows = rows, node->columns = columns, node->padding = padding, node->scale = scale, node->type = weight.scalar_type();
            torch::autograd::set_history(out, node);
        }
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- layer norm

struct NormRows {
    Tensor x, weight, bias;       // as they were given
    double eps = 0;

    // of a row's columns, float32 or of the rows' type, both of one
    bool fit() const {
        const int64_t columns = x.size(x.dim() - 1);
        for (const Tensor *t : {&weight, &bias})
            if (t->defined() && (t->dim() != 1 || t->size(0) != columns || (t->scalar_type() != at::kFloat && t->scalar_type() != x.scalar_type()))) return false;
        return !weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type();
    }
    // rows, w and b are what x, weight and bias are laid out as
    lffn_layer_norm_rows arguments(const TokenRows &rows, const Tensor &w, const Tensor &b) const {
        lffn_layer_norm_rows a{};
        a.x = rows.t.data_ptr();
        a.weight = w.defined() ? w.data_ptr() : nullptr;
        a.bias = b.defined() ? b.data_ptr() : nullptr;
        a.rows = rows.rows; a.columns = rows.columns; a.stride = rows.stride;
        a.eps = (float)eps;
        a.format = format_of(x);
        a.weight_f32 = (weight.defined() ? weight : bias.defined() ? bias : x).scalar_type() == at::kFloat;
        return a;
    }
};
Tensor together(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

struct LayerNormRowsBackward : public torch::autograd::Node {
    SavedVariable x, weight, stats;
    Saved x_was, weight_was;
    bool weighted = false, biased = false;
    at::ScalarType bias_type{};

    std::string name() const override { return "LayerNormRowsBackward"; }

    void release_variables() override {
        for (SavedVariable *s : {&x, &weight, &stats}) s->reset_data();
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
        NormRows in{x.unpack(self), weight.unpack(self), Tensor(), 0};
        const Tensor g = grads[0].contiguous(), stats_ = stats.unpack(self).contiguous();
        const at::Device dev = g.device();
        const c10::DeviceGuard guard(dev);
        TORCH_CHECK(x_was == in.x && in.x.device() == dev && alike(in.x, g) && in.weight.defined() == weighted &&
                        (!weighted || (weight_was == in.weight && in.weight.device() == dev)) && stats_.scalar_type() == at::kFloat && stats_.device() == dev,
                    OTHER);
        const TokenRows rows(in.x, false);
        TORCH_CHECK(stats_.dim() == 2 && stats_.size(0) == rows.rows && stats_.size(1) == 2, OTHER);
        const Tensor w = together(in.weight);
        lffn_layer_norm_rows a = in.arguments(rows, w, Tensor());
        if (!weighted && biased) a.weight_f32 = bias_type == at::kFloat;
        if (task_should_compute_output(0)) out[0] = at::empty(in.x.sizes(), in.x.options());
        if (weighted && task_should_compute_output(1)) out[1] = at::empty({rows.columns}, in.weight.options());
        if (biased && task_should_compute_output(2)) out[2] = at::empty({rows.columns}, in.x.options().dtype(bias_type));
        int64_t bytes = 0;
        Tensor ws;
        if (out[1].defined() || out[2].defined()) {
            CALL(lffn_layer_norm_rows_bwd_workspace_bytes, &a, &bytes);
            ws = empty_bytes(bytes, dev);
        }
        auto at = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
        CALL(lffn_layer_norm_rows_bwd, &a, f32(stats_), g.data_ptr(), at(out[0]), at(out[1]), at(out[2]), at(ws), bytes, stream_on(dev));
        return out;
    }
};

// layer_norm(x, weight or None, bias or None, eps) -> a tensor, or None: not for this path
PyObject *layer_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 4, "layer_norm: 4 arguments");
    if (watched_over() || !plain(args[0])) Py_RETURN_NONE;
    NormRows in;
    in.x = THPVariable_Unpack(args[0]);
    const at::Device dev = in.x.device();
    if (c10::hip::current_device() != dev.index() || in.x.dim() < 1 || in.x.numel() == 0 || format_of(in.x) < 0 || !optional_tensor(args[1], dev, in.weight) ||
        !optional_tensor(args[2], dev, in.bias) || !number(args[3], in.eps) || !(in.eps >= 0) || !in.fit() || in.x.size(in.x.dim() - 1) > 1 << 24 ||
        in.x.numel() / in.x.size(in.x.dim() - 1) >= 1 << 24)
        Py_RETURN_NONE;
    if (any_tangent({&in.x, &in.weight, &in.bias})) Py_RETURN_NONE;
    const bool grads = any_gradient({&in.x, &in.weight, &in.bias});
    if (grads) refuse_foreign_leaves({&in.x, &in.weight, &in.bias}, dev);
    Tensor out;
    {
        const WithoutInterpreter unlocked;
        at::AutoGradMode no_grad(false);
        const TokenRows rows(in.x, false);
        const Tensor w = together(in.weight), b = together(in.bias);
        const lffn_layer_norm_rows a = in.arguments(rows, w, b);
        out = at::empty(in.x.sizes(), in.x.options());
        Tensor stats;
        if (grads) stats = empty_f32({rows.rows, 2}, dev);
        CALL(lffn_layer_norm_rows_fwd, &a, out.data_ptr(), f32(stats), stream_on(dev));
        if (grads) {
            auto node = std::shared_ptr<LayerNormRowsBackward>(new LayerNormRowsBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(in.x, in.weight, in.bias));
            node->x = SavedVariable(in.x, false);
            node->weight = SavedVariable(in.weight, false);
            node->stats = SavedVariable(stats, false);
            node->x_was = Saved(in.x);
            node->weighted = in.weight.defined(), node->biased = in.bias.defined();
            if (node->weighted) node->weight_was = Saved(in.weight);
            if (node->biased) node->bias_type = in.bias.scalar_type();
            torch::autograd::set_history(out, node);
        }
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- softmax cross entropy of a projection

struct LossInputs {
    Tensor hidden, weight, bias, labels;
    int64_t ignore = -100;
    int32_t reduction = 1;

    bool fit() const {
        if (hidden.dim() < 1 || hidden.numel() == 0 || format_of(hidden) < 0 || weight.dim() != 2 || weight.numel() == 0 || weight.scalar_type() != hidden.scalar_type()) return false;
        const int64_t columns = hidden.size(hidden.dim() - 1);
        return columns % 8 == 0 && columns <= 65536 && weight.size(1) == columns && weight.size(0) <= 1 << 22 && token_numbers(labels) &&
               labels.sizes() == hidden.sizes().slice(0, hidden.dim() - 1) && labels.numel() <= 1 << 24 && hidden.numel() <= int64_t(1) << 32 &&
               (!bias.defined() || (bias.dim() == 1 && bias.size(0) == weight.size(0) && (bias.scalar_type() == at::kFloat || bias.scalar_type() == hidden.scalar_type())));
    }
    // rows, table, b and y are what hidden, weight, bias and labels are laid out as
    lffn_linear_cross_entropy arguments(const TokenRows &rows, const TokenRows &table, const Tensor &b, const Tensor &y) const {
        lffn_linear_cross_entropy a{};
        a.hidden = rows.t.data_ptr(); a.weight = table.t.data_ptr(); a.labels = y.data_ptr();
        a.bias = b.defined() ? b.data_ptr() : nullptr;
        a.tokens = rows.rows; a.vocabulary = table.rows; a.columns = rows.columns;
        a.hidden_stride = rows.stride; a.weight_stride = table.stride;
        a.ignore_index = ignore;
        a.format = format_of(hidden);
        a.bias_format = b.defined() ? format_of(b) : 0;
        a.labels_64 = y.scalar_type() == at::kLong;
        a.reduction = reduction;
        return a;
    }
};

struct LinearCrossEntropyBackward : public torch::autograd::Node {
    SavedVariable hidden, weight, bias, labels, kept;
    Saved hidden_was, weight_was, bias_was, labels_were;
    bool biased = false;
    int64_t ignore = -100;
    int32_t reduction = 1;

    std::string name() const override { return "LinearCrossEntropyBackward"; }

    void release_variables() override {
        for (SavedVariable *s : {&hidden, &weight, &bias, &labels, &kept}) s->reset_data();
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
        const LossInputs in{hidden.unpack(self), weight.unpack(self), bias.unpack(self), labels.unpack(self), ignore, reduction};
        const Tensor kept_ = aligned_contiguous(kept.unpack(self)), g = grads[0].contiguous();
        const at::Device dev = in.hidden.device();
        const c10::DeviceGuard guard(dev);
        TORCH_CHECK(hidden_was == in.hidden && weight_was == in.weight && in.weight.device() == dev && labels_were == in.labels && in.labels.device() == dev &&
                        in.bias.defined() == biased && (!biased || (bias_was == in.bias && in.bias.device() == dev)) && kept_.scalar_type() == at::kByte && kept_.dim() == 1 &&
                        kept_.device() == dev && g.device() == dev && g.scalar_type() == at::kFloat && g.numel() == (reduction == 0 ? in.labels.numel() : 1),
                    OTHER);
        const TokenRows rows(in.hidden, true), table(in.weight, true);
        const Tensor b = together(in.bias), y = in.labels.contiguous();
        const lffn_linear_cross_entropy a = in.arguments(rows, table, b, y);
        const bool of_bias = biased && task_should_compute_output(2), of_weight = task_should_compute_output(1);
        if (task_should_compute_output(0)) out[0] = at::empty(in.hidden.sizes(), in.hidden.options());
        // (the bias's gradient is formed beside the weight's)
        Tensor g_weight;
        if (of_weight || of_bias) g_weight = at::empty(in.weight.sizes(), in.weight.options());
        if (of_weight) out[1] = g_weight;
        if (of_bias) out[2] = at::empty(in.bias.sizes(), in.bias.options());
        int64_t bytes = 0;
        CALL(lffn_linear_cross_entropy_kept_bytes, &a, &bytes);
        TORCH_CHECK(kept_.numel() == bytes, OTHER);
        CALL(lffn_linear_cross_entropy_bwd_workspace_bytes, &a, &bytes);
        const Tensor ws = empty_bytes(bytes, dev);
        auto at = [](const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
        CALL(lffn_linear_cross_entropy_bwd, &a, kept_.data_ptr(), f32(g), at(out[0]), at(g_weight), at(out[2]), ws.data_ptr(), bytes, stream_on(dev));
        return out;
    }
};

// linear_cross_entropy(hidden, weight, bias or None, labels, ignore_index, reduction) -> a tensor, or None: not for this path
PyObject *linear_cross_entropy(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 6, "linear_cross_entropy: 6 arguments");
    if (watched_over() || !plain(args[0]) || !plain(args[1]) || !plain(args[3])) Py_RETURN_NONE;
    LossInputs in;
    in.hidden = THPVariable_Unpack(args[0]);
    in.weight = THPVariable_Unpack(args[1]);
    in.labels = THPVariable_Unpack(args[3]);
    const at::Device dev = in.hidden.device();
    if (c10::hip::current_device() != dev.index() || in.weight.device() != dev || in.labels.device() != dev || !optional_tensor(args[2], dev, in.bias) ||
        !whole(args[4], in.ignore) || !PyUnicode_Check(args[5]) || !in.fit())
        Py_RETURN_NONE;
    if (PyUnicode_CompareWithASCIIString(args[5], "none") == 0) in.reduction = 0;
    else if (PyUnicode_CompareWithASCIIString(args[5], "mean") == 0) in.reduction = 1;
    else if (PyUnicode_CompareWithASCIIString(args[5], "sum") == 0) in.reduction = 2;
    else Py_RETURN_NONE;
    if (any_tangent({&in.hidden, &in.weight, &in.bias})) Py_RETURN_NONE;
    const bool grads = any_gradient({&in.hidden, &in.weight, &in.bias});
    if (grads) refuse_foreign_leaves({&in.hidden, &in.weight, &in.bias}, dev);
    Tensor out;
    {
        const WithoutInterpreter unlocked;
        at::AutoGradMode no_grad(false);
        const TokenRows rows(in.hidden, true), table(in.weight, true);
        const Tensor b = together(in.bias), y = in.labels.contiguous();
        const lffn_linear_cross_entropy a = in.arguments(rows, table, b, y);
        out = in.reduction == 0 ? empty_f32(in.labels.sizes(), dev) : empty_f32({}, dev);
        int64_t bytes = 0;
        Tensor kept;
        if (grads) {
            CALL(lffn_linear_cross_entropy_kept_bytes, &a, &bytes);
            kept = empty_bytes(bytes, dev);
        }
        CALL(lffn_linear_cross_entropy_workspace_bytes, &a, &bytes);
        const Tensor ws = empty_bytes(bytes, dev);
        CALL(lffn_linear_cross_entropy_fwd, &a, f32(out), grads ? kept.data_ptr() : nullptr, ws.data_ptr(), bytes, stream_on(dev));
        if (grads) {
            auto node = std::shared_ptr<LinearCrossEntropyBackward>(new LinearCrossEntropyBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(in.hidden, in.weight, in.bias));
            node->hidden = SavedVariable(in.hidden, false);
            node->weight = SavedVariable(in.weight, false);
            node->bias = SavedVariable(in.bias, false);
            node->labels = SavedVariable(in.labels, false);
            node->kept = SavedVariable(kept, false);
            node->hidden_was = Saved(in.hidden), node->weight_was = Saved(in.weight), node->labels_were = Saved(in.labels);
            node->biased = in.bias.defined();
            if (node->biased) node->bias_was = Saved(in.bias);
            node->ignore = in.ignore, node->reduction = in.reduction;
            torch::autograd::set_history(out, node);
        }
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}
