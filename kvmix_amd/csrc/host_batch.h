// The host side of the operators on batches of requests (adapters, beams): part of host.cpp, whose helpers it uses.

struct AdapterPlan : PlanList {
    kvmix_adapter_plan_t c{};
};

AdapterPlan adapter_plan(const std::vector<int64_t> &adapters, const std::vector<int64_t> &counts, int64_t n_adapters, const at::Device &device)
{
    if (!device.is_cuda()) fail("KVmix operators run on the GPU only: got " + device.str());
    if (adapters.size() != counts.size()) fail("adapter_plan: as many adapters as sequences");
    for (int64_t n : counts)
        if (n < 0) fail("adapter_plan: a negative number of tokens");
    if (captures(device)) fail("adapter_plan: a plan cannot be made while a graph is captured");
    AdapterPlan plan;
    const int64_t n = (int64_t)adapters.size();
    check(api.adapter_plan(adapters.data(), counts.data(), n, n_adapters, nullptr, 0, &plan.c));
    plan.make(plan.c.words, device, [&](int32_t *words) { check(api.adapter_plan(adapters.data(), counts.data(), n, n_adapters, words, plan.c.words, &plan.c)); });
    return plan;
}

bool in_pieces(const Tensor &t)
{
    bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t d = 0; d + 1 < t.dim(); d++) ok = ok && (t.size(d) <= 1 || t.stride(d) % 8 == 0);
    return ok;
}

Tensor pieces_of(const Tensor &t) { return in_pieces(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

// Whether what two tensors span has no byte in common.
bool spans_apart(const Tensor &a, const Tensor &b)
{
    if (!a.numel() || !b.numel()) return true;
    auto span = [](const Tensor &t) {
        int64_t n = 1;
        for (int64_t d = 0; d < t.dim(); d++) n += (t.size(d) - 1) * t.stride(d);
        return n * (int64_t)t.element_size();
    };
    const int64_t from_a = (int64_t)a.data_ptr(), from_b = (int64_t)b.data_ptr();
    return from_a + span(a) <= from_b || from_b + span(b) <= from_a;
}

// Whether the rows of `a` and what `b` spans have no memory in common: columns beside one another of the same wider rows are apart.
bool apart(const Tensor &a, const Tensor &b)
{
    if (spans_apart(a, b)) return true;
    const int64_t from_a = (int64_t)a.data_ptr(), from_b = (int64_t)b.data_ptr();
    const Tensor c = b.dim() == 2 ? b : b.dim() == 3 && (b.size(0) == 1 || b.size(1) == 1) ? b.squeeze(b.size(1) == 1 ? 1 : 0) : Tensor();
    if (!c.defined() || a.size(0) == 1 || c.size(0) == 1 || a.stride(0) != c.stride(0) || a.stride(1) != 1 || c.stride(1) != 1 || a.stride(0) < a.size(1)) return false;
    const int64_t row = a.stride(0) * a.element_size(), off = ((from_b - from_a) % row + row) % row;
    return off >= a.size(1) * (int64_t)a.element_size() && off + c.size(1) * (int64_t)c.element_size() <= row;
}

// [..., n] as [tokens, n]: a view, or where there is none and one is not needed a copy
Tensor as_rows(const Tensor &t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

Tensor add_adapters(const Tensor &base_in, const Tensor &x_in, const Tensor &a_in, const Tensor &b_in, const AdapterPlan &plan, const OptTensor &scales_in,
                    const OptTensor &out_in)
{
    need_no_record("add_adapters", {&base_in, &x_in, &a_in, &b_in});
    if (scales_in) need_no_record("add_adapters", {&*scales_in});
    if (out_in) need_no_record("add_adapters", {&*out_in});
    need_gpu({&base_in});
    need_with(base_in, {&x_in, &a_in, &b_in, &plan.list});
    if (base_in.scalar_type() != at::kHalf && base_in.scalar_type() != at::kBFloat16)
        fail("add_adapters: tensors must be float16 or bfloat16, got " + dtype_name(base_in));
    for (const Tensor *t : {&x_in, &a_in, &b_in})
        if (t->scalar_type() != base_in.scalar_type()) fail("add_adapters: base, x and the adapters must be of one type");
    if (base_in.dim() < 2 || x_in.dim() != base_in.dim() || x_in.sizes().slice(0, x_in.dim() - 1) != base_in.sizes().slice(0, base_in.dim() - 1))
        fail("add_adapters: base must be [..., n] and x [..., k], of the same tokens");
    const int64_t k = x_in.size(-1), n = base_in.size(-1);
    if (a_in.dim() != 3 || b_in.dim() != 3 || b_in.size(0) != a_in.size(0) || a_in.size(2) != k || b_in.size(1) != n || b_in.size(2) != a_in.size(1))
        fail("add_adapters: the adapters must be a [adapters, rank, k] and b [adapters, n, rank]");
    const int64_t rank = a_in.size(1);
    if (rank <= 0 || rank > 128 || rank % 8 || k <= 0 || k % 8 || n <= 0 || n % 8)
        fail("add_adapters: rank (at most 128), k and n must be multiples of 8");
    if (base_in.numel() / n != plan.c.tokens) fail("add_adapters: the plan is of another number of tokens");
    if (plan.c.adapters > a_in.size(0)) check(KVMIX_ERR_ADAPTER);
    if (scales_in) {
        need_with(base_in, {&*scales_in});
        if (scales_in->scalar_type() != at::kFloat || scales_in->dim() != 1 || scales_in->size(0) != a_in.size(0))
            fail("add_adapters: scales must be float32 [adapters]");
    }
    Tensor out = out_in ? *out_in : at::empty(base_in.sizes(), base_in.options()), rows;
    if (out_in) {
        need_with(base_in, {&out});
        if (out.scalar_type() != base_in.scalar_type() || out.sizes() != base_in.sizes()) fail("add_adapters: out must be like base");
    }
    rows = as_rows(out);
    // (a copy would not be what the caller holds; tokens that lie on one another cannot be written)
    if (rows.data_ptr() != out.data_ptr() || !in_pieces(rows) || (rows.size(0) > 1 && rows.stride(0) < n))
        fail("add_adapters: out must have rows that 16-byte pieces can be written to");
    if (out_in) {
        const bool in_place = out.data_ptr() == base_in.data_ptr() && out.strides() == base_in.strides();
        if (!in_place && !apart(rows, base_in)) fail("add_adapters: out may be base, but not overlap it otherwise");
        if (!apart(rows, x_in) || !apart(rows, a_in) || !apart(rows, b_in) || (scales_in && !spans_apart(rows, *scales_in))) fail("add_adapters: out must not overlap what is read");
    }
    const Tensor base = out.data_ptr() == base_in.data_ptr() ? rows : pieces_of(as_rows(base_in)), x = pieces_of(as_rows(x_in));
    const Tensor a = pieces_of(a_in), b = pieces_of(b_in), scales = scales_in ? scales_in->contiguous() : Tensor();
    kvmix_adapters_t c{};
    c.x = x.data_ptr(), c.a = a.data_ptr(), c.b = b.data_ptr(), c.base = base.data_ptr(), c.out = rows.data_ptr();
    c.x_token_stride = stride_of(x, 0), c.a_adapter_stride = stride_of(a, 0), c.a_rank_stride = stride_of(a, 1), c.b_adapter_stride = stride_of(b, 0);
    c.b_row_stride = stride_of(b, 1), c.base_token_stride = stride_of(base, 0), c.out_token_stride = stride_of(rows, 0);
    c.scales = scales_in ? scales.data_ptr<float>() : nullptr;
    c.adapters = a.size(0), c.rank = rank, c.k = k, c.n = n, c.dtype = base.scalar_type() == at::kHalf ? KVMIX_F16 : KVMIX_BF16;
    const int64_t need = api.add_adapters_workspace_bytes(&plan.c, &c);
    Tensor ws;
    if (need) ws = at::empty({need}, base.options().dtype(at::kByte));
    const c10::DeviceGuard guard(base.device());
    check(api.add_adapters(&plan.c, plan.words(), &c, need ? ws.data_ptr() : nullptr, need, stream_of(base)));
    return out;
}

std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor &logits, const Tensor &scores_in, const std::optional<int64_t> &count_in, const OptTensor &done_in,
                                               const std::optional<int64_t> &end, bool stay)
{
    need_no_record("beam_select", {&logits, &scores_in});
    need_gpu({&logits});
    need_with(logits, {&scores_in});
    if (logits.scalar_type() != at::kHalf && logits.scalar_type() != at::kBFloat16 && logits.scalar_type() != at::kFloat)
        fail("beam_select: logits must be float16, bfloat16 or float32, got " + dtype_name(logits));
    if (logits.dim() != 3 || logits.size(1) == 0 || logits.size(2) == 0) fail("beam_select: logits must be [requests, beams, vocabulary], with a beam and a token at least");
    const int64_t requests = logits.size(0), beams = logits.size(1), vocab = logits.size(2), count = count_in.value_or(beams);
    if (scores_in.scalar_type() != at::kFloat || scores_in.dim() != 2 || scores_in.size(0) != requests || scores_in.size(1) != beams)
        fail("beam_select: scores must be float32 [requests, beams]");
    if (beams > 64 || count < 1 || count > 64 || count > vocab) fail("beam_select: at most 64 beams, a count between 1 and 64 that is not more than there are tokens");
    if (vocab > (1 << 20) || beams * vocab > (1 << 25)) fail("beam_select: a vocabulary of at most 2^20 tokens, 2^25 with all beams of a request");
    if (stay && count != beams) fail("beam_select: results stay in their beams' places only where there are as many as beams");
    if (done_in) {
        need_with(logits, {&*done_in});
        if (done_in->scalar_type() != at::kBool || done_in->sizes() != scores_in.sizes()) fail("beam_select: done must be bool [requests, beams]");
        if (!end || *end < 0 || *end >= vocab) fail("beam_select: beams that have ended need the token that ends them, one of the vocabulary");
    }
    const Tensor x = score_rows2(logits), scores = scores_in.contiguous(), done = done_in ? done_in->contiguous() : Tensor();
    Tensor out = at::empty({requests, count}, scores.options()), parents = at::empty({requests, count}, scores.options().dtype(at::kLong));
    Tensor tokens = at::empty_like(parents), ws;
    kvmix_beam_select_t c{};
    c.logits = x.data_ptr(), c.row_stride = x.size(0) > 1 ? x.stride(0) : vocab;
    c.dtype = x.scalar_type() == at::kHalf ? KVMIX_F16 : x.scalar_type() == at::kFloat ? KVMIX_F32 : KVMIX_BF16;
    c.scores = scores.data_ptr<float>(), c.done = done_in ? (const uint8_t *)done.data_ptr() : nullptr, c.end = end.value_or(0);
    c.requests = requests, c.beams = beams, c.vocab = vocab, c.count = count, c.stay = stay;
    c.out_scores = out.data_ptr<float>(), c.parents = parents.data_ptr<int64_t>(), c.tokens = tokens.data_ptr<int64_t>();
    const int64_t need = api.beam_select_workspace_bytes(&c);
    if (need) ws = at::empty({need}, x.options().dtype(at::kByte));
    const c10::DeviceGuard guard(x.device());
    check(api.beam_select(&c, need ? ws.data_ptr() : nullptr, need, stream_of(x)));
    return {out, parents, tokens};
}

// A tensor's first dimension and what belongs to one entry of it.
kvmix_reorder_t reorder_item(const Tensor &t)
{
    const int64_t size = (int64_t)t.element_size();
    struct Dim {
        int64_t size, stride;
    };
    std::vector<Dim> dims;
    for (int64_t d = 1; d < t.dim(); d++)
        if (t.size(d) > 1) dims.push_back({t.size(d), t.stride(d) * size});
    std::sort(dims.begin(), dims.end(), [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
    std::vector<Dim> all = dims;
    if (t.size(0) > 1) all.push_back({t.size(0), t.stride(0) * size});
    std::sort(all.begin(), all.end(), [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
    int64_t extent = size;  // of what the dimensions so far span
    for (const Dim &d : all) {
        if (d.stride < extent) fail("reorder_rows: entries of a tensor must not overlap");
        extent += (d.size - 1) * d.stride;
    }
    kvmix_reorder_t item{};
    item.base = t.data_ptr(), item.batch_stride = t.size(0) > 1 ? t.stride(0) * size : extent;
    int64_t run = size;
    std::vector<Dim> outer;
    for (const Dim &d : dims) {
        if (outer.empty() && d.stride == run) run *= d.size;
        else if (!outer.empty() && d.stride == outer.back().stride * outer.back().size) outer.back().size *= d.size;
        else outer.push_back(d);
    }
    if (outer.size() > 2) fail("reorder_rows: an entry of a tensor must be rows of memory in at most two dimensions");
    item.row_bytes = run;
    item.inner = outer.size() > 0 ? outer[0].size : 1, item.inner_stride = outer.size() > 0 ? outer[0].stride : 0;
    item.outer = outer.size() > 1 ? outer[1].size : 1, item.outer_stride = outer.size() > 1 ? outer[1].stride : 0;
    return item;
}

void reorder_rows(const std::vector<Tensor> &tensors, const Tensor &index_in)
{
    if (torch::jit::tracer::isTracing()) fail("reorder_rows cannot be part of a trace");
    need_gpu({&index_in});
    if (index_in.scalar_type() != at::kLong || index_in.dim() != 1) fail("reorder_rows: the index must be int64 [rows]");
    const int64_t rows = index_in.size(0);
    if (rows > 1024) fail("reorder_rows: at most 1024 rows");
    std::vector<kvmix_reorder_t> items;
    for (const Tensor &t : tensors) {
        need_no_record("reorder_rows", {&t});
        need_gpu({&t});
        need_with(index_in, {&t});
        if (t.dim() < 1 || t.size(0) != rows) fail("reorder_rows: every tensor must have as many entries as the index");
        if (t.numel() == 0) continue;
        items.push_back(reorder_item(t));
    }
    Tensor index = index_in.contiguous();
    for (const Tensor &t : tensors)  // (it is read while they are written)
        if (!spans_apart(t, index)) {
            index = index.clone();
            break;
        }
    const c10::DeviceGuard guard(index.device());
    check(api.reorder_rows(items.data(), (int64_t)items.size(), index.data_ptr<int64_t>(), rows, stream_of(index)));
}
