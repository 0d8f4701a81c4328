// The host side of the paged cache's operators and of the token likelihoods: part of host.cpp, whose helpers it uses.

c10::Stream torch_stream(const at::Device &device) { return c10::impl::VirtualGuardImpl(device.type()).getStream(device); }

bool captures(const at::Device &device)
{
    const c10::DeviceGuard guard(device);
    return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

struct PagedPlan {
    kvmix_paged_plan_t c{};
    Tensor list;  // the plan's words on the device
    std::optional<c10::Stream> made_on;
    std::shared_ptr<c10::Event> made;  // when they are there

    Tensor slots() const { return list.narrow(0, c.slots_at, c.tokens); }

    // The words for a call on the current stream.  On another stream than the plan was made on they are waited for, and their memory is
    // given to nobody else before the call has read it (they are hidden from the caller, who could not see to it).  A
    // capture begins with the device idle and cannot wait for what lies outside it.
    const int32_t *words() const
    {
        const c10::Stream now = torch_stream(list.device());
        if (now != *made_on) {
            if (!captures(list.device())) made->block(now);
            list.record_stream(now);
        }
        return list.data_ptr<int32_t>();
    }
};

// Nothing here has a derivative (the likelihoods have one, backwards, which the caller records): a call that should record one, or
// whose result a trace would keep as a constant, is refused.
void need_no_record(const char *name, std::initializer_list<const Tensor *> ts)
{
    if (torch::jit::tracer::isTracing()) fail(std::string(name) + " cannot be part of a trace");
    for (const Tensor *t : ts)
        if ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())
            fail(std::string(name) + " has no derivative for this tensor: call it under torch.no_grad() or with detached tensors");
}

// Page numbers as the library takes them, in 32 bits.  What is beyond them is no page: -1.
Tensor page_numbers(const Tensor &t)
{
    if (c10::elementSize(t.scalar_type()) < 4 || t.scalar_type() == at::kInt) return t.to(at::kInt).contiguous();
    const Tensor from = t.to(at::kLong).contiguous(), to = at::empty(t.sizes(), at::kInt);
    const int64_t *x = from.data_ptr<int64_t>();
    int32_t *y = to.data_ptr<int32_t>();
    for (int64_t i = 0; i < from.numel(); i++) y[i] = x[i] < 0 || x[i] > 0x7fffffff ? -1 : (int32_t)x[i];
    return to;
}

// page numbers in host memory, [n] or [n, 2]
Tensor host_list(const Tensor &t, int64_t dim, const char *what)
{
    if (t.is_cuda() || !at::isIntegralType(t.scalar_type(), false) || t.dim() != dim || (dim == 2 && t.size(1) != 2))
        fail(std::string(what) + " must be a tensor of whole numbers in host memory, " + (dim == 2 ? "[n, 2]" : "[n]"));
    return page_numbers(t);
}

void use_rows(kvmix_paged_pool_t &p, const Tensor &rows)
{
    need_gpu({&rows});
    need_half({&rows});
    if (rows.dim() != 5 || rows.size(2) != 2 || !rows.is_contiguous()) fail("fp16 pages must be contiguous [pages, kv_heads, 2, page_size, head_dim]");
    p.rows = rows.data_ptr(), p.row_pages = rows.size(0), p.kv_heads = rows.size(1), p.page_size = rows.size(3), p.head_dim = rows.size(4);
}

void use_packed(kvmix_paged_pool_t &p, const Tensor &packed, int64_t kv_heads, int64_t page_size, int64_t head_dim, int64_t k_bits, int64_t v_bits)
{
    check_bits(k_bits);
    check_bits(v_bits);
    need_gpu({&packed});
    if (packed.scalar_type() != at::kInt || packed.dim() != 3 || packed.size(1) != kv_heads || !packed.is_contiguous() ||
        packed.size(2) != page_size / 32 * head_dim * (k_bits + v_bits + 2))
        fail("packed pages must be contiguous int32 [pages, kv_heads, page_size / 32 * head_dim * (k_bits + v_bits + 2)]");
    p.packed = packed.data_ptr(), p.packed_pages = packed.size(0);
    p.kv_heads = kv_heads, p.page_size = page_size, p.head_dim = head_dim, p.k_bits = (int)k_bits, p.v_bits = (int)v_bits;
}

// [tokens, heads, D] as 16-byte pieces can be read from it
Tensor pieces3(const Tensor &t)
{
    const bool ok = t.stride(2) == 1 && (t.size(0) <= 1 || t.stride(0) % 8 == 0) && (t.size(1) <= 1 || t.stride(1) % 8 == 0) &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

int64_t stride_of(const Tensor &t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

PagedPlan paged_plan(const Tensor &table_in, const std::vector<int64_t> &kv_lens, const std::vector<int64_t> &packed_lens, const std::vector<int64_t> &q_lens,
                     int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size, const at::Device &device)
{
    if (table_in.is_cuda() || !at::isIntegralType(table_in.scalar_type(), false) || table_in.dim() != 2)
        fail("paged_plan: the table must be whole numbers in host memory, [sequences, pages]");
    if (!device.is_cuda()) fail("KVmix operators run on the GPU only: got " + device.str());
    // (a replay would copy the list again, from memory that is no longer its own)
    if (captures(device)) fail("paged_plan: a plan cannot be made while a graph is captured");
    const Tensor table = page_numbers(table_in);
    const int64_t n = table.size(0);
    for (const auto *lens : {&kv_lens, &packed_lens, &q_lens})
        if ((int64_t)lens->size() != n) fail("paged_plan: as many lengths as the table has sequences");
    const kvmix_paged_batch_t b = {table.data_ptr<int32_t>(), table.size(1), kv_lens.data(), packed_lens.data(), q_lens.data(), n, heads, kv_heads, head_dim, page_size};
    PagedPlan plan;
    check(api.paged_plan(&b, nullptr, 0, &plan.c));
    Tensor host = at::empty({plan.c.words}, at::TensorOptions(at::kInt).pinned_memory(true));
    check(api.paged_plan(&b, host.data_ptr<int32_t>(), plan.c.words, &plan.c));
    plan.list = at::empty({plan.c.words}, at::TensorOptions(at::kInt).device(device));
    plan.list.copy_(host, true);
    plan.made_on = torch_stream(device);
    plan.made = std::make_shared<c10::Event>(device.type());
    plan.made->record(*plan.made_on);
    return plan;
}

void paged_append(const Tensor &k_in, const Tensor &v_in, const Tensor &rows, const PagedPlan &plan)
{
    need_no_record("paged_append", {&k_in, &v_in, &rows});
    kvmix_paged_pool_t p{};
    use_rows(p, rows);
    need_half({&k_in, &v_in});
    need_with(rows, {&k_in, &v_in, &plan.list});
    for (const Tensor *t : {&k_in, &v_in})
        if (t->dim() != 3 || t->size(0) != plan.c.tokens || t->size(1) != p.kv_heads || t->size(2) != p.head_dim)
            fail("paged_append: keys and values must be [the plan's new tokens, kv_heads, head_dim]");
    if (plan.c.page_size != p.page_size) fail("paged_append: the plan is for pages of another size");
    if (plan.c.row_pages > p.row_pages) check(KVMIX_ERR_PAGE);
    const Tensor k = pieces3(k_in), v = pieces3(v_in);
    const c10::DeviceGuard guard(rows.device());
    check(api.paged_append(&p, &plan.c, plan.words(), k.data_ptr(), stride_of(k, 0), stride_of(k, 1), v.data_ptr(), stride_of(v, 0),
                           stride_of(v, 1), stream_of(rows)));
}

void paged_quantize(const Tensor &rows, const Tensor &packed, const Tensor &pairs_in, int64_t k_bits, int64_t v_bits)
{
    need_no_record("paged_quantize", {&rows});
    kvmix_paged_pool_t p{};
    use_rows(p, rows);
    use_packed(p, packed, p.kv_heads, p.page_size, p.head_dim, k_bits, v_bits);
    need_with(rows, {&packed});
    const Tensor pairs = host_list(pairs_in, 2, "paged_quantize: pairs");
    const c10::DeviceGuard guard(rows.device());
    check(api.paged_quantize(&p, pairs.data_ptr<int32_t>(), pairs.size(0), stream_of(rows)));
}

std::tuple<Tensor, Tensor> paged_read(const Tensor &pool, const Tensor &pages_in, const std::optional<int64_t> &k_bits, const std::optional<int64_t> &v_bits,
                                      const std::optional<int64_t> &head_dim)
{
    need_no_record("paged_read", {&pool});
    kvmix_paged_pool_t p{};
    const bool packed = k_bits || v_bits;
    if (packed) {
        if (!k_bits || !v_bits || !head_dim) fail("paged_read: packed pages need both widths and the head dimension");
        if (*head_dim != 64 && *head_dim != 128) fail("paged_read: the head dimension is 64 or 128");
        check_bits(*k_bits);
        check_bits(*v_bits);
        if (pool.dim() != 3) fail("packed pages must be contiguous int32 [pages, kv_heads, page_size / 32 * head_dim * (k_bits + v_bits + 2)]");
        use_packed(p, pool, pool.size(1), pool.size(2) / (*head_dim * (*k_bits + *v_bits + 2)) * 32, *head_dim, *k_bits, *v_bits);
    } else {
        use_rows(p, pool);
    }
    const Tensor pages = host_list(pages_in, 1, "paged_read: pages");
    const int64_t n = pages.size(0);
    const auto options = at::TensorOptions(at::kHalf).device(pool.device());
    Tensor k = at::empty({n, p.page_size, p.kv_heads, p.head_dim}, options), v = at::empty_like(k);
    const c10::DeviceGuard guard(pool.device());
    check(api.paged_read(&p, packed, pages.data_ptr<int32_t>(), n, k.data_ptr(), v.data_ptr(), stream_of(pool)));
    return {k, v};
}

void paged_copy(const std::vector<Tensor> &pools, const Tensor &pairs_in)
{
    const Tensor pairs = host_list(pairs_in, 2, "paged_copy: pairs");
    if (pools.empty()) return;
    std::vector<void *> at(pools.size());
    std::vector<int64_t> bytes(pools.size());
    const int64_t pages = pools[0].dim() ? pools[0].size(0) : 0;
    for (size_t i = 0; i < pools.size(); i++) {
        const Tensor &t = pools[i];
        need_no_record("paged_copy", {&t});
        need_gpu({&t});
        need_with(pools[0], {&t});
        if (t.dim() < 2 || t.size(0) != pages || !t.is_contiguous()) fail("paged_copy: pools must be contiguous, with the same number of pages");
        at[i] = t.data_ptr(), bytes[i] = pages ? (int64_t)t.nbytes() / pages : 0;
    }
    const c10::DeviceGuard guard(pools[0].device());
    check(api.paged_copy(at.data(), bytes.data(), (int64_t)pools.size(), pages, pairs.data_ptr<int32_t>(), pairs.size(0), stream_of(pools[0])));
}

Tensor paged_attention(const Tensor &q_in, const Tensor &rows, const Tensor &packed, const PagedPlan &plan, int64_t k_bits, int64_t v_bits,
                       const std::optional<double> &scale)
{
    need_no_record("paged_attention", {&q_in, &rows});
    kvmix_paged_pool_t p{};
    use_rows(p, rows);
    use_packed(p, packed, p.kv_heads, p.page_size, p.head_dim, k_bits, v_bits);
    need_half({&q_in});
    need_with(rows, {&packed, &q_in, &plan.list});
    if (q_in.dim() != 3 || q_in.size(0) != plan.c.tokens || q_in.size(1) != plan.c.heads || q_in.size(2) != p.head_dim)
        fail("paged_attention: queries must be [the plan's new tokens, heads, head_dim]");
    if (plan.c.kv_heads != p.kv_heads || plan.c.page_size != p.page_size) fail("paged_attention: the plan is for pages of another shape");
    const Tensor q = pieces3(q_in);
    Tensor out = at::empty({q.size(0), q.size(1), q.size(2)}, q.options());
    const int64_t need = api.paged_attention_workspace_bytes(&plan.c);
    Tensor ws;
    if (need) ws = at::empty({need}, q.options().dtype(at::kByte));
    kvmix_paged_attn_t c{};
    c.q = q.data_ptr(), c.q_token_stride = stride_of(q, 0), c.q_head_stride = stride_of(q, 1);
    c.out = out.data_ptr(), c.out_token_stride = out.stride(0), c.out_head_stride = out.stride(1);
    c.list = plan.words();
    c.scale = scale ? (float)*scale : 1.0f / std::sqrt((float)p.head_dim);
    const c10::DeviceGuard guard(rows.device());
    check(api.paged_attention(&p, &plan.c, &c, need ? ws.data_ptr() : nullptr, need, stream_of(rows)));
    return out;
}

// The descriptor that both directions of the likelihoods share; `x`: rows with unit stride.
kvmix_token_logprobs_t score_call(const Tensor &x, const Tensor &targets)
{
    kvmix_token_logprobs_t c{};
    c.logits = x.data_ptr(), c.rows = x.size(0), c.vocab = x.size(1), c.row_stride = x.size(0) > 1 ? x.stride(0) : x.size(1);
    c.dtype = x.scalar_type() == at::kHalf ? KVMIX_F16 : x.scalar_type() == at::kFloat ? KVMIX_F32 : KVMIX_BF16;
    c.targets = targets.data_ptr<int64_t>();
    return c;
}

Tensor score_rows2(const Tensor &logits)
{
    Tensor x = logits.dim() == 2 ? logits : logits.reshape({-1, logits.size(-1)});
    return x.stride(1) == 1 && (x.size(0) <= 1 || x.stride(0) >= x.size(1)) ? x : x.contiguous();
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor &logits, const Tensor &targets_in, int64_t top, bool want_stats)
{
    need_no_record("token_logprobs", {&logits});
    need_gpu({&logits});
    need_with(logits, {&targets_in});
    if (logits.scalar_type() != at::kHalf && logits.scalar_type() != at::kBFloat16 && logits.scalar_type() != at::kFloat)
        fail("token_logprobs: logits must be float16, bfloat16 or float32, got " + dtype_name(logits));
    if (targets_in.scalar_type() != at::kLong) fail("token_logprobs: targets must be int64, got " + dtype_name(targets_in));
    if (logits.dim() < 1 || logits.size(-1) == 0 || targets_in.sizes() != logits.sizes().slice(0, logits.dim() - 1))
        fail("token_logprobs: targets must have the shape of the logits without their last dimension, which must not be empty");
    if (top < 0 || top > 64 || top > logits.size(-1)) fail("token_logprobs: top must be between 0 and 64, and not more than there are tokens");
    const Tensor x = score_rows2(logits), targets = targets_in.contiguous();
    kvmix_token_logprobs_t c = score_call(x, targets);
    auto sizes = targets_in.sizes().vec();
    const auto floats = x.options().dtype(at::kFloat);
    Tensor lp = at::empty(sizes, floats), entropy = at::empty(sizes, floats), stats, top_lp, top_id, ws;
    c.logprob = lp.data_ptr<float>(), c.entropy = entropy.data_ptr<float>();
    if (want_stats) stats = at::empty({x.size(0), 4}, floats), c.stats = stats.data_ptr<float>();
    if (top > 0) {
        sizes.push_back(top);
        top_lp = at::empty(sizes, floats), top_id = at::empty(sizes, x.options().dtype(at::kLong));
        c.top = top, c.top_logprob = top_lp.data_ptr<float>(), c.top_id = top_id.data_ptr<int64_t>();
    }
    const int64_t need = api.token_logprobs_workspace_bytes(&c);
    if (need) ws = at::empty({need}, x.options().dtype(at::kByte));
    const c10::DeviceGuard guard(x.device());
    check(api.token_logprobs(&c, need ? ws.data_ptr() : nullptr, need, stream_of(x)));
    return {lp, entropy, top_lp, top_id, stats};
}

Tensor token_logprobs_grad(const Tensor &logits, const Tensor &targets_in, const Tensor &stats, const OptTensor &grad_logprob, const OptTensor &grad_entropy)
{
    const Tensor x = score_rows2(logits), targets = targets_in.contiguous();
    kvmix_token_logprobs_t c = score_call(x, targets);
    c.stats = stats.data_ptr<float>();
    Tensor a, b, dx = at::empty({x.size(0), x.size(1)}, x.options());
    if (grad_logprob) a = grad_logprob->to(at::kFloat).contiguous();
    if (grad_entropy) b = grad_entropy->to(at::kFloat).contiguous();
    const c10::DeviceGuard guard(x.device());
    check(api.token_logprobs_grad(&c, grad_logprob ? a.data_ptr<float>() : nullptr, grad_entropy ? b.data_ptr<float>() : nullptr, dx.data_ptr(),
                                  x.size(1), stream_of(x)));
    return dx.view(logits.sizes());
}
