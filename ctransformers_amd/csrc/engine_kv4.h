// The 4-bit KV cache of a handle (CT_AMD_KV=q4) and its contexts (CT_AMD_CONTEXTS) — part of engine.cc, included there inside namespace ctamd.  Not a stand-alone header.
//
// The mat-vec launches leave fp16 K / V rows at their positions as without it, in buffers of ONE layer that all layers use in turn; behind them every layer quantizes
// the new rows into its pages (kv4_append) and attends to the pages (kv4_attention), the new rows among them.  A page is 64 tokens (CT_AMD_KV_PAGE: 32, 64, 128, 256) of all KV heads of a
// layer; one page table serves all layers.  A handle holds n contexts (sequences) on one set of weights: evals read and write the active one, a fork shares pages, and
// positions in shared pages are given pages of their own before they are written (kv_reserve copies a partly filled one).  The pool has room for every context's
// full length, so making room never fails.  The tables change only where an eval enters positions without room of their own (once every 64 tokens of a plain
// continuation): token steps replay their graphs, which read the active context's row of the table at a fixed address.

bool Engine::kv4_setup(std::string& err) {
    const char* kind = getenv("CT_AMD_KV");
    const int n = std::max(1, env_int("CT_AMD_CONTEXTS", 1));
    kv4_ = kind && !strcmp(kind, "q4");
    if (kind && *kind && !kv4_ && strcmp(kind, "f16")) { err = std::string("CT_AMD_KV=") + kind + ": f16 or q4"; return false; }
    if (!kv4_) {
        if (n > 1) { err = "CT_AMD_CONTEXTS needs the paged cache: CT_AMD_KV=q4"; return false; }
        return true;
    }
    if (hp_.legacy() || l0_ != 0 || l1_ != hp_.n_layer) { err = "CT_AMD_KV=q4 serves llama and falcon models on one GPU"; return false; }
    dbg_kv4_fail_ = env_int("CT_AMD_DBG_KV4_FAIL", 0);
    if (n > 256) { err = "CT_AMD_CONTEXTS: at most 256"; return false; }
    ctxs_.assign((size_t)n, Context());
    kv_page_ = env_int("CT_AMD_KV_PAGE", 64);
    kv_page_bytes_ = kv4_page_bytes(hp_.n_head_kv, hp_.head_dim(), kv_page_);
    if (!kv_page_bytes_) { err = "CT_AMD_KV=q4: head size, or CT_AMD_KV_PAGE (32, 64, 128, 256), not supported"; return false; }
    kv_width_ = (n_ctx_ + kv_page_ - 1) / kv_page_;
    kv_n_pages_ = n * kv_width_;
    const size_t pool = (size_t)hp_.n_layer * kv_n_pages_ * kv_page_bytes_;
    if (!dev_alloc(dev_allocs_, &kv_pool_, pool, err)) return false;
    HIP_OK(hipMemset(kv_pool_, 0, pool));
    for (int b = 0; b < 2; ++b)
        if (!dev_alloc(dev_allocs_, &kv_table_[b], (size_t)kv_n_pages_, err) || !dev_alloc(dev_allocs_, &kv_lens_[b], (size_t)n, err) ||
            !dev_alloc(dev_allocs_, &kv_refs_[b], (size_t)kv_n_pages_, err)) return false;
    HIP_OK(hipMemset(kv_table_[0], 0xFF, (size_t)kv_n_pages_ * 4));
    HIP_OK(hipMemset(kv_lens_[0], 0, (size_t)n * 4));
    HIP_OK(hipMemset(kv_refs_[0], 0, (size_t)kv_n_pages_ * 4));
    KvPages a = KvPages();
    a.n_seq = n; a.n_pages = kv_n_pages_;
    if (!dev_alloc(dev_allocs_, &kv_row_, (size_t)kv_width_, err) || !dev_alloc(dev_allocs_, &kv_args_, (size_t)2 * n + 1, err) ||
        !dev_alloc(dev_allocs_, &kv_ws_, (size_t)kv_pages_ws_ints(a), err)) return false;
    HIP_OK(hipMemset(kv_row_, 0xFF, (size_t)kv_width_ * 4));
    HIP_OK(hipHostMalloc(&h_kv_, ((size_t)2 * n + 1) * 4));
    // the workspace of the widest attention launch a step or a chunk of any size asks for
    for (int rows = 1; rows <= kPfChunkFast; ++rows) {
        Kv4Attn at = Kv4Attn();
        const char* why = nullptr;
        if (!kv4_cache(at.c, 0, rows, why)) { err = why; return false; }
        at.n_head = hp_.n_head;
        kv_attn_ws_n_ = std::max(kv_attn_ws_n_, kv4_attention_plan(at, rows));
    }
    return kv_attn_ws_n_ == 0 || dev_alloc(dev_allocs_, &kv_attn_ws_, (size_t)kv_attn_ws_n_, err);
}

bool Engine::kv4_cache(Kv4Cache& c, int layer, int rows, const char*& why) {
    c.pages = kv_pool_ + (size_t)layer * kv_n_pages_ * kv_page_bytes_;
    c.page_stride = kv_page_bytes_;
    c.table = kv_row_;
    c.lens = d_state_ ? d_state_ + 1 : (const int*)kv_row_;   // the cursor's position: tokens before the step's rows (not read while the sizes are planned)
    c.len_add = rows;
    c.n_pages = kv_n_pages_; c.table_stride = c.table_width = kv_width_;
    c.n_seq = 1; c.total = rows; c.n_head_kv = hp_.n_head_kv; c.head_dim = hp_.head_dim();
    return kv4_check(c, kv_page_, why);
}

// the layer's rows of this step from the fp16 buffers into its pages, then attention over the pages
bool Engine::kv4_attend(const uint16_t* kc, const uint16_t* vc, int nt, std::string& err) {
    const int rows = std::max(1, nt), hd = hp_.head_dim();
    const char* why = nullptr;
    Kv4Append ap = Kv4Append();
    bool ok = kv4_cache(ap.c, cur_layer_, rows, why);
    ap.absolute = 1;
    ap.k.p = kc; ap.k.row = hd; ap.k.head = (long long)n_ctx_ * hd; ap.k.dim = 1; ap.k.type = KV4_F16;
    ap.v.p = vc; ap.v.row = 1; ap.v.head = (long long)hd * v_stride_; ap.v.dim = v_stride_; ap.v.type = KV4_F16;
    ok = ok && kv4_append(ap, rows, stream_, why);
    AttnArgsX ax = AttnArgsX();
    fill_attn_args(ax, nullptr, nullptr, nt);
    Kv4Attn at = Kv4Attn();
    at.c = ap.c;
    at.q.p = ax.q_f16; at.q.row = ax.q_stride; at.q.head = hd; at.q.dim = 1; at.q.type = KV4_F16;
    at.out = ax.out; at.o_row = ax.out_stride; at.o_head = hd; at.out_type = KV4_F32;
    at.n_head = hp_.n_head; at.scale = ax.kq_scale; at.ws = kv_attn_ws_;
    if (dbg_kv4_fail_ > 0 && --dbg_kv4_fail_ == 0) { ok = false; why = "refused on purpose"; }
    ok = ok && kv4_attention(at, rows, kv_attn_ws_n_, stream_, why);
    if (!ok) { err = std::string("attention over the 4-bit cache: ") + (why ? why : "launch failed"); return false; }   // (a step without it is no step: nor is a graph of it)
    ++kv4_launches_;
    return true;
}

// One change of the tables: the two (n) vectors in kv_args_ — parents and kept lengths of a fork, or the tokens to make room for — are on their way; the call's
// outputs become the current tables.
bool Engine::kv4_tables(bool reserve, std::string& err) {
    const int n = (int)ctxs_.size();
    HIP_OK(hipMemcpyAsync(kv_args_, h_kv_, (size_t)2 * n * 4, hipMemcpyHostToDevice, stream_));
    const int i = kv_side_, o = i ^ 1;
    KvPages a = KvPages();
    a.table = kv_table_[i]; a.lens = kv_lens_[i]; a.refs = kv_refs_[i];
    a.table_o = kv_table_[o]; a.lens_o = kv_lens_[o]; a.refs_o = kv_refs_[o];
    a.n_seq = n; a.width = kv_width_; a.n_pages = kv_n_pages_; a.page_tokens = kv_page_;
    const char* why = nullptr;
    bool ok;
    if (reserve) {
        a.add = kv_args_;
        a.pages = kv_pool_; a.layers = hp_.n_layer; a.layer_stride = kv_n_pages_ * kv_page_bytes_; a.page_bytes = kv_page_bytes_;
        a.status = kv_args_ + 2 * n; a.ws = kv_ws_;
        ok = kv_reserve(a, stream_, why);
    } else {
        a.parents = kv_args_; a.keep = kv_args_ + n; a.n_new = n;
        ok = kv_fork(a, stream_, why);
    }
    if (!ok) { err = std::string("page tables: ") + why; return false; }
    if (reserve) HIP_OK(hipMemcpyAsync(h_kv_ + 2 * n, kv_args_ + 2 * n, 4, hipMemcpyDeviceToHost, stream_));
    HIP_OK(hipStreamSynchronize(stream_));   // (h_kv_ is free again)
    if (reserve && h_kv_[2 * n] != 0) { err = "page tables: no room (" + std::to_string(h_kv_[2 * n]) + ")"; return false; }
    kv_side_ = o;
    return true;
}
bool Engine::kv4_row(std::string& err) {   // the active context's row to where the launches read it
    HIP_OK(hipMemcpyAsync(kv_row_, kv_table_[kv_side_] + (size_t)active_ * kv_width_, (size_t)kv_width_ * 4, hipMemcpyDeviceToDevice, stream_));
    return true;
}

// pages of its own for positions [n_past, n_past + n) of the active context
bool Engine::kv4_room(int n_past, int n, std::string& err) {
    Context& c = ctxs_[active_];
    const int m = (int)ctxs_.size(), need = n_past + n;
    bool cut = false;
    if (n_past < c.own_from) {   // positions in pages that another context reads too: those from n_past on are given back, and new ones taken below
        for (int i = 0; i < m; ++i) { h_kv_[i] = i; h_kv_[m + i] = i == active_ ? n_past : 0x7FFFFFFF; }
        if (!kv4_tables(false, err)) return false;
        c.room = std::min(c.room, n_past);
        cut = true;
    } else if (need <= c.room) {
        c.len = need;
        return true;
    }
    const int end = std::min((need + kv_page_ - 1) / kv_page_ * kv_page_, kv_width_ * kv_page_);
    for (int i = 0; i < m; ++i) h_kv_[i] = i == active_ ? end - c.room : 0;
    if (!kv4_tables(true, err)) return false;
    const int from = c.room / kv_page_ * kv_page_;   // (a partly filled last page is the context's own now: reserve copied it if it was shared)
    c.own_from = cut ? from : std::min(c.own_from, from);
    c.room = end;
    c.len = need;
    return kv4_row(err);
}

bool Engine::context_use(int i, std::string& err) {
    if (!kv4_ || i < 0 || i >= (int)ctxs_.size()) { err = "no such context (CT_AMD_KV=q4, CT_AMD_CONTEXTS=n)"; return false; }
    HIP_OK(hipSetDevice(device_));
    active_ = i;
    last_pos_ = -1;   // (what is replayed for measurement is the last token of an eval of THIS context)
    return kv4_row(err);
}
bool Engine::context_fork(int src, int dst, std::string& err) {
    const int m = (int)ctxs_.size();
    if (!kv4_ || src < 0 || src >= m || dst < 0 || dst >= m || src == dst) { err = "no such pair of contexts (CT_AMD_KV=q4, CT_AMD_CONTEXTS=n)"; return false; }
    HIP_OK(hipSetDevice(device_));
    for (int i = 0; i < m; ++i) { h_kv_[i] = i == dst ? src : i; h_kv_[m + i] = i == dst ? ctxs_[src].len : 0x7FFFFFFF; }
    if (!kv4_tables(false, err)) return false;
    if (src == active_ || dst == active_) last_pos_ = -1;   // (its page is shared now, or what it was the last token of is gone: not to be written again by a measurement)
    const int len = ctxs_[src].len, shared = (len + kv_page_ - 1) / kv_page_ * kv_page_;
    ctxs_[src].own_from = std::max(ctxs_[src].own_from, shared);
    ctxs_[dst] = Context{len, len, shared};
    return kv4_row(err);
}
bool Engine::context_free(int i, std::string& err) {
    const int m = (int)ctxs_.size();
    if (!kv4_ || i < 0 || i >= m) { err = "no such context (CT_AMD_KV=q4, CT_AMD_CONTEXTS=n)"; return false; }
    HIP_OK(hipSetDevice(device_));
    for (int k = 0; k < m; ++k) { h_kv_[k] = k == i ? -1 : k; h_kv_[m + k] = 0x7FFFFFFF; }
    if (!kv4_tables(false, err)) return false;
    ctxs_[i] = Context();
    if (i == active_) last_pos_ = -1;
    return kv4_row(err);
}
int Engine::context_compact(std::string& err) {   // pages in use, -1: failed
    if (!kv4_) { err = "no paged cache (CT_AMD_KV=q4)"; return -1; }
    const int n = (int)ctxs_.size(), i = kv_side_, o = i ^ 1;
    (void)hipSetDevice(device_);
    KvPages a = KvPages();
    a.table = kv_table_[i]; a.refs = kv_refs_[i]; a.table_o = kv_table_[o]; a.refs_o = kv_refs_[o];
    a.n_seq = n; a.width = kv_width_; a.n_pages = kv_n_pages_; a.page_tokens = kv_page_;
    a.pages = kv_pool_; a.layers = hp_.n_layer; a.layer_stride = kv_n_pages_ * kv_page_bytes_; a.page_bytes = kv_page_bytes_;
    a.status = kv_args_ + 2 * n; a.ws = kv_ws_;
    const char* why = nullptr;
    if (!kv_compact(a, stream_, why)) { err = std::string("page tables: ") + why; return -1; }
    if (hipMemcpyAsync(kv_lens_[o], kv_lens_[i], (size_t)n * 4, hipMemcpyDeviceToDevice, stream_) != hipSuccess ||
        hipMemcpyAsync(h_kv_ + 2 * n, kv_args_ + 2 * n, 4, hipMemcpyDeviceToHost, stream_) != hipSuccess) { err = "page tables: copy failed"; return -1; }
    kv_side_ = o;
    if (!kv4_row(err)) return -1;
    if (hipStreamSynchronize(stream_) != hipSuccess) { err = "page tables: stream failed"; return -1; }
    return h_kv_[2 * n];
}
