// jdg_beamsearch.cuh — beam search of the own model (jdg_beam_search), part of jdg_engine.cu.
//
// A step is the batched decode step of the beams with three of its kernels replaced: the rotation
// and append go through jdg_paged_append, the attention through jdg_paged_attn and the pick
// through jdg_beam_select, with jdg_beam_reorder behind it.  The engine's slot cache is used as
// it lies, as a paged cache with pages of one row: row (slot, position) of a layer is page
// slot * L * max_seq + position of the layer's base.  A beam writes only rows of its own slot, each
// position once, so a row stays what it was for every beam that has it in its table, and no cache
// row is ever copied.  State that is indexed by beam (tables, EMAs, histories, scores, flags) is
// kept twice, and each step goes from one side to the other; the two directions are captured once
// each as a graph.
#pragma once

// what one side of the search holds
struct BeamSide {
    int *table, *hist, *done;  // [beams][max_seq] row numbers by position, [beams][max_new], [beams]
    float *cum, *consensus;    // [beams], [beams][L]
};
struct BeamRun {
    int beams, n, max_new, eos;
    BeamSide side[2];
    int *seq, *lens, *parent, *token;  // 0..beams-1; own rows; the selection
    void *ws_attn, *ws_sel;
    size_t ws_attn_bytes, ws_sel_bytes;
    int cur;  // the side that holds the state before the step
};

// the cache of layer l for one side's table; own: the table from the first own position on
static jdg_paged_kv beam_kv(const jdg_engine *e, int l, const BeamRun *r, bool own) {
    const size_t base = (size_t)l * e->max_seq * e->kd;
    jdg_paged_kv kv = {};
    kv.k = e->kc + base;
    kv.v = e->vc + base;
    kv.dt = JD_F32;
    kv.n_pages = (int)((size_t)e->B_max * e->L * e->max_seq - (size_t)l * e->max_seq);
    kv.page_size = 1;
    kv.n_kv_heads = e->KVH;
    kv.head_dim = e->HD;
    kv.page_stride = e->kd;
    kv.row_stride = e->kd;
    kv.head_stride = e->HD;
    kv.table = r->side[r->cur].table + (own ? r->n - 1 : 0);
    kv.table_stride = e->max_seq;
    kv.n_seqs = r->beams;
    return kv;
}
static jdg_attn_args beam_attn_args(const jdg_engine *e, const BeamRun *r, float scale) {
    jdg_attn_args a = {};
    a.q = e->qkv;
    a.q_stride = e->qkvd;
    a.out = e->att;
    a.out_stride = e->qd;
    a.n_heads = e->Hh;
    a.prefix = e->pf_pos;  // rows 0, 1, .. of slot 0: the prompt
    a.prefix_len = r->n - 1;
    a.lens = r->lens;
    a.max_len = r->max_new;
    a.scale = scale;
    a.clamp = e->clamp;
    a.status = e->err;
    return a;
}
static jdg_select_args beam_select_args(const jdg_engine *e, const BeamRun *r) {
    jdg_select_args a = {};
    a.logits = e->logits;
    a.dt = JD_F32;
    a.stride = e->ldl;
    a.groups = 1;
    a.beams = r->beams;
    a.vocab = e->V;
    a.n_out = r->beams;
    a.cum = r->side[r->cur].cum;
    a.done = r->eos >= 0 ? r->side[r->cur].done : nullptr;
    a.eos = r->eos >= 0 ? r->eos : 0;
    a.parent = r->parent;
    a.token = r->token;
    a.score = r->side[r->cur ^ 1].cum;  // the next step's scores
    return a;
}
// a message of the device operators (kept with no context) becomes the engine's
static int beam_op(jdg_engine *e, int rc) {
    if (rc != JD_OK) jdg_set_err(e->ctx, "jdg_beam_search: %s", jdg_last_error(nullptr));
    return rc;
}

static int beam_attention(jdg_engine *e, int l, int B, const BeamRun *r, float scale) {
    jdg_paged_kv kv = beam_kv(e, l, r, false);
    jdg_append_args a = {};
    a.q = a.q_out = e->qkv;  // in place
    a.k = e->qkv + e->qd;
    a.v = e->qkv + e->qd + e->kd;
    a.dt = JD_F32;
    a.n_tokens = B;
    a.n_heads = e->Hh;
    a.q_stride = a.k_stride = a.v_stride = a.q_out_stride = e->qkvd;
    a.seq = r->seq;
    a.pos = e->pos;
    a.cos = e->rope_cos;
    a.sin = e->rope_sin;
    a.n_pos = e->max_seq;
    a.rot_dim = e->HD;
    a.rope_norm = e->rope_norm;
    a.status = e->err;
    int rc = beam_op(e, jdg_paged_append(&kv, &a, e->st));
    if (rc != JD_OK) return rc;
    kv = beam_kv(e, l, r, true);
    const jdg_attn_args t = beam_attn_args(e, r, scale);
    rc = beam_op(e, jdg_paged_attn(&kv, &t, r->ws_attn, r->ws_attn_bytes, e->st));
    e->launches += 3;  // append, own rows, join (and the prefix's own kernel where it has one)
    return rc;
}

// After the selection: beam b continues its parent (already copied) with its token; one thread a beam.
static __global__ void k_beam_advance(int beams, int n, int max_new, int eos, int max_seq, int slot_rows,
                                      const int *__restrict__ parent, const int *__restrict__ token,
                                      const int *__restrict__ done_in, int *done, float *cum, int *table, int *hist, int *tok,
                                      int *pos, int *lens) {
    const int b = threadIdx.x;
    if (b >= beams) return;
    const int p = parent[b], t = token[b], step = pos[b] - (n - 1);  // tokens chosen before this one
    if (p < 0) {  // fewer continuations than beams: this one is dead from here on
        done[b] = 0;
        cum[b] = -INFINITY;
        tok[b] = 0;
    } else {
        done[b] = eos >= 0 && (done_in[p] || t == eos);
        tok[b] = t;
    }
    if (step < max_new) hist[(size_t)b * max_new + step] = p < 0 ? -1 : t;
    const int next = pos[b] + 1;
    if (next < max_seq) table[(size_t)b * max_seq + next] = b * slot_rows + next;  // its own row
    pos[b] = next < max_seq ? next : max_seq - 1;
    lens[b] = min(step + 2, max_new);
}

// one step from side cur to the other
static int enqueue_beam_step(jdg_engine *e, BeamRun *r) {
    const int B = r->beams;
    float *own_consensus = e->consensus;
    e->consensus = r->side[r->cur].consensus;  // the elections update this side's averages in place
    int rc = own_batch_layers(e, B, -1, r);
    e->consensus = own_consensus;
    if (rc != JD_OK) return rc;
    own_head(e, B);
    const jdg_select_args sel = beam_select_args(e, r);
    rc = beam_op(e, jdg_beam_select(&sel, r->ws_sel, r->ws_sel_bytes, e->st));
    if (rc != JD_OK) return rc;
    const BeamSide &a = r->side[r->cur], &b = r->side[r->cur ^ 1];
    jdg_reorder_args ro = {};
    ro.parent = r->parent;
    ro.parent_stride = ro.beams = B;
    ro.groups = 1;
    ro.n_states = 3;
    ro.state[0] = jdg_state{a.table, b.table, e->max_seq * 4ll, e->max_seq * 4ll, e->max_seq * 4ll};
    ro.state[1] = jdg_state{a.hist, b.hist, r->max_new * 4ll, r->max_new * 4ll, r->max_new * 4ll};
    ro.state[2] = jdg_state{a.consensus, b.consensus, e->L * 4ll, e->L * 4ll, e->L * 4ll};
    ro.status = e->err;
    rc = beam_op(e, jdg_beam_reorder(&ro, e->st));
    if (rc != JD_OK) return rc;
    k_beam_advance<<<1, 32, 0, e->st>>>(B, r->n, r->max_new, r->eos, e->max_seq, e->L * e->max_seq, r->parent, r->token,
                                        a.done, b.done, b.cum, b.table, b.hist, e->tok, e->pos, r->lens);
    e->launches += 4;
    return JD_OK;
}

// memory and graphs of one search, released with it
struct BeamMem {
    std::vector<void *> mem;
    cudaGraphExec_t graph[2] = {nullptr, nullptr};
    ~BeamMem() {
        for (cudaGraphExec_t g : graph)
            if (g) cudaGraphExecDestroy(g);
        for (void *p : mem) cudaFree(p);
    }
};

static int beam_search_impl(jdg_engine *e, const int *prompt, int n, int beams, int max_new, int eos, int *tokens, int *lens,
                            float *scores) {
    BeamMem own;
    BeamRun r = {};
    r.beams = beams;
    r.n = n;
    r.max_new = max_new;
    r.eos = eos;
    int rc;
    for (int b = 0; b < beams; b++)
        if ((rc = jdg_reset(e, b)) != JD_OK) return rc;
    if ((rc = jdg_set_prompt(e, 1, prompt, n, &n, nullptr)) != JD_OK) return rc;
    if ((rc = jdg_prefill(e, 1)) != JD_OK) return rc;
    auto take = [&](void **p, size_t bytes) {
        const cudaError_t err = cudaMalloc(p, bytes ? bytes : 16);
        if (err != cudaSuccess) {
            jdg_set_err(e->ctx, "jdg_beam_search: cudaMalloc(%zu) failed: %s", bytes, cudaGetErrorString(err));
            return JD_ENOMEM;
        }
        own.mem.push_back(*p);
        return JD_OK;
    };
#define BEAM_TAKE(ptr, bytes)                                              \
    do {                                                                   \
        if ((rc = take((void **)&(ptr), (size_t)(bytes))) != JD_OK) return rc; \
    } while (0)
    const size_t B = beams;
    for (BeamSide &s : r.side) {
        BEAM_TAKE(s.table, B * e->max_seq * 4);
        BEAM_TAKE(s.hist, B * max_new * 4);
        BEAM_TAKE(s.done, B * 4);
        BEAM_TAKE(s.cum, B * 4);
        BEAM_TAKE(s.consensus, B * e->L * 4);
    }
    BEAM_TAKE(r.seq, B * 4);
    BEAM_TAKE(r.lens, B * 4);
    BEAM_TAKE(r.parent, B * 4);
    BEAM_TAKE(r.token, B * 4);
    const float scale = 1.0f / sqrtf((float)e->HD);
    const jdg_paged_kv kv = beam_kv(e, 0, &r, true);
    const jdg_attn_args at = beam_attn_args(e, &r, scale);
    if ((rc = beam_op(e, jdg_paged_attn_check(&kv, &at))) != JD_OK) return rc;
    r.ws_attn_bytes = jdg_paged_attn_workspace(&kv, &at);
    const jdg_select_args sel = beam_select_args(e, &r);
    if ((rc = beam_op(e, jdg_beam_select_check(&sel))) != JD_OK) return rc;
    r.ws_sel_bytes = jdg_beam_select_workspace(&sel);
    BEAM_TAKE(r.ws_attn, r.ws_attn_bytes);
    BEAM_TAKE(r.ws_sel, r.ws_sel_bytes);
#undef BEAM_TAKE
    // all beams start as the prompt's sequence; only the first counts until the first selection
    std::vector<int> table(B * e->max_seq, 0), iota(B), ones(B, 1), tok(B, prompt[n - 1]), pos(B, n - 1), zero(B, 0);
    std::vector<float> cum(B, -INFINITY), cons(e->L);
    cum[0] = 0.f;
    for (int b = 0; b < beams; b++) {
        iota[b] = b;
        table[(size_t)b * e->max_seq + n - 1] = b * e->L * e->max_seq + n - 1;
    }
    CK(cudaMemcpyAsync(r.side[0].table, table.data(), table.size() * 4, cudaMemcpyHostToDevice, e->st));
    CK(cudaMemcpyAsync(r.side[1].table, table.data(), table.size() * 4, cudaMemcpyHostToDevice, e->st));
    CK(cudaMemsetAsync(r.side[0].hist, 0xff, B * max_new * 4, e->st));
    CK(cudaMemsetAsync(r.side[1].hist, 0xff, B * max_new * 4, e->st));
    CK(cudaMemcpyAsync(r.side[0].done, zero.data(), B * 4, cudaMemcpyHostToDevice, e->st));
    CK(cudaMemcpyAsync(r.side[0].cum, cum.data(), B * 4, cudaMemcpyHostToDevice, e->st));
    for (int b = 0; b < beams; b++)
        CK(cudaMemcpyAsync(r.side[0].consensus + (size_t)b * e->L, e->consensus, e->L * 4, cudaMemcpyDeviceToDevice, e->st));
    CK(cudaMemcpyAsync(r.side[1].consensus, r.side[0].consensus, B * e->L * 4, cudaMemcpyDeviceToDevice, e->st));
    CK(cudaMemcpyAsync(r.seq, iota.data(), B * 4, cudaMemcpyHostToDevice, e->st));
    CK(cudaMemcpyAsync(r.lens, ones.data(), B * 4, cudaMemcpyHostToDevice, e->st));
    CK(cudaMemcpyAsync(e->tok, tok.data(), B * 4, cudaMemcpyHostToDevice, e->st));
    CK(cudaMemcpyAsync(e->pos, pos.data(), B * 4, cudaMemcpyHostToDevice, e->st));
    CK(cudaStreamSynchronize(e->st));
    CK(cudaEventRecord(e->ev0, e->st));
    std::vector<int> flags(B);
    int steps = 0;
    for (; steps < max_new; steps++) {
        r.cur = steps & 1;
        cudaGraphExec_t &g = own.graph[r.cur];
        if (steps < 2) {
            // the first step in each direction runs as it is (the kernels' attributes are set on the way)
            if ((rc = enqueue_beam_step(e, &r)) != JD_OK) return rc;
            CK(cudaGetLastError());
        } else {
            if (!g) {
                cudaGraph_t raw = nullptr;
                CK(cudaStreamBeginCapture(e->st, cudaStreamCaptureModeThreadLocal));
                rc = enqueue_beam_step(e, &r);
                cudaError_t err = cudaStreamEndCapture(e->st, &raw);
                if (rc == JD_OK && err == cudaSuccess) err = cudaGraphInstantiate(&g, raw, 0);
                if (raw) cudaGraphDestroy(raw);
                if (rc != JD_OK) return rc;
                if (err != cudaSuccess) {
                    g = nullptr;
                    jdg_set_err(e->ctx, "jdg_beam_search: graph capture failed: %s", cudaGetErrorString(err));
                    return JD_ECUDA;
                }
            }
            CK(cudaGraphLaunch(g, e->st));
        }
        if (eos >= 0 && (steps & 15) == 15) {  // every beam finished: nothing changes any more
            CK(cudaMemcpyAsync(flags.data(), r.side[r.cur ^ 1].done, B * 4, cudaMemcpyDeviceToHost, e->st));
            CK(cudaStreamSynchronize(e->st));
            bool all = true;
            for (int f : flags) all = all && f;
            if (all) {
                steps++;
                break;
            }
        }
    }
    CK(cudaEventRecord(e->ev1, e->st));
    CK(cudaEventSynchronize(e->ev1));
    CK(cudaEventElapsedTime(&e->last_ms, e->ev0, e->ev1));
    if ((rc = check_err(e)) != JD_OK) return rc;
    const BeamSide &s = r.side[steps & 1];
    std::vector<int> hist(B * max_new);
    CK(cudaMemcpy(hist.data(), s.hist, B * max_new * 4, cudaMemcpyDeviceToHost));
    CK(cudaMemcpy(scores, s.cum, B * 4, cudaMemcpyDeviceToHost));
    for (int b = 0; b < beams; b++) {
        int len = 0;
        while (len < steps && hist[(size_t)b * max_new + len] >= 0) {
            tokens[(size_t)b * max_new + len] = hist[(size_t)b * max_new + len];
            if (eos >= 0 && hist[(size_t)b * max_new + len++] == eos) break;
            if (eos < 0) len++;
        }
        lens[b] = len;
    }
    return JD_OK;
}

extern "C" int jdg_beam_search(jdg_engine *e, const int *prompt, int n, int beams, int max_new, int eos, int *tokens,
                               int *lens, float *scores) {
    if (!e) return JD_EINVAL;
    if (e->kind != 0) {
        jdg_set_err(e->ctx, "jdg_beam_search: the own model only");
        return JD_EUNSUPPORTED;
    }
    if (!prompt || !tokens || !lens || !scores || n < 1 || beams < 1 || beams > e->B_max || beams > 32 || beams > e->V ||
        max_new < 1 || n > e->max_seq || max_new > e->max_seq - n || eos >= e->V) {
        jdg_set_err(e->ctx, "jdg_beam_search: bad arguments (prompt %d, %d beams, %d new tokens; %d slots, %d positions)", n,
                    beams, max_new, e->B_max, e->max_seq);
        return JD_EINVAL;
    }
    for (int i = 0; i < n; i++)
        if (prompt[i] < 0 || prompt[i] >= e->V) {
            jdg_set_err(e->ctx, "jdg_beam_search: token %d of the prompt outside [0, %d)", prompt[i], e->V);
            return JD_EINVAL;
        }
    if ((size_t)e->B_max * e->L * e->max_seq > 0x7fffffffu) {
        jdg_set_err(e->ctx, "jdg_beam_search: more than 2^31 cache rows");
        return JD_EUNSUPPORTED;
    }
    cudaSetDevice(e->ctx->device);
    int rc;
    try {
        rc = beam_search_impl(e, prompt, n, beams, max_new, eos, tokens, lens, scores);
    } catch (const std::bad_alloc &) {
        jdg_set_err(e->ctx, "jdg_beam_search: out of host memory");
        rc = JD_ENOMEM;
    }
    cudaStreamSynchronize(e->st);
    for (int b = 0; b < beams; b++) {
        const int r2 = jdg_reset(e, b);
        if (rc == JD_OK) rc = r2;
    }
    return rc;
}
