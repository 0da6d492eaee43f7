"""Performance cases of the operators around the full-attention layer: attention within a window, steps of
several drafted tokens over the paged cache, keeping the accepted ones, choosing the next token.

* window: softmax attention of q [B, H, N, D] over k, v [B, Hkv, N, D] (H = Hkv * G), where position i
  sees position j <= i if i - j < window or j < sinks; positions from a sequence's length on see nothing
  and are not seen.  A training pass returns the output and the three gradients, a prompt's pass the output.
* tree:   T tokens of each sequence, drafted as a tree: node i hangs on the earlier node ``parents[i]`` or,
  -1, on the last position of the cache.  Their rows go to positions pos .. pos + T - 1 of a paged cache (see
  operators.py for its layout), and node i, which stands at position pos + depth, attends the positions
  before pos, its ancestors and itself; with a window, those of them within it.  A chain of one token is
  the single-token step.
* accept: node 0's token is certain; from a node the walk goes to the first child whose token is the one that
  the model picked there.  The rows of the nodes on that path are then kept: written to pos, pos + 1, ..
* sample: a token of each row of logits by one uniform number.  Logits are divided by the temperature; the
  largest top_k stay, of those the ones before which less than or exactly top_p of their mass lies (the
  largest first, of equal ones the first), of those the ones of at least min_p times the largest probability.
  The token is the first whose running mass, in the order of the vocabulary, is above u times the
  mass that is left; its log probability there comes with it.  A temperature of zero takes the largest logit.

``own`` chooses between the framework's kernels and the same mathematics in elementary torch operations.
Steps write the same rows into the same places each time, so they can be repeated.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
          "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1, "int8": 1}


def _window(name, B, Hkv, G, N, D, window, sinks, dtype, grad=True, ragged=False):
    return dict(name=name, op="window", B=B, Hkv=Hkv, G=G, N=N, D=D, window=window, sinks=sinks, dtype=dtype,
                grad=grad, ragged=ragged)


def _tree(name, B, Hkv, G, D, T, length, page, dtype, cache, ragged=False, window=0, sinks=0):
    return dict(name=name, op="tree", B=B, Hkv=Hkv, G=G, D=D, T=T, length=length, page=page, dtype=dtype,
                cache=cache, ragged=ragged, window=window, sinks=sinks)


def _accept(name, B, Hkv, D, T, length, page, dtype, cache):
    return dict(name=name, op="accept", B=B, Hkv=Hkv, D=D, T=T, length=length, page=page, dtype=dtype, cache=cache,
                ragged=True)


def _sample(name, B, V, dtype, temperature, top_k=0, top_p=1.0, min_p=0.0, rows=False):
    """rows: each row has settings of its own around these, and some tokens are banned (-inf)."""
    return dict(name=name, op="sample", B=B, V=V, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, rows=rows)


def listed():
    return [
        # A training step of the 13M model's full-attention layer with a window.
        _window("window_train_13m", 8, 8, 1, 2048, 32, 256, 4, "bf16"),
        # One long document in training, shared key/value heads: the largest.
        _window("window_train_long", 1, 4, 4, 16384, 128, 1024, 4, "bf16"),
        # A padded batch of prompts of odd lengths before generation.
        _window("window_prompt_odd", 3, 2, 3, 1999, 80, 333, 1, "f16", grad=False, ragged=True),
        # One chat-sized sequence of the 13M model's layer in float32, a few drafted tokens.
        _tree("tree_77_f32", 1, 8, 1, 32, 7, 77, 64, "f32", "f32"),
        # Batched serving of the 85M model's layer, sequences of many lengths in small pages.
        _tree("tree_85m_batch", 32, 12, 1, 64, 26, 2048, 16, "bf16", "bf16", ragged=True),
        # Shared key/value heads over an 8-bit cache and a full tree.
        _tree("tree_shared_e4m3", 16, 8, 4, 128, 64, 8192, 64, "bf16", "e4m3", ragged=True),
        # The single-token step of a windowed layer: long caches of which little is read.
        _tree("tree_one_windowed", 32, 12, 1, 64, 1, 8191, 64, "bf16", "bf16", ragged=True, window=1024, sinks=4),
        # The accepted path of one chat: launches and host work.
        _accept("accept_one", 1, 8, 32, 7, 77, 64, "bf16", "bf16"),
        # ... of a full batch over an 8-bit cache.
        _accept("accept_batch_e4m3", 64, 8, 128, 64, 2048, 64, "bf16", "e4m3"),
        # One chat's next token over the reference's vocabulary, as generation asks for it.
        _sample("sample_one", 1, 32000, "f32", 0.8, top_p=0.9),
        # A batch of requests with settings of their own.
        _sample("sample_batch", 256, 32000, "bf16", 0.9, top_k=50, top_p=0.9, rows=True),
        # A large vocabulary, nothing but a nucleus and a floor.
        _sample("sample_wide", 64, 151001, "f32", 1.1, top_p=0.95, min_p=0.002),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _pairs(N, window, sinks):
    """Pairs of positions (i, j) that see each other, j <= i < N."""
    n = np.arange(1, N + 1, dtype=np.float64)
    return float((np.minimum(n, window) + np.clip(n - window, 0, sinks)).sum())


def draw(rng):
    op = rng.choice(["window", "window", "window", "tree", "tree", "tree", "accept", "sample", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    D = rng.choice([32, 64, 80, 96, 128])
    if op == "window":
        while True:
            B, Hkv, G, N = _log_int(rng, 1, 8), _log_int(rng, 1, 8), rng.choice([1, 1, 2, 3, 4, 8]), _log_int(rng, 1, 16384)
            window, sinks = _log_int(rng, 1, 2 * N), rng.choice([0, 0, 1, 4, 17, 64])
            if B * Hkv * G * D * _pairs(N, window, sinks) <= 16 * 128 * _pairs(16384, 1024, 4) / (8 if dtype == "f32" else 1):
                return dict(op=op, B=B, Hkv=Hkv, G=G, N=N, D=D, window=window, sinks=sinks, dtype=dtype,
                            grad=rng.random() < 0.7, ragged=rng.random() < 0.4)
    if op == "sample":
        while True:
            B, V = _log_int(rng, 1, 256), _log_int(rng, 100, 200000)
            if B * V <= 64 * 151001:
                break
        return dict(op=op, B=B, V=V, dtype=dtype, temperature=round(rng.uniform(0.3, 2.0), 3),
                    top_k=rng.choice([0, 0, 1, 5, 50, 1000]), top_p=rng.choice([1.0, 0.95, 0.9, 0.5]),
                    min_p=rng.choice([0.0, 0.0, 0.001, 0.05]), rows=rng.random() < 0.5)
    cache, page = rng.choice([dtype, dtype, "e4m3", "int8"]), rng.choice([16, 32, 64, 128, 256])
    G = rng.choice([1, 1, 2, 3, 4, 5, 8]) if op == "tree" else 1
    while True:
        B, Hkv, length, T = _log_int(rng, 1, 64), _log_int(rng, 1, 16), _log_int(rng, 1, 65536), _log_int(rng, 1, 64)
        rows = B * Hkv * D * (length + T)
        if rows * SIZES[cache] <= 1 << 26 and rows * T * G <= 1 << 32:
            break
    c = dict(op=op, B=B, Hkv=Hkv, D=D, T=T, length=length, page=page, dtype=dtype, cache=cache,
             ragged=rng.random() < 0.7)
    if op == "tree":
        window = _log_int(rng, 1, length + T) if rng.random() < 0.35 else 0
        c.update(G=G, window=window, sinks=rng.choice([0, 1, 4, 17, 64]) if window else 0)
    return c


def _lengths(n, B, ragged):
    """Lengths of each sequence: all n, or spread from n down to a quarter of it, the last of three or
    more a single one (a request that has just come in), in an order of no rule."""
    if not ragged:
        return [n] * B
    x = [max(1, n - (3 * n * i) // (4 * B)) for i in range(B)]
    if B > 2:
        x[-1] = 1
    random.Random(B * 1000003 + n).shuffle(x)
    return x


def _parents(c, seed):
    """A tree for each sequence: a few candidates for each next token, most of them for the likely ones; in
    larger batches the last is a plain chain."""
    rng = random.Random(seed * 7919 + c["B"] * 31 + c["T"])
    res = []
    for b in range(c["B"]):
        p = [-1]
        for i in range(1, c["T"]):
            p.append(rng.randrange(max(0, i - 1 - 2 * int(rng.expovariate(0.4))), i))
        res.append(p if b != 2 else list(range(-1, c["T"] - 1)))
    return res


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _tokens(c, seed):
    """Drafted tokens, and the token that the model picks at each node: mostly a child's."""
    rng = random.Random(seed * 104729 + c["B"] * 17 + c["T"])
    tokens, picks = [], []
    for parents in _parents(c, seed):
        t = [rng.randrange(32000) for _ in parents]
        p = []
        for i in range(len(parents)):
            kids = [j for j in range(len(parents)) if parents[j] == i]
            p.append(t[rng.choice(kids)] if kids and rng.random() < 0.8 else rng.randrange(32000))
        tokens.append(t)
        picks.append(p)
    return tokens, picks


def _walk(parents, tokens, picks):
    """Nodes of the accepted path."""
    path = [0]
    while True:
        kids = [j for j in range(len(parents)) if parents[j] == path[-1] and tokens[j] == picks[path[-1]]]
        if not kids:
            return path
        path.append(kids[0])


def _quantise(x, cache):
    """Rows of x as the 8-bit values' bytes and the scales' exponent bytes."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    # 448 = 0.875 * 2^9 and 127 = 0.9921875 * 2^7 are the types' largest values.
    e = e - 9 + (m > 0.875).int() if cache == "e4m3" else e - 7 + (m > 0.9921875).int()
    e = torch.where(m == 0, -127, e.clamp(min=-127))
    # 2^-e by its bits: the chip's pow may be off in the last one.
    y = x * ((127 - e) << 23).to(torch.int32).view(torch.float32)[..., None]
    y = y.to(torch.float8_e4m3fn) if cache == "e4m3" else y.round().to(torch.int8)
    return y.view(torch.uint8), (e + 127).to(torch.uint8)


def _prepare_cache(c, g):
    B, Hkv, D, T, page = c["B"], c["Hkv"], c["D"], c["T"], c["page"]
    ct = DTYPES[c["cache"]]
    n = _lengths(c["length"], B, c["ragged"])
    used = [-(-(x + T) // page) for x in n]
    M, P = -(-(c["length"] + T) // page), sum(used) + 2  # two pages that belong to nobody

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    # Keys differ in size from channel to channel, as those of trained models do.
    channel = torch.exp(0.5 * randn(D))

    def pool(ch):
        x = randn(P, Hkv, page, D) * ch
        if SIZES[c["cache"]] > 1:
            return x.to(ct), None
        y, e = _quantise(x, c["cache"])
        return y.view(ct), e.view(torch.float8_e8m0fnu)

    s = dict(case=c)
    s["k_pages"], s["k_scale"] = pool(channel)
    s["v_pages"], s["v_scale"] = pool(1.0)
    # Pages in an order of no rule; entries behind a sequence's last page name none.
    order = torch.randperm(P, generator=g, device=DEV)[:sum(used)].to(torch.int32).cpu()
    table = torch.full((B, M), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    s["page_table"] = table.to(DEV)
    s["pos"] = torch.tensor(n, dtype=torch.int64, device=DEV)
    # The drafted tokens' rows: head views of a projection's output.
    kv = randn(B, T, 2, Hkv, D)
    kv[:, :, 0] *= channel
    kv = kv.to(DTYPES[c["dtype"]])
    s["k"], s["v"] = (kv[:, :, i].permute(0, 2, 1, 3) for i in (0, 1))
    return s


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if c["op"] == "window":
        B, Hkv, H, N, D = c["B"], c["Hkv"], c["Hkv"] * c["G"], c["N"], c["D"]
        channel = torch.exp(0.5 * randn(D))
        # Head views of a projection's output.
        x = randn(B, N, H + 2 * Hkv, D)
        x[:, :, :H] *= 1.5
        x[:, :, H:H + Hkv] *= channel
        x = x.to(dt).permute(0, 2, 1, 3)
        s = dict(case=c, q=x[:, :H], k=x[:, H:H + Hkv], v=x[:, H + Hkv:])
        s["lengths"] = torch.tensor(_lengths(N, B, True), dtype=torch.int64, device=DEV) if c["ragged"] else None
        if c["grad"]:
            s["dout"] = randn(B, N, H, D).to(dt).permute(0, 2, 1, 3)
            for n in "qkv":
                s[n] = s[n].detach().requires_grad_()
        return s

    if c["op"] == "sample":
        B, V = c["B"], c["V"]
        # A few likely tokens over a broad floor, each row its own share.
        x = randn(B, V) * (1.0 + 1.5 * torch.rand(B, 1, generator=g, device=DEV))
        top = torch.randint(V, (B, min(V, 20)), generator=g, device=DEV)
        x.scatter_add_(1, top, 3.0 * randn(*top.shape).abs())
        s = dict(case=c, u=torch.rand(B, generator=g, device=DEV))
        if c["rows"]:
            r = torch.rand(B, 4, generator=g, device=DEV)
            x.masked_fill_(torch.rand(B, V, generator=g, device=DEV) < 0.01, -math.inf)
            x[:, V // 2] = 0.0  # no row is empty
            # Every seventh row is greedy, every fourth without one of the limits.
            i = torch.arange(B, device=DEV)
            s["temperature"] = torch.where(i % 7 == 3, 0.0, c["temperature"] * (0.7 + 0.6 * r[:, 0]))
            s["top_k"] = torch.where(i % 4 == 1, 0, (c["top_k"] * (0.5 + r[:, 1])).long())
            s["top_p"] = torch.where(i % 4 == 2, 1.0, c["top_p"] * (0.8 + 0.2 * r[:, 2]))
            s["min_p"] = torch.where(i % 4 == 3, 0.0, c["min_p"] * r[:, 3])
        else:
            for n in ("temperature", "top_k", "top_p", "min_p"):
                s[n] = c[n]
        s["logits"] = x.to(dt)
        return s

    s = _prepare_cache(c, g)
    s["parents"] = torch.tensor(_parents(c, seed), dtype=torch.int32, device=DEV)
    if c["op"] == "tree":
        s["q"] = (randn(c["B"], c["T"], c["Hkv"] * c["G"], c["D"]) * 1.5).to(dt).permute(0, 2, 1, 3)
    else:
        tokens, picks = _tokens(c, seed)
        s["tokens"] = torch.tensor(tokens, dtype=torch.int64, device=DEV)
        s["picks"] = torch.tensor(picks, dtype=torch.int64, device=DEV)
    return s


# ---- The framework's calls. ------------------------------------------------------------------

def _own_window(s):
    import dwarf_amd
    c = s["case"]
    out = dwarf_amd.window_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"], lengths=s["lengths"])
    if not c["grad"]:
        return dict(out=out)
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    return dict(out=out.detach(), dq=dq, dk=dk, dv=dv)


def _own_tree(s):
    import dwarf_amd
    c = s["case"]
    return dwarf_amd.paged_tree_step(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["pos"],
                                     s["parents"], window=c["window"] or None, sinks=c["sinks"], k_scale=s["k_scale"],
                                     v_scale=s["v_scale"])


def _own_accept(s):
    import dwarf_amd
    path, counts, token = dwarf_amd.draft_tree_accept(s["tokens"], s["parents"], s["picks"])
    dwarf_amd.paged_kv_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["pos"], counts=counts,
                             rows=path, k_scale=s["k_scale"], v_scale=s["v_scale"])
    return path, counts, token


def _own_sample(s):
    import dwarf_amd
    return dwarf_amd.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                   top_p=s["top_p"], min_p=s["min_p"], return_logprobs=True)


# ---- The same in elementary operations. --------------------------------------------------------

def _plain_window(s):
    c = s["case"]
    q, k, v = (s[n].detach().float() for n in "qkv")
    B, Hkv, G, N, D = c["B"], c["Hkv"], c["G"], c["N"], c["D"]
    W, S, scale = c["window"], c["sinks"], c["D"] ** -0.5
    q = q.reshape(B, Hkv, G, N, D)
    length = s["lengths"] if c["ragged"] else torch.full((B,), N, device=DEV)
    out = torch.empty(B, Hkv, G, N, D, device=DEV)
    if c["grad"]:
        dout = s["dout"].float().reshape(B, Hkv, G, N, D)
        dq, dk, dv = torch.empty_like(q), torch.zeros(B, Hkv, N, D, device=DEV), torch.zeros(B, Hkv, N, D, device=DEV)
    # Queries in blocks: scores of a block against the positions that any of it sees.
    step = max(1, min(N, (1 << 27) // max(1, B * Hkv * G * min(N, W + 1024))))
    for i0 in range(0, N, step):
        i1 = min(N, i0 + step)
        lo = max(0, i0 - W + 1)
        j = torch.cat([torch.arange(min(S, lo), device=DEV), torch.arange(lo, i1, device=DEV)])
        i = torch.arange(i0, i1, device=DEV)[:, None]
        sees = (j <= i) & ((i - j < W) | (j < S))
        sees = sees & (j < length[:, None, None]) & (i < length[:, None, None])
        sees = sees[:, None, None]
        x, kj, vj = q[:, :, :, i0:i1], k[:, :, j], v[:, :, j]
        p = torch.matmul(x.reshape(B, Hkv, -1, D), kj.transpose(2, 3)).view(B, Hkv, G, i1 - i0, -1) * scale
        p = p.masked_fill(~sees, -math.inf)
        top = p.amax(-1, keepdim=True)
        p = torch.exp(p - top.masked_fill(top == -math.inf, 0.0))
        total = p.sum(-1, keepdim=True)
        p = p / total.masked_fill(total == 0, 1.0)
        flat = p.view(B, Hkv, G * (i1 - i0), -1)
        o = torch.matmul(flat, vj)
        out[:, :, :, i0:i1] = o.view(B, Hkv, G, -1, D)
        if c["grad"]:
            do = dout[:, :, :, i0:i1].reshape(B, Hkv, -1, D)
            dv[:, :, j] += torch.matmul(flat.transpose(2, 3), do)
            ds = flat * (torch.matmul(do, vj.transpose(2, 3)) - (do * o).sum(-1, keepdim=True)) * scale
            dq[:, :, :, i0:i1] = torch.matmul(ds, kj).view(B, Hkv, G, -1, D)
            dk[:, :, j] += torch.matmul(ds.transpose(2, 3), x.reshape(B, Hkv, -1, D))
    dt = s["q"].dtype
    res = dict(out=out.view(B, Hkv * G, N, D).to(dt))
    if c["grad"]:
        res.update(dq=dq.view(B, Hkv * G, N, D).to(dt), dk=dk.to(dt), dv=dv.to(dt))
    return res


def _put(pages, scale, ids, slots, rows, cache):
    """rows [n, Hkv, D] to the slots of the pages."""
    if scale is None:
        pages[ids, :, slots] = rows.to(pages.dtype)
        return
    y, e = _quantise(rows, cache)
    pages.view(torch.uint8)[ids, :, slots] = y
    scale.view(torch.uint8)[ids, :, slots] = e


def _gather(pages, scale, table):
    """The values of every position of the table, [B, Hkv, M * page, D] float32."""
    B, M = table.shape
    at = table.clamp(min=0).long()
    _, H, page, D = pages.shape
    if scale is None:
        x = pages[at].float()
    else:
        x = pages.view(torch.uint8)[at].view(pages.dtype).float()
        x = x * scale.view(torch.uint8)[at].view(scale.dtype).float()[..., None]
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, M * page, D)


def _plain_put(s, k, v, counts):
    """Rows i < counts[b] of k and v [B, Hkv, T, D] to positions pos[b] + i."""
    c = s["case"]
    i = torch.arange(k.shape[2], device=DEV)
    b, i = torch.nonzero(i < counts[:, None], as_tuple=True)
    at = s["pos"][b] + i
    ids, slots = s["page_table"][b, at // c["page"]].long(), at % c["page"]
    _put(s["k_pages"], s["k_scale"], ids, slots, k[b, :, i], c["cache"])
    _put(s["v_pages"], s["v_scale"], ids, slots, v[b, :, i], c["cache"])


def _plain_tree(s):
    c, q, pos = s["case"], s["q"], s["pos"]
    B, Hkv, G, T, D = c["B"], c["Hkv"], c["G"], c["T"], c["D"]
    _plain_put(s, s["k"], s["v"], torch.full((B,), T, device=DEV))
    k = _gather(s["k_pages"], s["k_scale"], s["page_table"])
    L = k.shape[2]
    # Each node's ancestors, itself among them, one step towards the root at a time.
    parents = s["parents"].long()
    above = torch.zeros(B, T, T + 1, dtype=torch.bool, device=DEV)
    at = torch.arange(T, device=DEV).expand(B, T)
    for _ in range(T):
        above.scatter_(2, torch.where(at < 0, T, at)[:, :, None], True)
        at = torch.where(at < 0, -1, parents.gather(1, at.clamp(min=0)))
    above = above[:, :, :T]
    depth = above.sum(-1) - 1
    t = torch.arange(L, device=DEV)
    node = t - pos[:, None]                                    # [B, L]
    inside = (node >= 0) & (node < T)
    sees = (node < 0)[:, None, :] | (above.gather(2, node.clamp(0, T - 1)[:, None].expand(B, T, L)) & inside[:, None, :])
    if c["window"]:
        place = torch.where(inside, pos[:, None] + depth.gather(1, node.clamp(0, T - 1)), t)
        own_place = pos[:, None] + depth
        near = own_place[:, :, None] - place[:, None, :] < c["window"]
        sees = sees & (near | (place < c["sinks"])[:, None, :])
    x = torch.matmul(q.float().reshape(B, Hkv, G * T, D), k.transpose(2, 3)) * D ** -0.5
    del k
    x = x.view(B, Hkv, G, T, L).masked_fill(~sees[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    # Values that no node sees are no part of a sum, whatever the pages hold there.
    v = _gather(s["v_pages"], s["v_scale"], s["page_table"]).masked_fill(~sees.any(1)[:, None, :, None], 0.0)
    return torch.matmul(x.view(B, Hkv, G * T, L), v).view(B, Hkv * G, T, D).to(q.dtype)


def _plain_accept(s):
    tokens, parents, picks = s["tokens"], s["parents"].long(), s["picks"]
    B, T = tokens.shape
    at = torch.zeros(B, dtype=torch.int64, device=DEV)
    path = torch.full((B, T), -1, dtype=torch.int64, device=DEV)
    path[:, 0] = 0
    going = torch.ones(B, dtype=torch.bool, device=DEV)
    i = torch.arange(T, device=DEV)
    for step in range(1, T):
        fits = (parents == at[:, None]) & (tokens == picks.gather(1, at[:, None]))
        first = torch.where(fits, i, T).amin(1)
        going = going & (first < T)
        at = torch.where(going, first, at)
        path[:, step] = torch.where(going, first, -1)
    counts = (path >= 0).sum(1)
    index = path.clamp(min=0)[:, None, :, None].expand(B, s["k"].shape[1], T, s["k"].shape[3])
    _plain_put(s, s["k"].gather(2, index), s["v"].gather(2, index), counts)
    return path, counts, picks.gather(1, at[:, None])[:, 0]


def _plain_sample(s):
    # In 64 bits: the running sums decide between neighbours.
    x = s["logits"].double()
    B, V = x.shape

    def rows(n):
        t = s[n]
        return t.double()[:, None] if torch.is_tensor(t) else torch.full((B, 1), t, dtype=torch.float64, device=DEV)

    temperature, top_k, top_p, min_p = (rows(n) for n in ("temperature", "top_k", "top_p", "min_p"))
    x, index = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / temperature.clamp(min=1e-30))
    w = torch.where((top_k > 0) & (torch.arange(V, device=DEV) >= top_k), 0.0, w)
    run = torch.cumsum(w, 1)
    w = torch.where((top_p < 1) & (run - w > top_p * run[:, -1:]), 0.0, w)
    w = torch.where(w < min_p, 0.0, w)
    w = torch.zeros_like(w).scatter_(1, index, w)
    run = torch.cumsum(w, 1)
    token = (run <= s["u"].double()[:, None] * run[:, -1:]).sum(1)
    logprob = torch.log(w.gather(1, token[:, None]) / run[:, -1:])[:, 0]
    hot = temperature[:, 0] > 0
    return torch.where(hot, token, index[:, 0]), torch.where(hot, logprob, 0.0).float()


def run(s):
    op = s["case"]["op"]
    if op == "window":
        return _own_window(s) if own else _plain_window(s)
    if op == "sample":
        return _own_sample(s) if own else _plain_sample(s)
    if op == "tree":
        res = dict(out=_own_tree(s) if own else _plain_tree(s))
    else:
        res = dict(zip(("path", "counts", "token"), _own_accept(s) if own else _plain_accept(s)))
    # The updated state: an 8-bit pool is its values up to the rows' scales, and those.
    return dict(res, k_pages=s["k_pages"], v_pages=s["v_pages"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def work(c):
    e = SIZES[c["dtype"]]
    if c["op"] == "sample":
        return dict(bytes=c["B"] * (c["V"] * e + 16 + (20 if c["rows"] else 0)), flops=0.0)
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    if c["op"] == "window":
        H = Hkv * c["G"]
        pairs = sum(_pairs(n, c["window"], c["sinks"]) for n in _lengths(c["N"], B, c["ragged"]))
        row = B * c["N"] * D * e
        # Queries, keys and values read and the output written; in training dout read and three gradients written.
        return dict(bytes=row * (4 * H + 4 * Hkv) if c["grad"] else row * (2 * H + 2 * Hkv),
                    flops=pairs * H * D * (14.0 if c["grad"] else 4.0))
    z, T = SIZES[c["cache"]], c["T"]
    row = 2 * Hkv * (D * z + (z == 1))  # a position's key and value rows in the pools
    new = 2 * Hkv * D * e               # ... as the caller has them
    if c["op"] == "accept":
        n = sum(len(_walk(p, t, x)) for p, t, x in zip(_parents(c, 0), *_tokens(c, 0)))
        return dict(bytes=n * (new + row) + B * (T * 28 + 8 + 16) + 4 * B, flops=0.0)
    H = Hkv * c["G"]
    read = pairs = pages = 0
    for b, n in enumerate(_lengths(c["length"], B, c["ragged"])):
        depth = _depths(_parents(c, 0)[b])
        # Stored positions that some node sees, and the pairs of nodes and stored or drafted positions.
        first = max(0, n - c["window"] + 1) if c["window"] else 0
        read += n - first + min(c["sinks"], first)
        pages += -(-(n - first + T) // c["page"]) + (c["sinks"] > 0)
        for d in depth:
            lo = max(0, n + d - c["window"] + 1) if c["window"] else 0
            pairs += n + d + 1 - lo + min(c["sinks"], lo)
    return dict(bytes=read * row + B * T * (new + row) + 2 * B * H * T * D * e + 4 * pages + 8 * B + 4 * B * T,
                flops=4.0 * pairs * H * D)


# ---- From the definition, in 64 bits. -----------------------------------------------------------

def _pow2(e):
    """2^e exactly, e whole numbers in float64."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored64(x, cache):
    """What an 8-bit cache keeps of the rows x (float64)."""
    top, bits = (448.0, 3) if cache == "e4m3" else (127.0, None)
    size = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(size / top)).clamp(min=-200.0)
    e = torch.where(size > top * _pow2(e), e + 1, torch.where(size <= top * _pow2(e - 1), e - 1, e))
    e = torch.where(size == 0, torch.full_like(e, -127.0), e.clamp(min=-127.0))
    y = x / _pow2(e)
    if bits is None:
        step = torch.ones_like(y)
    else:  # three bits behind the leading one, down to steps of 2^-9
        lead = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30)))
        lead = torch.where(y.abs() >= _pow2(lead + 1), lead + 1, torch.where(y.abs() < _pow2(lead), lead - 1, lead))
        step = _pow2(lead.clamp(min=-6.0) - bits)
    return torch.round(y / step) * step * _pow2(e)


def _stored_rows(s, n, b, length):
    """The rows 0 .. length - 1 of sequence b in pool n ("k" or "v"), [Hkv, length, D] float64."""
    page = s["case"]["page"]
    ids = s["page_table"][b, :-(-length // page)].tolist()
    rows = torch.cat([s[n + "_pages"][i].double() for i in ids], dim=1)
    if s[n + "_scale"] is not None:
        e = torch.cat([s[n + "_scale"][i].view(torch.uint8) for i in ids], dim=1).double()
        rows = rows * _pow2(e - 127.0)[..., None]
    return rows[:, :length].clone()


def _exact_window(c, s):
    B, Hkv, G, N, D = c["B"], c["Hkv"], c["G"], c["N"], c["D"]
    H = Hkv * G
    res = {"out": torch.zeros(B, H, N, D, dtype=torch.float64, device=DEV)}
    if c["grad"]:
        res.update(dq=torch.zeros_like(res["out"]), dk=torch.zeros(B, Hkv, N, D, dtype=torch.float64, device=DEV),
                   dv=torch.zeros(B, Hkv, N, D, dtype=torch.float64, device=DEV))
    for b, n in enumerate(_lengths(N, B, c["ragged"])):
        i = torch.arange(n, device=DEV)
        hidden = (i > i[:, None]) | ((i[:, None] - i >= c["window"]) & (i >= c["sinks"]))
        for h in range(H):
            q, k, v = (s[t][b, x, :n].detach().double().requires_grad_(c["grad"])
                       for t, x in (("q", h), ("k", h // G), ("v", h // G)))
            with torch.set_grad_enabled(c["grad"]):
                out = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), dim=-1) @ v
            res["out"][b, h, :n] = out.detach()
            if c["grad"]:
                dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"][b, h, :n].double())
                res["dq"][b, h, :n] = dq
                res["dk"][b, h // G, :n] += dk
                res["dv"][b, h // G, :n] += dv
    return res


def _exact_tree(c, s, seed):
    B, Hkv, G, T, D, cache = c["B"], c["Hkv"], c["G"], c["T"], c["D"], c["cache"]
    keep = (lambda x: _stored64(x, cache)) if SIZES[cache] == 1 else (lambda x: x)
    out = torch.empty(B, Hkv, G, T, D, dtype=torch.float64, device=DEV)
    for b, (n, parents) in enumerate(zip(_lengths(c["length"], B, c["ragged"]), _parents(c, seed))):
        depth = _depths(parents)
        k, v = (torch.cat([_stored_rows(s, x, b, n), keep(s[x][b].double())], dim=1) for x in "kv")
        place = list(range(n)) + [n + d for d in depth]
        sees = np.zeros((T, n + T), dtype=bool)
        for i in range(T):
            lo = max(0, n + depth[i] - c["window"] + 1) if c["window"] else 0
            line = {i}
            while parents[min(line)] >= 0:
                line.add(parents[min(line)])
            sees[i, lo:n] = True
            sees[i, :min(n, c["sinks"])] = True
            for j in line:
                sees[i, n + j] = place[n + j] >= lo or place[n + j] < c["sinks"]
        hidden = ~torch.from_numpy(sees).to(DEV)
        x = s["q"][b].double().view(Hkv, G, T, D) @ k.mT.contiguous()[:, None] / math.sqrt(D)
        out[b] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v[:, None]
    return dict(out=out.view(B, Hkv * G, T, D), k_pages=None, v_pages=None, k_scale=None, v_scale=None)


def _exact_accept(c, seed):
    parents, (tokens, picks) = _parents(c, seed), _tokens(c, seed)
    paths = [_walk(p, t, x) for p, t, x in zip(parents, tokens, picks)]
    T = c["T"]
    return dict(path=torch.tensor([p + [-1] * (T - len(p)) for p in paths], device=DEV),
                counts=torch.tensor([len(p) for p in paths], device=DEV),
                token=torch.tensor([x[p[-1]] for p, x in zip(paths, picks)], device=DEV),
                k_pages=None, v_pages=None, k_scale=None, v_scale=None)


def _exact_sample(c, s):
    x = s["logits"].double().cpu().numpy()
    B, V = x.shape
    u = s["u"].double().cpu().numpy()

    def rows(n):
        return s[n].double().cpu().numpy() if torch.is_tensor(s[n]) else np.full(B, s[n], dtype=np.float64)

    temperature, top_k, top_p, min_p = (rows(n) for n in ("temperature", "top_k", "top_p", "min_p"))
    tokens, logprobs = np.empty(B, dtype=np.int64), np.zeros(B)
    for b in range(B):
        order = np.argsort(-x[b], kind="stable")
        if temperature[b] <= 0:
            tokens[b] = order[0]
            continue
        if top_k[b] > 0:
            order = order[:int(top_k[b])]
        w = np.exp((x[b][order] - x[b][order[0]]) / temperature[b])
        before = np.concatenate([[0.0], np.cumsum(w)])
        if top_p[b] < 1:
            n = int(np.searchsorted(before[:-1], top_p[b] * before[-1], side="right"))
            order, w = order[:n], w[:n]
        order, w = order[w >= min_p[b]], w[w >= min_p[b]]
        by_index = np.argsort(order)
        total = np.cumsum(w[by_index])
        at = by_index[np.searchsorted(total, u[b] * total[-1], side="right")]
        tokens[b], logprobs[b] = order[at], math.log(w[at]) - math.log(total[-1])
    return torch.from_numpy(tokens).to(DEV), torch.from_numpy(logprobs).to(DEV)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "window":
        return _exact_window(c, s)
    if c["op"] == "tree":
        return _exact_tree(c, s, seed)
    if c["op"] == "accept":
        return _exact_accept(c, seed)
    return _exact_sample(c, s)
