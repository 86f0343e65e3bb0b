"""Speculation on a tree of drafted tokens: the four operators of one
iteration, each by itself, at the sizes a serving loop calls them with.

* ``draft``  -- the n-gram drafter that merges the continuations of several
  earlier occurrences of the last tokens into one tree of at most T nodes.
* ``attn``   -- attention of the T nodes of every sequence over its cached
  slots and over the node's own ancestors, with head RMSNorm and RoPE at the
  node's position folded in; the nodes' keys and values are left in buffers
  of their own.
* ``accept`` -- the walk down the tree along the model's greedy picks, which
  extends the history and the lengths.
* ``commit`` -- the accepted path's keys and values copied into the cache, in
  every layer.

A tree is ``parents[b, t] < t`` (node 0 is the root, the current token; -1 or
any other value is no node, nor are its descendants).  Layouts are those of
include/qdec.h: K cache ``[batch, kv heads, cap, D]``, V cache
``[batch, kv heads, cap/8, D, 8]``, node keys and values
``[batch, kv heads, T, D]`` per layer.

Cached keys and values, and the raw projection rows, are N(0, 1); norm gains
are N(1, 0.05).
"""

import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
THETA = 5e6
VOCAB = 151936
# query heads, kv heads, head_dim: the small test configuration, then the
# layouts of the Qwen3 family (2, 4, 5 and 8 query heads per kv head)
LAYOUTS = [(8, 2, 64), (16, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 128)]


def _attn(name, layout, batch, t, lo, hi):
    nq, nkv, d = layout
    return {"name": name, "kind": "attn", "nq": nq, "nkv": nkv, "d": d, "batch": batch, "t": t, "lo": lo, "hi": hi}


def _draft(name, batch, lo, hi, t, depth, matches):
    return {"name": name, "kind": "draft", "batch": batch, "lo": lo, "hi": hi, "t": t, "depth": depth,
            "matches": matches}


def _accept(name, batch, t, lo, hi):
    return {"name": name, "kind": "accept", "batch": batch, "t": t, "lo": lo, "hi": hi}


def _commit(name, layers, nkv, d, batch, t, lo, hi):
    return {"name": name, "kind": "commit", "layers": layers, "nkv": nkv, "d": d, "batch": batch, "t": t, "lo": lo,
            "hi": hi}


def listed():
    return [
        # The smallest call: the two-layer test configuration, one sequence
        # of 200 tokens, 8 nodes.  Launch latency.
        _attn("attn-tiny", LAYOUTS[0], 1, 8, 200, 200),
        # One user of Qwen3-4B half way through the headline workload (512
        # prompt tokens, 256 new), the 16 nodes that fill one matrix tile.
        _attn("attn-b1-t16", LAYOUTS[2], 1, 16, 640, 640),
        # The widest tree on one user's long chat.
        _attn("attn-b1-t64", LAYOUTS[2], 1, 64, 4100, 4100),
        # A small server batch of unequal lengths, one of them just begun.
        _attn("attn-b8-t8", LAYOUTS[2], 8, 8, 0, 1600),
        # A large batch with few nodes each: the cache read bounds it.
        _attn("attn-b32-t4", LAYOUTS[1], 32, 4, 2000, 4224),
        # The largest: two long documents, wide trees, 8 query heads per kv
        # head (512 query rows on every kv head).
        _attn("attn-b2-t64-g8", LAYOUTS[4], 2, 64, 30011, 32700),
        # The drafter on one user's chat, and on a batch of long histories.
        _draft("draft-b1", 1, 600, 600, 16, 8, 16),
        _draft("draft-b16-long", 16, 8000, 32000, 8, 12, 32),
        # Acceptance of one user's tree and of a whole batch's.
        _accept("accept-b1", 1, 16, 640, 640),
        _accept("accept-b32", 32, 4, 2000, 4224),
        # The accepted path of one tree, 36 layers of 8 kv heads; and of a
        # batch's trees, the widest that 128 verify rows allow it.
        _commit("commit-b1", 36, 8, 128, 1, 16, 640, 640),
        _commit("commit-b8", 36, 8, 128, 8, 16, 500, 1600),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_rows(rng):
    """Batch and nodes of a pass of at most 128 rows."""
    batch = _log_int(rng, 1, 64)
    return batch, _log_int(rng, 1, min(64, 128 // batch))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "draft", "accept", "commit"])
    batch, t = _draw_rows(rng)
    if kind == "draft":
        hi = _log_int(rng, 2, min(31000, 300000 // batch))
        c = _draft("", batch, rng.randint(0, hi), hi, t, rng.randint(1, 12), rng.randint(1, 32 if batch <= 16 else 16))
    elif kind == "attn":
        layout = rng.choice(LAYOUTS)
        hi = _log_int(rng, 1, min(31000, 62000 // batch))
        c = _attn("", layout, batch, t, rng.choice([0, hi // 2, hi]), hi)
    elif kind == "accept":
        hi = _log_int(rng, 1, 4224 if batch <= 32 else 2048)
        c = _accept("", batch, t, rng.randint(0, hi), hi)
    else:
        layers, (nkv, d) = rng.choice([2, 24, 28, 36]), rng.choice([(2, 64), (8, 128), (4, 128)])
        # the caches of the largest listed case
        hi = _log_int(rng, 1, min(4224, 450_000_000 // (layers * batch * nkv * d)))
        c = _commit("", layers, nkv, d, batch, t, rng.randint(0, hi), hi)
    del c["name"]
    return c


# ------------------------------------------------------------------- inputs


def _lens(case, rnd):
    """Cached slots of every sequence: the ends of the range are met."""
    n = case["batch"]
    out = [rnd.randint(case["lo"], case["hi"]) for _ in range(n)]
    out[-1] = case["hi"]
    if n > 1:
        out[0] = case["lo"]
    return out


def _cap(case):
    return (case["hi"] + case["t"] + 1 + 31) // 32 * 32


def _trees(case, rnd):
    """Parents of every sequence's nodes as a drafter leaves them: runs with
    side branches, and in some sequences fewer nodes than rows."""
    rows = []
    for b in range(case["batch"]):
        t = case["t"]
        live = t if rnd.random() < 0.6 else rnd.randint(1, t)
        p = [-1] * t
        for i in range(1, live):
            p[i] = i - 1 if rnd.random() < 0.7 else rnd.randrange(i)
        rows.append(p)
    return rows


def _gen(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _history(rnd, length, cap):
    """Tokens made of recurring phrases, as code and chats are."""
    phrases = [[rnd.randrange(VOCAB) for _ in range(rnd.randint(3, 14))] for _ in range(40)]
    h = []
    while len(h) < length + 1:
        p = rnd.choice(phrases)
        h += p[:rnd.randint(2, len(p))]
        if rnd.random() < 0.2:
            h.append(rnd.randrange(VOCAB))
    return h[:length + 1] + [0] * (cap - length - 1)


def _path(parents, rnd):
    """A walk down the tree that stops somewhere, as node indices."""
    path = [0]
    while rnd.random() < 0.75:
        kids = [i for i, p in enumerate(parents) if p == path[-1] and i > path[-1]]
        if not kids:
            break
        path.append(rnd.choice(kids))
    return path


def _inputs(case, seed):
    rnd = random.Random(seed)
    g = _gen(seed, DEV)
    B, T, cap = case["batch"], case["t"], _cap(case)
    lens = _lens(case, rnd)
    st = {"case": case, "cap": cap, "lens": _i32(lens)}

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)

    if case["kind"] == "draft":
        st["hist"] = _i64([_history(rnd, n, cap) for n in lens])
        st["ids"] = torch.zeros((B, T), dtype=torch.int64, device=DEV)
        st["parents"] = torch.zeros((B, T), dtype=torch.int32, device=DEV)
        return st
    trees = _trees(case, rnd)
    st["parents"] = _i32(trees)
    if case["kind"] == "attn":
        nq, nkv, d = case["nq"], case["nkv"], case["d"]
        st["qkv"] = normal(B * T, (nq + 2 * nkv) * d)
        st["q_norm"] = (1 + 0.05 * normal(d).float()).to(torch.bfloat16)
        st["k_norm"] = (1 + 0.05 * normal(d).float()).to(torch.bfloat16)
        st["k_cache"] = normal(B, nkv, cap, d)
        st["v_cache"] = normal(B, nkv, cap // 8, d, 8)
        inv = 1.0 / (THETA ** (torch.arange(0, d, 2, dtype=torch.float32) / d))
        ang = torch.arange(cap, dtype=torch.float32)[:, None] * inv[None, :]
        ang = torch.cat((ang, ang), -1)
        st["cos"], st["sin"] = ang.cos().to(DEV, torch.bfloat16), ang.sin().to(DEV, torch.bfloat16)
        st["out"] = torch.zeros((B * T, nq * d), dtype=torch.bfloat16, device=DEV)
        st["k_nodes"] = torch.zeros((B, nkv, T, d), dtype=torch.bfloat16, device=DEV)
        st["v_nodes"] = torch.zeros((B, nkv, T, d), dtype=torch.bfloat16, device=DEV)
        return st
    paths = [_path(p, rnd) for p in trees]
    if case["kind"] == "accept":
        # Children of one node hold different tokens; along a path the pick
        # equals the child's token, elsewhere it is any token.
        ids = [[rnd.randrange(VOCAB // T) * T + t for t in range(T)] for _ in range(B)]
        pick = [[rnd.randrange(VOCAB) for _ in range(T)] for _ in range(B)]
        for b, p in enumerate(paths):
            for i in range(len(p) - 1):
                pick[b][p[i]] = ids[b][p[i + 1]]
        st["ids"], st["out_tok"] = _i64(ids), _i64(pick)
        st["hist"] = _i64([_history(rnd, n, cap) for n in lens])
        st["lens_out"], st["naccept"] = torch.zeros_like(st["lens"]), torch.zeros_like(st["lens"])
        st["path"] = torch.zeros((B, T), dtype=torch.int32, device=DEV)
        st["emit"] = torch.zeros((B, T), dtype=torch.int64, device=DEV)
        # the last sequence of a larger batch already has all its tokens
        st["stop"] = max(lens) if B > 1 else max(lens) + 8
        return st
    nl, nkv, d = case["layers"], case["nkv"], case["d"]
    st["k_nodes"], st["v_nodes"] = normal(nl, B, nkv, T, d), normal(nl, B, nkv, T, d)
    st["k_cache"], st["v_cache"] = normal(nl, B, nkv, cap, d), normal(nl, B, nkv, cap // 8, d, 8)
    st["path"] = _i32([p + [-1] * (T - len(p)) for p in paths])
    st["naccept"] = _i32([len(p) - 1 for p in paths])
    st["lens"] = _i32([n + len(p) for n, p in zip(lens, paths)])  # lengths after the acceptance
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _prepare_own(st)
    return st


def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


# ------------------------------------------------------- the framework's calls


def _prepare_own(st):
    """The argument block, the workspace and the library handle that a
    decode loop builds once per shape and keeps."""
    pkg = os.path.join(os.getcwd(), "dryft-challenge_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from qdec import capi

    c = st["case"]
    lib = st["lib"] = capi.lib()
    ptr = {k: v.data_ptr() for k, v in st.items() if isinstance(v, torch.Tensor)}
    if c["kind"] == "draft":
        a = capi.TreeDraftArgs()
        a.primary, a.backoff, a.depth, a.matches = 3, 2, c["depth"], c["matches"]
    elif c["kind"] == "attn":
        a = capi.TreeAttnArgs()
        a.nq, a.nkv, a.head_dim, a.eps, a.sm_scale = c["nq"], c["nkv"], c["d"], EPS, c["d"] ** -0.5
        ptr.update(q_norm_w=ptr["q_norm"], k_norm_w=ptr["k_norm"], cos_tab=ptr["cos"], sin_tab=ptr["sin"])
    elif c["kind"] == "accept":
        a = capi.TreeAcceptArgs()
        a.stop_len = st["stop"]
    else:
        a = capi.TreeCommitArgs()
        a.n_layers, a.nkv, a.head_dim = c["layers"], c["nkv"], c["d"]
    a.batch, a.cap, a.t_rows = c["batch"], st["cap"], c["t"]
    fields = {f[0] for f in a._fields_}
    for k, v in ptr.items():
        if k in fields:
            setattr(a, k, v)
    if c["kind"] == "attn":
        pb, _ = lib.tree_attn_workspace(a)  # no counters
        st["partial"] = torch.zeros((max(pb, 16) // 4,), dtype=torch.float32, device=DEV)
        a.partial = st["partial"].data_ptr()
    st["args"] = a


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_draft(st):
    st["lib"].tree_draft(st["args"], _stream())
    return st["ids"], st["parents"]


def _own_attn(st):
    st["lib"].tree_attn(st["args"], _stream())
    return st["out"], st["k_nodes"], st["v_nodes"]


def _own_accept(st):
    st["lib"].tree_accept(st["args"], _stream())
    return st["hist"], st["lens_out"], st["naccept"], st["path"], st["emit"]


def _own_commit(st):
    st["lib"].tree_commit(st["args"], _stream())
    return st["k_cache"], st["v_cache"]


_OWN = {"draft": _own_draft, "attn": _own_attn, "accept": _own_accept, "commit": _own_commit}


# --------------------------------------------------------------- plain forms


def _plain_draft(st, primary=3, backoff=2):
    """The trie of the candidates, all at once: candidate m adds the nodes
    past its longest common prefix with an earlier candidate, and nodes are
    numbered by (candidate, depth)."""
    c = st["case"]
    hist, L, cap = st["hist"], st["lens"].long()[:, None], st["cap"]
    B, T, K, M = c["batch"], c["t"], c["depth"], c["matches"]
    pos = torch.arange(cap, device=DEV)[None, :]
    starts, lengths = [], []
    for n in (primary, backoff):
        # e: the last position of an earlier occurrence of the pattern that ends at L
        ok = (pos >= n - 1) & (pos <= L - 1)
        for i in range(n):
            want = hist.gather(1, (L - i).clamp(min=0))
            ok &= (hist.roll(i, 1) == want) & (L - i >= 0)
        rank = torch.where(ok, pos, -1)
        e = rank.topk(min(M, cap), dim=1).values  # most recent first
        starts.append(e + 1)
        lengths.append(torch.where(e >= 0, (L - e).clamp(max=K), 0))
    s, n = torch.cat(starts, 1), torch.cat(lengths, 1)
    N = s.shape[1]
    d = torch.arange(K, device=DEV)
    tok = hist.gather(1, (s[:, :, None] + d).clamp(max=cap - 1).reshape(B, -1)).view(B, N, K)
    inside = d < n[:, :, None]
    same = (tok[:, :, None] == tok[:, None]) & inside[:, :, None] & inside[:, None]
    lcp = same.long().cumprod(-1).sum(-1)  # [B, N, N]
    earlier = torch.ones((N, N), device=DEV, dtype=torch.bool).tril(-1)
    best = torch.where(earlier, lcp, 0).amax(-1)
    new = n - best
    first = 1 + new.cumsum(1) - new
    # node of (m, d): its own when d >= best[m], else that of the first
    # candidate that shares its first d + 1 tokens
    node = torch.where(d >= best[:, :, None], first[:, :, None] + d - best[:, :, None], 0)
    shares = (lcp[:, :, :, None] > d) & earlier[None, :, :, None]  # [B, N, N, K]
    owner = shares.long().argmax(2)  # the first
    inherited = node.gather(1, owner)
    node = torch.where(d >= best[:, :, None], node, inherited)
    parent = torch.cat((torch.zeros_like(node[:, :, :1]), node[:, :, :-1]), 2)
    keep = inside & (d >= best[:, :, None]) & (node < T)
    slot = torch.where(keep, node, T).reshape(B, -1)  # T: thrown away
    ids = torch.zeros((B, T + 1), dtype=torch.int64, device=DEV)
    par = torch.full((B, T + 1), -1, dtype=torch.int64, device=DEV)
    ids.scatter_(1, slot, tok.reshape(B, -1))
    par.scatter_(1, slot, parent.reshape(B, -1))
    ids[:, 0] = hist.gather(1, L)[:, 0]
    par[:, 0] = -1
    return ids[:, :T].contiguous(), par[:, :T].to(torch.int32)


def _ancestors(parents):
    """[B, T, T] truth values: node j is t or an ancestor of t; rows of no
    node are empty."""
    B, T = parents.shape
    t = torch.arange(T, device=DEV)
    p = parents.long()
    anc = torch.zeros((B, T, T), dtype=torch.bool, device=DEV)
    anc[:, 0, 0] = True
    for i in range(1, T):
        pi = p[:, i]
        up = anc.gather(1, pi.clamp(0, T - 1)[:, None, None].expand(B, 1, T))[:, 0]
        ok = (pi >= 0) & (pi < i) & up.any(1)
        anc[:, i] = ok[:, None] & (up | (t == i))
    return anc


def _plain_attn(st):
    c = st["case"]
    nq, nkv, D, B, T, cap = c["nq"], c["nkv"], c["d"], c["batch"], c["t"], st["cap"]
    G = nq // nkv
    anc = _ancestors(st["parents"])
    live = anc.any(2)
    pos = (st["lens"].long()[:, None] + anc.sum(2) - 1).clamp(0, cap - 1)
    x = st["qkv"].float().view(B, T, nq + 2 * nkv, D)
    q, k, v = x[:, :, :nq], x[:, :, nq:nq + nkv], x[:, :, nq + nkv:]
    cos, sin = st["cos"].float()[pos][:, :, None], st["sin"].float()[pos][:, :, None]

    def norm_rope(y, w):
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        rot = torch.cat((-y[..., D // 2:], y[..., :D // 2]), -1)
        return y * cos + rot * sin

    q, k = norm_rope(q, st["q_norm"]), norm_rope(k, st["k_norm"])
    k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)  # [B, nkv, T, D]
    q = q.view(B, T, nkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, D)
    kc = st["k_cache"].float()
    vc = st["v_cache"].float().permute(0, 1, 2, 4, 3).reshape(B, nkv, cap, D)
    keys, vals = torch.cat((kc, k), 2), torch.cat((vc, v), 2)
    cached = torch.arange(cap, device=DEV)[None, None] < st["lens"].long()[:, None, None]
    sees = torch.cat((cached & live[:, :, None], anc), 2)  # [B, T, cap + T]
    sees = sees[:, None, :, None].expand(B, 1, T, G, cap + T).reshape(B, 1, T * G, cap + T)
    s = torch.matmul(q, keys.transpose(2, 3).contiguous()) * D ** -0.5
    s = torch.where(sees, s, -torch.inf)
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)  # a row that sees nothing
    p = torch.exp(s - m)
    o = torch.matmul(p, vals) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(B, nkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(B * T, nq * D)
    st["out"].copy_(o)
    put = live[:, None, :, None]
    st["k_nodes"].copy_(torch.where(put, k, st["k_nodes"].float()))
    st["v_nodes"].copy_(torch.where(put, v, st["v_nodes"].float()))
    return st["out"], st["k_nodes"], st["v_nodes"]


def _plain_accept(st):
    c = st["case"]
    B, T, cap = c["batch"], c["t"], st["cap"]
    ids, pick, L = st["ids"], st["out_tok"], st["lens"].long()
    par = st["parents"].long()
    t = torch.arange(T, device=DEV)[None]
    live = L < st["stop"]
    cur = torch.zeros((B, 1), dtype=torch.int64, device=DEV)
    going = live[:, None]
    path = torch.full((B, T), -1, dtype=torch.int64, device=DEV)
    emit = torch.full((B, T), -1, dtype=torch.int64, device=DEV)
    count = torch.zeros((B, 1), dtype=torch.int64, device=DEV)
    for i in range(T):
        path[:, i:i + 1] = torch.where(going, cur, -1)
        want = pick.gather(1, cur)
        emit[:, i:i + 1] = torch.where(going, want, -1)
        count += going
        child = (par == cur) & (t > cur) & (ids == want) & going
        going = child.any(1, keepdim=True)
        cur = torch.where(going, child.long().argmax(1, keepdim=True), cur)
    at = L[:, None] + 1 + t
    ok = (emit >= 0) & (at >= 0) & (at < cap)
    # entries that are not written put the row's last kept value back
    at = torch.where(ok, at, L[:, None].clamp(0, cap - 1))
    val = torch.where(ok, emit, st["hist"].gather(1, L[:, None].clamp(0, cap - 1)))
    st["hist"].scatter_(1, at, val)
    st["lens_out"].copy_(L + count[:, 0])
    st["naccept"].copy_((count[:, 0] - 1).clamp(min=0))
    st["path"].copy_(path)
    st["emit"].copy_(emit)
    return st["hist"], st["lens_out"], st["naccept"], st["path"], st["emit"]


def _plain_commit(st):
    c = st["case"]
    B, T, cap, nkv, D, nl = c["batch"], c["t"], st["cap"], c["nkv"], c["d"], c["layers"]
    path = st["path"].long()
    n = st["naccept"].long()[:, None] + 1
    t = torch.arange(T, device=DEV)[None]
    ok = (t < n) & (path >= 0)
    # entries past the path repeat its first one
    src = torch.where(ok, path, path[:, :1]).clamp(min=0)
    dst = st["lens"].long()[:, None] - n + torch.where(ok, t, 0)
    b = torch.arange(B, device=DEV)[:, None].expand(B, T)
    k = st["k_nodes"][:, b, :, src]  # [B, T, layers, nkv, D]
    v = st["v_nodes"][:, b, :, src]
    st["k_cache"][:, b, :, dst] = k
    # [B, T, layers, nkv, D]: slot dst of the channel-major cache
    st["v_cache"][:, b, :, dst // 8, :, dst % 8] = v
    return st["k_cache"], st["v_cache"]


_PLAIN = {"draft": _plain_draft, "attn": _plain_attn, "accept": _plain_accept, "commit": _plain_commit}


# ------------------------------------------------- what a pass cannot do without


def work(case):
    B, T, kind = case["batch"], case["t"], case["kind"]
    mean = (case["lo"] + case["hi"]) / 2 if B > 1 else case["hi"]
    if kind == "draft":
        return {"bytes": int(B * (8 * (mean + 1) + 4 + 12 * T)), "flops": int(B * mean)}
    if kind == "accept":
        return {"bytes": B * (T * (8 + 8 + 4 + 4 + 8) + 12 + 8 * T), "flops": B * T}
    if kind == "commit":
        # a path of about four nodes; each value read once and written once
        n = min(T, 4)
        return {"bytes": case["layers"] * B * case["nkv"] * n * case["d"] * 2 * 2 * 2, "flops": 1}
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    cache = 2 * 2 * B * nkv * mean * d
    rows = 2 * B * T * d * ((nq + 2 * nkv) + nq + 2 * nkv)
    return {"bytes": int(cache + rows), "flops": int(4 * B * T * nq * d * (mean + (T + 1) / 2))}


# --------------------------------------------------------- the definition, in 64 bits


def _exact_draft(case, st):
    B, T, K, M = case["batch"], case["t"], case["depth"], case["matches"]
    ids, par = [], []
    for h, L in zip(st["hist"].tolist(), st["lens"].tolist()):
        toks, parents, kids = [h[L]], [-1], [{}]
        for n in (3, 2):
            if L < n:
                continue
            pattern, found = h[L - n + 1:L + 1], 0
            for j in range(L - n, -1, -1):
                if found == M:
                    break
                if h[j + n - 1] != pattern[-1] or h[j:j + n] != pattern:
                    continue
                found += 1
                cur = 0
                for x in h[j + n:min(j + n + K, L + 1)]:
                    if x not in kids[cur]:
                        if len(toks) == T:
                            break
                        kids[cur][x] = len(toks)
                        toks.append(x)
                        parents.append(cur)
                        kids.append({})
                    cur = kids[cur][x]
        ids.append(toks + [0] * (T - len(toks)))
        par.append(parents + [-1] * (T - len(parents)))
    return _i64(ids), _i32(par)


def _up(parents):
    """Per node the list of its ancestors from the root to itself, or None."""
    out = [[0]]
    for t, p in enumerate(parents):
        if t:
            out.append(out[p] + [t] if 0 <= p < t and out[p] is not None else None)
    return out


def _exact_attn(case, st):
    nq, nkv, D, T, cap = case["nq"], case["nkv"], case["d"], case["t"], st["cap"]
    G = nq // nkv
    out = torch.zeros((case["batch"], T, nq, D), dtype=torch.float64, device=DEV)
    kn, vn = st["k_nodes"].double(), st["v_nodes"].double()
    x = st["qkv"].double().view(case["batch"], T, -1, D)
    cos, sin = st["cos"].double(), st["sin"].double()
    for b, (parents, L) in enumerate(zip(st["parents"].tolist(), st["lens"].tolist())):
        up = _up(parents)
        nodes = [t for t in range(T) if up[t] is not None]
        pos = _i64([L + len(up[t]) - 1 for t in nodes])

        def turned(rows, w):
            r = rows / torch.sqrt(rows.square().mean(-1, keepdim=True) + EPS) * w.double()
            half = torch.cat([r[..., D // 2:].neg(), r[..., :D // 2]], -1)
            return r * cos[pos][:, None] + half * sin[pos][:, None]

        xb = x[b, nodes]
        q, k = turned(xb[:, :nq], st["q_norm"]), turned(xb[:, nq:nq + nkv], st["k_norm"])
        v = xb[:, nq + nkv:]
        kn[b][:, nodes], vn[b][:, nodes] = k.transpose(0, 1), v.transpose(0, 1)
        index = {t: i for i, t in enumerate(nodes)}
        mask = torch.full((len(nodes), len(nodes)), -math.inf, dtype=torch.float64)
        for i, t in enumerate(nodes):
            mask[i, [index[j] for j in up[t]]] = 0.0
        mask = mask.to(DEV)
        for h in range(nkv):
            keys = st["k_cache"][b, h, :L].double()
            vals = st["v_cache"][b, h].double().transpose(1, 2).reshape(cap, D)[:L]
            for g in range(G):
                qh = q[:, h * G + g]
                s = torch.cat([qh @ keys.t(), qh @ k[:, h].t() + mask], 1) / math.sqrt(D)
                out[b, nodes, h * G + g] = torch.softmax(s, 1) @ torch.cat([vals, v[:, h]], 0)
    return out.view(-1, nq * D), kn, vn


def _exact_accept(case, st):
    T, cap = case["t"], st["cap"]
    hist, lens, acc, paths, emits = st["hist"].tolist(), [], [], [], []
    for b, (par, ids, pick, L) in enumerate(zip(st["parents"].tolist(), st["ids"].tolist(), st["out_tok"].tolist(),
                                                st["lens"].tolist())):
        path = []
        if L < st["stop"]:
            path = [0]
            while True:
                kids = [t for t in range(path[-1] + 1, T) if par[t] == path[-1] and ids[t] == pick[path[-1]]]
                if not kids:
                    break
                path.append(kids[0])
        for i, t in enumerate(path):
            if L + 1 + i < cap:
                hist[b][L + 1 + i] = pick[t]
        lens.append(L + len(path))
        acc.append(max(len(path) - 1, 0))
        paths.append(path + [-1] * (T - len(path)))
        emits.append([pick[t] for t in path] + [-1] * (T - len(path)))
    return _i64(hist), _i32(lens), _i32(acc), _i32(paths), _i64(emits)


def _exact_commit(case, st):
    k, v = st["k_cache"].double(), st["v_cache"].double()
    for b, (path, a, L) in enumerate(zip(st["path"].tolist(), st["naccept"].tolist(), st["lens"].tolist())):
        for i in range(a + 1):
            slot = L - a - 1 + i
            k[:, b, :, slot] = st["k_nodes"][:, b, :, path[i]].double()
            v[:, b, :, slot // 8, :, slot % 8] = st["v_nodes"][:, b, :, path[i]].double()
    return k, v


_EXACT = {"draft": _exact_draft, "attn": _exact_attn, "accept": _exact_accept, "commit": _exact_commit}


def exact(case, seed):
    return _EXACT[case["kind"]](case, _inputs(case, seed))
