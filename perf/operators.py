"""Operators of a serving program around the grouped-query cache: an 8-bit cache (quantised as it is written, read back, attended over), and drafted
trees (attention of a tree of tokens over a cache, and the commit of its accepted path).

A case is a dict of plain values.  `kind` names the call:

  write    new rows of a batch quantised into the 8-bit cache, and read back from it
  read     whole cached contexts read back into dense device memory
  attend   new rows written past the cursor of the 8-bit cache, then causal attention of their queries: a decode step (S = 1), the verify of a
           chain of drafted tokens, or a prompt's next chunk
  tree     the same for a tree of drafted tokens, over a bf16 or an 8-bit cache
  commit   the rows of the accepted path of a tree moved up behind the cursor, on every layer, and read back

Sequences lie in pages of 64 tokens behind a page table.  An 8-bit row is, per kv head, 128 whole numbers of [-127, 127] and one float32 scale: the
largest magnitude of the row divided by 127."""
import math
import random

import numpy as np
import torch

own = False

PAGE, D = 64, 128
TINY = 1e-36      # rows with no value above this are stored as zeros
_DEV = []


def listed():
    return [
        # one decode step's rows of a batch of uneven sequences
        dict(name="write_b32_s1_ctx3k", kind="write", B=32, S=1, ctx=3001, H=32, Hkv=8, ragged=True, f32=False),
        # prompts of new requests, float32 activations
        dict(name="write_b8_s2048", kind="write", B=8, S=2048, ctx=0, H=32, Hkv=8, ragged=False, f32=True),
        # contexts that leave the cache (to another worker, or to a kernel that takes bf16)
        dict(name="read_b4_ctx8k", kind="read", B=4, ctx=8192, H=32, Hkv=8, ragged=True),
        # one user, one token: the smallest attention call
        dict(name="attend_b1_s1_ctx700", kind="attend", B=1, S=1, ctx=700, H=32, Hkv=8, ragged=False),
        # verify of four drafted tokens at full batch
        dict(name="attend_b128_s4_ctx8k", kind="attend", B=128, S=4, ctx=8192, H=32, Hkv=8, ragged=False),
        # the next chunk of a prompt behind cached tokens
        dict(name="attend_b4_s500_ctx1500", kind="attend", B=4, S=500, ctx=1500, H=32, Hkv=8, ragged=False),
        # a small tree for one user
        dict(name="tree_bf16_b1_s8_ctx2k", kind="tree", int8=False, B=1, S=8, ctx=2000, H=32, Hkv=8, ragged=False),
        # the usual tree of a few dozen nodes, a batch of uneven sequences
        dict(name="tree_bf16_b16_s60_ctx4k", kind="tree", int8=False, B=16, S=60, ctx=4096, H=32, Hkv=8, ragged=True),
        # small trees at a large batch over the 8-bit cache
        dict(name="tree_int8_b64_s16_ctx8k", kind="tree", int8=True, B=64, S=16, ctx=8192, H=32, Hkv=8, ragged=False),
        # large trees of a model with more query heads, long contexts
        dict(name="tree_int8_b8_s64_ctx32k", kind="tree", int8=True, B=8, S=64, ctx=32768, H=64, Hkv=8, ragged=False),
        # one user's accepted path, a small model's layers
        dict(name="commit_bf16_b1_l4", kind="commit", int8=False, B=1, S=26, ctx=1000, H=32, Hkv=8, layers=4, ragged=False),
        # a batch's accepted paths on all layers of a model
        dict(name="commit_int8_b64_l32", kind="commit", int8=True, B=64, S=60, ctx=300, H=32, Hkv=8, layers=32, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "tree", "tree", "tree", "commit"])
    H, Hkv = rng.choice([(32, 8), (32, 8), (16, 8), (64, 8), (32, 4), (8, 8)])
    ragged = rng.random() < 0.5
    if kind == "write":
        return dict(kind=kind, B=_log(rng, 1, 64), S=_log(rng, 1, 2048), ctx=rng.choice([0, _log(rng, 1, 4000)]), H=H, Hkv=Hkv, ragged=ragged,
                    f32=rng.random() < 0.5)
    if kind == "read":
        return dict(kind=kind, B=_log(rng, 1, 32), ctx=_log(rng, 1, 16384), H=H, Hkv=Hkv, ragged=ragged)
    if kind == "attend":
        S = rng.choice([1, 1, 2, 3, 4, 5, _log(rng, 6, 1000)])
        return dict(kind=kind, B=_log(rng, 1, 128 if S < 6 else 8), S=S, ctx=_log(rng, 1, 16384 if S < 6 else 4000), H=H, Hkv=Hkv, ragged=ragged)
    if kind == "tree":
        return dict(kind=kind, int8=rng.random() < 0.5, B=_log(rng, 1, 64), S=_log(rng, 2, 64), ctx=_log(rng, 1, 32768), H=H, Hkv=Hkv, ragged=ragged)
    return dict(kind=kind, int8=rng.random() < 0.5, B=_log(rng, 1, 64), S=_log(rng, 8, 64), ctx=_log(rng, 100, 1000), H=H, Hkv=Hkv,
                layers=_log(rng, 1, 32), ragged=ragged)


def draw(rng):
    """One more case of the ranges above, with no more bytes and no more operations than the largest listed ones."""
    most = {w: max(work(c)[w] for c in listed()) for w in ("bytes", "flops")}
    while True:
        c = _draw(rng)
        if all(v <= most[w] for w, v in work(c).items()):
            return c


# --- sizes -----------------------------------------------------------------------------------------------------------------

def _lens(case):
    """Cached tokens of the sequences: `ctx` each, or (ragged) uniform down to 1/32 of it, the same for every seed."""
    B, ctx = case["B"], case["ctx"]
    if not case.get("ragged"):
        return np.full(B, ctx, np.int32)
    r = random.Random(11)
    return np.asarray([r.randint(max(min(1, ctx), ctx // 32), ctx) for _ in range(B)], np.int32)


def _tree(case, seed):
    """(parents [B][S], nodes [B]): node i continues node parents[i] < i, or (-1) the cached tokens.  The first few continue the cached tokens, as
    the best first tokens of a draft do, the others a random earlier one.  A ragged batch's trees have half as many nodes and up (numbers of nodes, and lengths of paths, are the same for every seed)."""
    B, S, r = case["B"], case["S"], np.random.default_rng(seed)
    nodes = np.random.default_rng(11).integers((S + 1) // 2, S + 1, B).astype(np.int32) if case["ragged"] else np.full(B, S, np.int32)
    roots = max(1, min(10, S // 3))
    parents = np.full((B, S), -1, np.int32)
    for i in range(roots, S):
        parents[:, i] = r.integers(0, i, B)
    return parents, nodes


def _paths(case, seed):
    """(path [B][8], length [B]): an accepted path of each sequence's tree, up to seven nodes, each node past the places that the path moves to."""
    B, S, r = case["B"], case["S"], np.random.default_rng(seed + 1)
    top = max(1, min(7, S // 2))
    n = np.random.default_rng(11).integers(0, top + 1, B).astype(np.int32)
    n[0] = max(1, n[0])
    path = np.zeros((B, 8), np.int32)
    for b in range(B):
        path[b, :n[b]] = np.sort(r.choice(np.arange(top, S), n[b], replace=False))
    return path, n


def _row_bytes(case):
    return case["Hkv"] * (2 * D + 8 if case.get("int8", True) else 4 * D)


def work(case):
    kind, B, H, Hkv, lens = case["kind"], case["B"], case["H"], case["Hkv"], _lens(case).astype(np.float64)
    row, dense = _row_bytes(case), Hkv * D * 4       # a cached token, and the same in dense bf16
    if kind == "write":
        n = B * case["S"]
        return dict(bytes=float(n * (dense * (2 if case["f32"] else 1) + row + dense)), flops=float(n * Hkv * D * 4))
    if kind == "read":
        n = lens.sum()
        return dict(bytes=float(n * (row + dense)), flops=float(n * Hkv * D * 2))
    if kind == "commit":
        n = _paths(case, 1)[1].sum() * case["layers"]
        return dict(bytes=float(max(1, n) * (2 * row + dense)), flops=float(max(1, n) * Hkv * D * 2))
    S = case["S"]
    new = float(_tree(case, 1)[1].sum()) if kind == "tree" else float(B * S)
    seen = S * lens.sum() + (B * S * (S + 1) / 2.0 if kind == "attend" else 4.0 * new)   # a tree's node has a few ancestors
    return dict(bytes=float(lens.sum() * row + new * (dense + row) + 4.0 * B * S * H * D), flops=float(4 * D * H * seen))


# --- inputs ----------------------------------------------------------------------------------------------------------------

class _State:
    def __init__(self, case):
        self.case, self.pool = case, None

    def __del__(self):
        if self.pool is not None:
            try:
                self.pool.dev.sync()
                self.pool.destroy()
            except Exception:
                pass


def _rows(seed, what, n, Hkv, dtype=torch.bfloat16):
    """Keys or values of n tokens: heads of different size, a few dims far larger than the others in keys, tokens of different size."""
    g = torch.Generator("cuda").manual_seed(seed * 8 + what)
    x = torch.randn((n, Hkv, D), generator=g, device="cuda", dtype=dtype)
    x.mul_(torch.exp2(torch.randn((n, Hkv, 1), generator=g, device="cuda")).to(dtype))
    if what % 2 == 0:
        x[..., 5::32] *= 4
    return x


def _inputs(case, seed):
    """What both sides, and the definition, start from: cached rows per layer, new rows, queries, lengths, the tree or the path."""
    kind, B, H, Hkv, S = case["kind"], case["B"], case["H"], case["Hkv"], case.get("S", 0)
    s = dict(lens=_lens(case), layers=case.get("layers", 1))
    s["n_new"] = np.full(B, S, np.int32)
    s["parents"] = None
    if kind == "tree":
        s["parents"], s["n_new"] = _tree(case, seed)
    if kind == "commit":
        s["path"], s["path_len"] = _paths(case, seed)
    per = (int(s["lens"].max()) + S + PAGE - 1) // PAGE
    s["table"] = np.random.default_rng(seed).permutation(B * per).astype(np.int32).reshape(B, per)
    # the cached rows that the call finds: the drafted rows too, where it commits them
    s["have"] = s["lens"] + (s["n_new"] if kind == "commit" else 0)
    total = int(s["have"].sum())
    s["k"] = [_rows(seed + 100 * l, 0, total, Hkv) for l in range(s["layers"])]
    s["v"] = [_rows(seed + 100 * l, 1, total, Hkv) for l in range(s["layers"])]
    if kind in ("write", "attend", "tree"):
        dt = torch.float32 if case.get("f32") else torch.bfloat16
        n = int(s["n_new"].sum())
        s["nk"], s["nv"] = _rows(seed, 2, n, Hkv, dt), _rows(seed, 3, n, Hkv, dt)
    if kind in ("attend", "tree"):
        g = torch.Generator("cuda").manual_seed(seed * 8 + 4)
        s["q"] = torch.randn((B, S, H, D), generator=g, device="cuda", dtype=torch.bfloat16)
    return s


def _spread(n, at0, table):
    """(sequence, page, slot) of rows at0[b] .. at0[b] + n[b] - 1 of every sequence, in order."""
    b = np.repeat(np.arange(len(n)), n)
    t = np.repeat(at0, n) + np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n)
    return torch.from_numpy(b).cuda(), torch.from_numpy(table[b, t // PAGE].astype(np.int64)).cuda(), torch.from_numpy(t % PAGE).cuda()


def prepare(case, seed):
    st, x, B, Hkv = _State(case), _inputs(case, seed), case["B"], case["Hkv"]
    int8 = case.get("int8", True)
    st.x = x
    st.zero = np.zeros(B, np.int32)
    if "q" in x:
        st.out = torch.empty_like(x["q"])
    back = {"write": x["n_new"], "read": x["lens"], "commit": x.get("path_len")}.get(case["kind"])
    if back is not None:
        st.back = back
        st.rk, st.rv = (torch.empty((x["layers"], int(back.sum()), Hkv, D), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    if own:
        import relux_b200 as rb
        from relux_b200 import lib as L
        if not _DEV:
            _DEV.append(rb.Device(torch.cuda.current_device()))
        pages = x["table"].size
        st.L = L
        st.pool = rb.Pool(_DEV[0], L.POOL_GQA, x["layers"], pages, PAGE, B, x["table"].shape[1], num_kv_heads=Hkv, head_dim=D, cache_int8=int8)
        st.pool.set_tables(x["table"])
        torch.cuda.synchronize()
        for l in range(x["layers"]):
            if x["have"].sum():
                st.pool.append(l, x["k"][l].data_ptr(), x["v"][l].data_ptr(), B, n_new=x["have"], dtype=L.DTYPE_BF16)
        st.pool.set_len(-1, x["lens"])
        st.pool.dev.sync()
    else:
        shape = (x["layers"], x["table"].size, Hkv, PAGE)
        st.cache = [torch.zeros(shape + (D,), device="cuda", dtype=torch.int8 if int8 else torch.bfloat16) for _ in range(2)]
        st.scale = [torch.zeros(shape, device="cuda") for _ in range(2)] if int8 else [None, None]
        _, page, slot = _spread(x["have"], st.zero, x["table"])
        for l in range(x["layers"]):
            _put(st, l, page, slot, x["k"][l], x["v"][l])
        st.at_new = _spread(x["n_new"], x["lens"], x["table"])
        st.tab = torch.from_numpy(x["table"].astype(np.int64)).cuda()
        if case["kind"] == "commit":
            b = np.repeat(np.arange(B), x["path_len"])
            j = np.arange(int(x["path_len"].sum())) - np.repeat(np.cumsum(x["path_len"]) - x["path_len"], x["path_len"])
            t = x["lens"][b] + x["path"][b, j]
            st.src = tuple(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (x["table"][b, t // PAGE].astype(np.int64), t % PAGE))
        if back is not None:
            st.at_back = _spread(back, st.zero if case["kind"] == "read" else x["lens"], x["table"])
        if "q" in x:
            st.mask = torch.from_numpy(_visible(case, x)).cuda()
    # inputs that the pool, or the pages, hold now
    x["k"] = x["v"] = None
    torch.cuda.synchronize()
    return st


def _visible(case, x):
    """[B][S][S]: does new token i see new token j?"""
    B, S = case["B"], case["S"]
    if x["parents"] is None:
        return np.broadcast_to(np.tril(np.ones((S, S), bool)), (B, S, S)).copy()
    see, at = np.zeros((B, S, S), bool), np.arange(B)
    for i in range(S):
        up = x["parents"][:, i]
        see[:, i] = np.where((up >= 0)[:, None], see[at, np.maximum(up, 0)], False)
        see[:, i, i] = True
    there = np.arange(S)[None, :] < x["n_new"][:, None]
    return see & there[:, :, None] & there[:, None, :]


# --- the plain forms -------------------------------------------------------------------------------------------------------

def _quantise(x):
    """int8 rows and their scales."""
    x = x.float()
    top = x.abs().amax(-1)
    some = top >= TINY
    codes = torch.round(x * torch.where(some, 127.0 / top, 0.0)[..., None]).clamp(-127, 127).to(torch.int8)
    return codes, torch.where(some, top / 127.0, 0.0)


def _put(st, l, page, slot, k, v):
    for i, x in enumerate((k, v)):
        if st.scale[i] is None:
            st.cache[i][l][page, :, slot] = x.to(torch.bfloat16)
        else:
            st.cache[i][l][page, :, slot], st.scale[i][l][page, :, slot] = _quantise(x)


def _back(st):
    _, page, slot = st.at_back
    every = slice(None)
    for i, out in enumerate((st.rk, st.rv)):
        c = st.cache[i][every, page, :, slot].float()        # [rows][layers][Hkv][D]
        if st.scale[i] is not None:
            c = c * st.scale[i][every, page, :, slot][..., None]
        out.copy_(c.transpose(0, 1))
    return {"k": st.rk, "v": st.rv}


def _attend(st):
    c, x = st.case, st.x
    B, S, H, Hkv = c["B"], c["S"], c["H"], c["Hkv"]
    dense = []
    for i in range(2):      # [B][Hkv][T][D] in float32
        y = st.cache[i][0][st.tab].float()
        if st.scale[i] is not None:
            y = y * st.scale[i][0][st.tab][..., None]
        dense.append(y.permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D))
    T = dense[0].shape[2]
    lens = torch.from_numpy(x["lens"].astype(np.int64)).cuda()
    t = torch.arange(T, device="cuda")
    node = (t[None, :] - lens[:, None])                     # [B][T]: which new token a row is
    new = torch.gather(st.mask, 2, node.clamp(0, S - 1)[:, None, :].expand(B, S, T)) & (node < S)[:, None, :]
    there = torch.from_numpy(np.arange(S)[None, :] < x["n_new"][:, None]).cuda()
    see = torch.where((node < 0)[:, None, :], there[:, :, None], new)     # [B][S][T]
    q = x["q"].float().reshape(B, S, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, (H // Hkv) * S, D)
    s = torch.matmul(q, dense[0].transpose(2, 3)).mul_(D ** -0.5).reshape(B, Hkv, H // Hkv, S, T)
    s.masked_fill_(~see[:, None, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = p.sum(-1).clamp_min(1e-30)
    o = torch.matmul(p.reshape(B, Hkv, -1, T), dense[1]).reshape(B, Hkv, H // Hkv, S, D) / total[..., None]
    st.out.copy_(o.permute(0, 3, 1, 2, 4).reshape(B, S, H, D))
    return st.out


# --- one pass --------------------------------------------------------------------------------------------------------------

def run(st):
    c, x, kind = st.case, st.x, st.case["kind"]
    B, H, S = c["B"], c["H"], c.get("S", 0)
    if own:
        L, pool = st.L, st.pool
        if kind == "write":
            pool.set_len(0, x["lens"])
            pool.append(0, x["nk"].data_ptr(), x["nv"].data_ptr(), B, n_new=x["n_new"], dtype=L.DTYPE_F32 if c["f32"] else L.DTYPE_BF16)
        elif kind == "attend":
            pool.verify(0, B, x["q"].data_ptr(), st.out.data_ptr(), x["nk"].data_ptr(), x["nv"].data_ptr(), H, D, D ** -0.5, S,
                        q_dtype=L.DTYPE_BF16, out_dtype=L.DTYPE_BF16, kv_dtype=L.DTYPE_BF16)
            return st.out
        elif kind == "tree":
            pool.tree_verify(0, B, x["q"].data_ptr(), st.out.data_ptr(), x["nk"].data_ptr(), x["nv"].data_ptr(), H, D, D ** -0.5, x["parents"],
                             n_nodes=x["n_new"], q_dtype=L.DTYPE_BF16, out_dtype=L.DTYPE_BF16, kv_dtype=L.DTYPE_BF16)
            return st.out
        elif kind == "commit":
            pool.set_len(-1, x["lens"])
            pool.tree_commit(-1, x["path"], x["path_len"])
        pool.read_kv(-1, B, st.rk.data_ptr(), st.rv.data_ptr(), st.zero if kind == "read" else x["lens"], st.back, dtype=L.DTYPE_BF16)
        return {"k": st.rk, "v": st.rv}
    if kind in ("write", "attend", "tree"):
        _put(st, 0, st.at_new[1], st.at_new[2], x["nk"], x["nv"])
    if kind in ("attend", "tree"):
        return _attend(st)
    if kind == "commit":
        _, page, slot = st.at_back
        every = slice(None)
        for y in st.cache + [z for z in st.scale if z is not None]:
            y[every, page, :, slot] = y[every, st.src[0], :, st.src[1]]
    return _back(st)


# --- the definition, in 64 bits --------------------------------------------------------------------------------------------

def exact(case, seed):
    """Sequence by sequence from the cached rows themselves: no pages, no table."""
    x, int8, kind, Hkv = _inputs(case, seed), case.get("int8", True), case["kind"], case["Hkv"]

    def held(rows):          # what the cache holds of these rows
        r = rows.to(torch.float64)
        if not int8:
            return r.to(torch.bfloat16).to(torch.float64)
        step = r.abs().max(dim=-1, keepdim=True).values / 127
        return torch.where(step > 0, torch.round(r / torch.where(step > 0, step, 1)) * step, 0)

    if kind in ("write", "read", "commit"):
        if kind == "write":
            return {"k": held(x["nk"])[None], "v": held(x["nv"])[None]}
        if kind == "read":
            return {"k": held(x["k"][0])[None], "v": held(x["v"][0])[None]}
        first = np.cumsum(x["have"]) - x["have"] + x["lens"]
        pick = torch.tensor([int(first[b] + x["path"][b, j]) for b in range(case["B"]) for j in range(x["path_len"][b])], device="cuda", dtype=torch.int64)
        return {n: torch.stack([held(layer[pick]) for layer in x[n]]) for n in ("k", "v")}
    S, H = case["S"], case["H"]
    g, out = H // Hkv, torch.zeros((case["B"], S, H, D), device="cuda", dtype=torch.float64)
    at = at_new = 0
    for b in range(case["B"]):
        n, m = int(x["lens"][b]), int(x["n_new"][b])
        K, V = (torch.cat([held(x[o][0][at:at + n]), held(x[w][at_new:at_new + m])]) for o, w in (("k", "nk"), ("v", "nv")))
        at, at_new = at + n, at_new + m
        see = torch.zeros((m, n + m), dtype=torch.bool)
        see[:, :n] = True
        for i in range(m):
            j = i
            while j >= 0:
                see[i, n + j] = True
                j = int(x["parents"][b, j]) if x["parents"] is not None else j - 1
        see = see.cuda()
        for h in range(Hkv):
            q = x["q"][b, :m, h * g:(h + 1) * g].to(torch.float64).transpose(0, 1)          # [g][m][D]
            s = (q @ K[:, h].T / math.sqrt(D)).masked_fill(~see, -math.inf)
            out[b, :m, h * g:(h + 1) * g] = (torch.softmax(s, dim=-1) @ V[:, h]).transpose(0, 1)
    return out
