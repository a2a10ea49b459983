"""Operators of a serving program around a block's projections: the norm with the residual's addition, products of 8-bit rows with 8-bit weights, and
low-rank adapters of many requests beside a shared projection.

A case is a dict of plain values.  `kind` names the call:

  norm   h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, row by row: the updated residual and the norm's rows
  int8   rows brought to 8 bits (behind such a norm, or as they are), then multiplied with 8-bit weights
  lora   a shared projection with the low-rank adapter of each row's request added

An 8-bit row is d whole numbers of [-127, 127] and one float32 scale, the largest magnitude of the row divided by 127; 8-bit weights have a scale an
output.  An adapter is A [rank][k] and B [n][rank], bf16, in one of the slots of a pool, and a factor; a request may have none."""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-5
TINY = 1e-36      # rows with no value above this are zeros in 8 bits
_DEV = []


def listed():
    return [
        # one token's row between two layers: the smallest call
        dict(name="norm_1x4096", kind="norm", M=1, d=4096, residual=True, f32=False),
        # query and key heads normalised by themselves, a prompt chunk of odd length
        dict(name="norm_heads_20440x128", kind="norm", M=511 * 40, d=128, residual=False, f32=False),
        # a batch's rows, float32 residual stream of a wide model
        dict(name="norm_60x16384_f32", kind="norm", M=60, d=16384, residual=True, f32=True),
        # prompts of new requests
        dict(name="norm_8192x8192", kind="norm", M=8192, d=8192, residual=True, f32=False),
        # one token through a norm and a projection
        dict(name="int8_1x4096x4096", kind="int8", M=1, K=4096, N=4096, norm=True, f32=False),
        # a batch's tokens through the wide projection of a feed-forward layer
        dict(name="int8_64x4096x16384", kind="int8", M=64, K=4096, N=16384, norm=True, f32=False),
        # attention's output of a verify step, quantised as it is, float32 result
        dict(name="int8_300x8192x4096_f32", kind="int8", M=300, K=8192, N=4096, norm=False, f32=True),
        # prompts: the largest call
        dict(name="int8_8192x4096x16384", kind="int8", M=8192, K=4096, N=16384, norm=True, f32=False),
        # one token of a request with an adapter
        dict(name="lora_1x4096x4096_r16", kind="lora", B=1, S=1, K=4096, N=4096, rank=16, slots=8, ragged=False, f32=True),
        # a step of many requests over many adapters, some with none; query, key and value projection in one
        dict(name="lora_64x4096x6144_r16", kind="lora", B=64, S=1, K=4096, N=6144, rank=16, slots=48, ragged=False, f32=True),
        # prompts of a few requests, uneven
        dict(name="lora_6x700x4096x4096_r64", kind="lora", B=6, S=700, K=4096, N=4096, rank=64, slots=8, ragged=True, f32=False),
        # long prompts, small adapters
        dict(name="lora_4x2048x4096x4096_r8", kind="lora", B=4, S=2048, K=4096, N=4096, rank=8, slots=4, ragged=False, f32=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _draw(rng):
    kind = rng.choice(["norm", "int8", "int8", "lora", "lora"])
    if kind == "norm":
        return dict(kind=kind, M=_log(rng, 1, 32768), d=8 * _log(rng, 8, 2048), residual=rng.random() < 0.7, f32=rng.random() < 0.4)
    K, N = 16 * _log(rng, 16, 1024), 8 * _log(rng, 32, 2048)
    if kind == "int8":
        norm = rng.random() < 0.6
        return dict(kind=kind, M=_log(rng, 1, 8192), K=K, N=N, norm=norm, f32=not norm and rng.random() < 0.5)
    S = rng.choice([1, 1, 1, 2, 5, _log(rng, 6, 2048)])
    return dict(kind=kind, B=_log(rng, 1, 128 if S < 6 else 8), S=S, K=K, N=N, rank=rng.choice([8, 16, 16, 32, 64, 128]), slots=_log(rng, 1, 64),
                ragged=rng.random() < 0.5, f32=rng.random() < 0.5)


def draw(rng):
    """One more case of the ranges above, with no more bytes and no more operations than the largest listed ones."""
    most = {w: max(work(c)[w] for c in listed()) for w in ("bytes", "flops")}
    while True:
        c = _draw(rng)
        if all(v <= most[w] for w, v in work(c).items()):
            return c


# --- sizes -----------------------------------------------------------------------------------------------------------------

def _requests(case):
    """(rows, adapter) of every request: S rows each, or (ragged) uniform down to one; adapters at random, an eighth of the requests with none.  The same for
    every seed."""
    r = random.Random(11)
    rows = [r.randint(1, case["S"]) if case["ragged"] else case["S"] for _ in range(case["B"])]
    adapter = [r.randrange(case["slots"]) if i == 0 or r.random() >= 0.125 else -1 for i in range(case["B"])]
    return np.asarray(rows, np.int32), np.asarray(adapter, np.int32)


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, e = case["M"] * case["d"], 4 if case["f32"] else 2
        return dict(bytes=float(n * e * (4 if case["residual"] else 2) + 2 * case["d"]), flops=float(n * 5))
    K, N = case["K"], case["N"]
    if kind == "int8":
        M = case["M"]
        rows = M * K * (6 if case["norm"] else 2)       # bf16 rows, and the residual's way in and out
        return dict(bytes=float(rows + N * K + 4 * N + M * N * (4 if case["f32"] else 2)), flops=float(2 * M * N * K))
    rows, adapter = _requests(case)
    M, R, used = int(rows.sum()), case["rank"], len(set(adapter[adapter >= 0].tolist()))
    with_one = int(rows[adapter >= 0].sum())
    return dict(bytes=float(M * K * (4 if case["f32"] else 2) + 2 * K * N + 2 * used * R * (K + N) + 2 * M * N),
                flops=float(2 * M * K * N + 2 * with_one * R * (K + N)))


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


def _rows(g, n, d, dtype):
    """Activations: tokens of different size, a few features far larger than the others."""
    x = torch.randn((n, d), generator=g, device="cuda", dtype=dtype)
    x.mul_(torch.exp2(torch.randn((n, 1), generator=g, device="cuda")).to(dtype))
    x[:, 7::61] *= 6
    return x


def _inputs(case, seed):
    """What both sides, and the definition, start from."""
    g = torch.Generator("cuda").manual_seed(seed)
    kind, s = case["kind"], {}
    bf16 = torch.bfloat16
    if kind == "norm":
        dt = torch.float32 if case["f32"] else bf16
        s["x"] = _rows(g, case["M"], case["d"], dt)
        s["residual"] = _rows(g, case["M"], case["d"], dt) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(case["d"], generator=g, device="cuda")).to(bf16)
        return s
    K, N = case["K"], case["N"]
    s["w"] = torch.randn((K, N), generator=g, device="cuda", dtype=bf16).mul_(K ** -0.5)
    if kind == "int8":
        s["w"].mul_(torch.exp2(torch.randn(N, generator=g, device="cuda")).to(bf16))      # outputs of different size
        s["x"] = _rows(g, case["M"], K, bf16)
        s["residual"] = _rows(g, case["M"], K, bf16) if case["norm"] else None
        s["weight"] = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(bf16)
        return s
    s["rows"], s["adapter"] = _requests(case)
    s["x"] = _rows(g, int(s["rows"].sum()), K, torch.float32 if case["f32"] else bf16)
    s["a"] = torch.randn((case["slots"], case["rank"], K), generator=g, device="cuda", dtype=bf16).mul_(K ** -0.5)
    s["b"] = torch.randn((case["slots"], N, case["rank"]), generator=g, device="cuda", dtype=bf16).mul_(case["rank"] ** -0.5)
    s["factor"] = 0.5 + torch.rand(case["slots"], generator=g, device="cuda")
    return s


def prepare(case, seed):
    st, x, kind = _State(case), _inputs(case, seed), case["kind"]
    st.x, bf16 = x, torch.bfloat16
    if kind == "norm":
        st.h = torch.empty_like(x["x"]) if case["residual"] else None
        st.out = torch.empty_like(x["x"])
    else:
        M, K, N = x["x"].shape[0], case["K"], case["N"]
        st.out = torch.empty((M, N), device="cuda", dtype=torch.float32 if kind == "int8" and case["f32"] else bf16)
    if kind == "int8":
        st.h = torch.empty_like(x["x"]) if case["norm"] else None
        st.codes, st.scales = torch.empty((M, K), device="cuda", dtype=torch.int8), torch.empty(M, device="cuda")
        st.w, st.w_scales = torch.empty((N, K), device="cuda", dtype=torch.int8), torch.empty(N, device="cuda")
    if own:
        import relux_b200 as rb
        from relux_b200 import lib as L
        if not _DEV:
            _DEV.append(rb.Device(torch.cuda.current_device()))
        st.L = L
        st.pool = rb.Pool(_DEV[0], L.POOL_GQA, 1, 1, num_kv_heads=1, head_dim=128)
        if kind == "int8":
            torch.cuda.synchronize()
            st.pool.int8_weights(K, N, x["w"].data_ptr(), st.w.data_ptr(), st.w_scales.data_ptr(), dtype=L.DTYPE_BF16)
            st.pool.dev.sync()
    elif kind == "int8":
        st.w, st.w_scales = _quantise(x["w"].t().float())
    elif kind == "lora":
        # [rows][slots]: the factor of the row's adapter, at its slot
        at = torch.from_numpy(np.repeat(x["adapter"], x["rows"]).astype(np.int64)).cuda()
        st.pick = torch.where(at[:, None] == torch.arange(case["slots"], device="cuda"), x["factor"], 0.0)
    torch.cuda.synchronize()
    return st


# --- the plain forms -------------------------------------------------------------------------------------------------------

def _quantise(x):
    """int8 rows of float32 ones, and their scales.  (Quotients of two tensors: with a number on one side they are a reciprocal and a product.)"""
    top = x.abs().amax(-1)
    some, most = top >= TINY, torch.full_like(top, 127)
    codes = torch.round(x * torch.where(some, most / top, 0.0)[:, None]).clamp(-127, 127).to(torch.int8)
    return codes, torch.where(some, top / most, 0.0)


def _norm(x, residual, weight):
    h = x.float() if residual is None else x.float() + residual.float()
    return h, h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * weight.float()


def run(st):
    c, x, kind = st.case, st.x, st.case["kind"]
    if own:
        L, pool = st.L, st.pool
        act = L.DTYPE_F32 if x["x"].dtype == torch.float32 else L.DTYPE_BF16
        if kind == "norm":
            pool.rmsnorm(c["M"], c["d"], x["x"].data_ptr(), x["weight"].data_ptr(), EPS, out=st.out.data_ptr(), dtype=act,
                         residual=x["residual"].data_ptr() if c["residual"] else None, residual_out=st.h.data_ptr() if c["residual"] else None)
            return {"y": st.out, "h": st.h} if c["residual"] else {"y": st.out}
        if kind == "int8":
            M, K, N = c["M"], c["K"], c["N"]
            if c["norm"]:
                pool.rmsnorm(M, K, x["x"].data_ptr(), x["weight"].data_ptr(), EPS, codes=st.codes.data_ptr(), scales=st.scales.data_ptr(), dtype=act,
                             residual=x["residual"].data_ptr(), residual_out=st.h.data_ptr())
            else:
                pool.int8_rows(M, K, x["x"].data_ptr(), st.codes.data_ptr(), st.scales.data_ptr(), dtype=act)
            pool.matmul_int8(M, K, N, st.codes.data_ptr(), st.scales.data_ptr(), st.w.data_ptr(), st.w_scales.data_ptr(), st.out.data_ptr(),
                             out_dtype=L.DTYPE_F32 if c["f32"] else L.DTYPE_BF16)
            return {"c": st.out, "h": st.h} if c["norm"] else {"c": st.out}
        pool.matmul_lora(x["x"].shape[0], c["K"], c["N"], x["x"].data_ptr(), x["w"].data_ptr(), st.out.data_ptr(), x["a"].data_ptr(), x["b"].data_ptr(),
                         c["rank"], c["slots"], x["adapter"], rows=x["rows"], factors=x["factor"].data_ptr(), x_dtype=act, out_dtype=L.DTYPE_BF16)
        return st.out
    if kind == "norm":
        h, y = _norm(x["x"], x["residual"], x["weight"])
        st.out.copy_(y)
        if not c["residual"]:
            return {"y": st.out}
        st.h.copy_(h)
        return {"y": st.out, "h": st.h}
    if kind == "int8":
        y = x["x"].float()
        if c["norm"]:
            h, y = _norm(x["x"], x["residual"], x["weight"])
            st.h.copy_(h)
        codes, scales = _quantise(y)
        st.out.copy_(torch.matmul(codes.float(), st.w.float().t()) * scales[:, None] * st.w_scales)
        return {"c": st.out, "h": st.h} if c["norm"] else {"c": st.out}
    f = x["x"].float()
    slots, rank, K = x["a"].shape
    t = torch.matmul(f, x["a"].float().reshape(slots * rank, K).t()).reshape(-1, slots, rank) * st.pick[:, :, None]
    low = torch.matmul(t.reshape(-1, slots * rank), x["b"].float().permute(0, 2, 1).reshape(slots * rank, -1))
    st.out.copy_(torch.matmul(f, x["w"].float()).add_(low))
    return st.out


# --- the definition, in 64 bits --------------------------------------------------------------------------------------------

def exact(case, seed):
    """Row by row and request by request."""
    x, kind, f64 = _inputs(case, seed), case["kind"], torch.float64

    def normed():
        h = x["x"].to(f64)
        if x["residual"] is not None:
            h = h + x["residual"].to(f64)
        return h, h / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[-1] + EPS) * x["weight"].to(f64)

    def eight(y):      # the numbers of a row are defined by float32 operations: the factor 127 / a, and the product with it
        y = y.to(torch.float32)
        a = y.abs().max(dim=-1, keepdim=True).values
        a = torch.where(a < TINY, 0, a)
        up = (torch.full_like(a, 127, dtype=f64) / a.to(f64)).to(torch.float32)
        return torch.where(a > 0, (y * up).to(f64).round(), 0), (a.to(f64) / torch.full_like(a, 127, dtype=f64)).to(torch.float32).to(f64)

    if kind == "norm":
        h, y = normed()
        return {"y": y, "h": h} if case["residual"] else {"y": y}
    if kind == "int8":
        h, y = normed() if case["norm"] else (None, x["x"].to(f64))
        (a, sa), (w, sw) = eight(y), eight(x["w"].to(f64).t().contiguous())
        c = (a @ w.t()) * sa * sw.t()
        return {"c": c, "h": h} if case["norm"] else {"c": c}
    out, at = x["x"].to(f64) @ x["w"].to(f64), 0
    for n, s in zip(x["rows"].tolist(), x["adapter"].tolist()):
        if s >= 0:
            t = x["x"][at:at + n].to(f64) @ x["a"][s].to(f64).t()
            out[at:at + n] += float(x["factor"][s]) * (t @ x["b"][s].to(f64).t())
        at += n
    return out
