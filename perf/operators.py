"""The operators of scenes in codes (splats that name rows of a learned codebook), each as a user's program calls it.

A case is a plain dict:

  op       "lookup"    lookup_codes: attributes of splats from their codes
           "probs"     code_log_probs: log probabilities of codes, entropy, best codes
           "balance"   code_balance: counts per code and the balance loss
  train    forward and backward (every gradient comes back), or the forward under no_grad
  B, G     images (0: inputs without a batch axis) and splats per image
  K        codes in the codebook
  D        values per code (lookup)
  dtype    "f32", "bf16" or "f16": of the codebook or the logits
  long     codes of 64 bits instead of 32
  scales   a factor per splat (lookup)
  skew     80% of the splats share eight codes
  top      alternatives asked for (probs)
  T        temperature (probs)
  masked   a tenth of the logits at -inf, and one row in a thousand wholly so
  S        codes per splat (balance)

In every case about one splat in fifty has no code (-1): a splat that was pruned.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _package():
    path = os.path.join(os.getcwd(), "fast-mac-gsplat_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import torch_gsplat_bridge_fast as gs

    return gs


def _lookup(name, train, B, G, K, D, dtype="f32", long=False, scales=True, skew=False):
    return dict(name=name, op="lookup", train=train, B=B, G=G, K=K, D=D, dtype=dtype, long=long, scales=scales, skew=skew)


def _probs(name, train, B, G, K, dtype="f32", top=0, T=1.0, masked=False, long=False):
    return dict(name=name, op="probs", train=train, B=B, G=G, K=K, dtype=dtype, top=top, T=T, masked=masked, long=long)


def _balance(name, train, B, G, K, dtype="f32", S=1, masked=False, skew=False, long=False):
    return dict(name=name, op="balance", train=train, B=B, G=G, K=K, dtype=dtype, S=S, masked=masked, skew=skew, long=long)


def listed():
    return [
        # fitting a small image: colours from a small codebook, thousands of steps; the calls' own cost
        _lookup("lookup_train_512", True, 0, 512, 64, 3),
        # a frame of a stored scene: all eleven attributes of 64K splats from their codes
        _lookup("lookup_eval_64k", False, 0, 65536, 1024, 11, scales=False),
        # four images of splats in a batch, features in 16 bits, most splats sharing a few codes
        _lookup("lookup_train_clustered_b4", True, 4, 65536, 4096, 48, dtype="bf16", long=True, skew=True),
        # a training step of a million splats with wide features
        _lookup("lookup_train_1m", True, 0, 1 << 20, 16384, 128),
        # one splat's choice among a very large codebook (a scene edited splat by splat)
        _probs("probs_one_splat", False, 0, 1, 131072, top=8),
        # a batch of ragged small images, an odd codebook, pruned codes
        _probs("probs_train_ragged_b5", True, 5, 4001, 257, dtype="f16", top=4, T=0.5, masked=True, long=True),
        # assigning a million splats to their best code, with the rate
        _probs("probs_eval_1m", False, 0, 1 << 20, 512, top=1),
        # an ordinary training step: 64K splats
        _probs("probs_train_64k", True, 0, 65536, 1024, dtype="bf16", top=1),
        # the largest: a training step with a large codebook
        _probs("probs_train_64k_16k", True, 0, 65536, 16384, dtype="bf16", top=8, T=0.7),
        # the balance term when fitting a small image
        _balance("balance_train_512", True, 0, 512, 64),
        # four images, each balanced by itself, two codes per splat, most splats on a few codes
        _balance("balance_train_b4", True, 4, 65536, 256, S=2, skew=True),
        # 200K splats and a large codebook with pruned codes
        _balance("balance_train_200k_4k", True, 0, 200003, 4096, dtype="bf16", masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("lookup", "probs", "balance"))
    dtype = rng.choice(("f32", "f32", "bf16", "f16"))
    train = rng.random() < 0.7
    B = rng.choice((0, 0, 1, 2, 5))
    long = rng.random() < 0.3
    if op == "lookup":
        D = rng.choice((1, 3, 4, 11, 48, 64, 128, _log(rng, 1, 1024)))
        rows = max(1, min(_log(rng, 300, 1 << 20), (1 << 26) // D))
        c = _lookup("", train, B, max(1, rows // max(B, 1)), _log(rng, 16, 65536), D, dtype, long, rng.random() < 0.6,
                    rng.random() < 0.3)
        if c["K"] * D > 1 << 24:
            c["K"] = max(16, (1 << 24) // D)
    else:
        K = _log(rng, 8, 131072 if op == "probs" else 16384)
        rows = max(1, min(_log(rng, 1 if op == "probs" else 300, 1 << 20), (1 << 29) // K))
        G = max(1, rows // max(B, 1))
        if op == "probs":
            c = _probs("", train, B, G, K, dtype, min(K, rng.choice((0, 1, 1, 4, 8, 20))), rng.choice((1.0, 1.0, 0.5, 2.0)),
                       rng.random() < 0.4, long)
        else:
            c = _balance("", train, B, G, K, dtype, rng.choice((1, 1, 2, 4)), rng.random() < 0.4, rng.random() < 0.4, long)
    del c["name"]
    return c


def _shape(case):
    return ((case["B"],) if case["B"] else ()) + (case["G"],)


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    shape, K, dtype = _shape(case), case["K"], DTYPES[case["dtype"]]

    def normal(*s):
        return torch.randn(*s, device=dev, generator=gen)

    def codes_of(*s):
        c = torch.randint(0, K, s, device=dev, generator=gen)
        if case.get("skew"):
            few = torch.randint(0, K, (8,), device=dev, generator=gen)
            pick = torch.randint(0, 8, s, device=dev, generator=gen)
            c = torch.where(torch.rand(s, device=dev, generator=gen) < 0.8, few[pick], c)
        c = torch.where(torch.rand(s, device=dev, generator=gen) < 0.02, torch.full_like(c, -1), c)
        return c if case["long"] else c.to(torch.int32)

    s = dict(case=case, op=case["op"], train=case["train"], scales=None)
    if case["op"] == "lookup":
        s["codes"] = codes_of(*shape)
        s["codebook"] = normal(K, case["D"]).to(dtype).requires_grad_(case["train"])
        if case["scales"]:
            s["scales"] = normal(*shape).exp().requires_grad_(case["train"])
        if case["train"]:
            s["grad"] = normal(*shape, case["D"]).to(dtype)
        return s
    x = normal(*shape, K)
    # spread like the distances of splats to codes: a few good ones, a long tail
    x.mul_(3.0)
    if case["masked"]:
        x[torch.rand(*shape, K, device=dev, generator=gen) < 0.1] = -math.inf
        x[torch.rand(shape, device=dev, generator=gen) < 1e-3] = -math.inf
    s["logits"] = x.to(dtype).requires_grad_(case["train"])
    if case["op"] == "probs":
        s.update(codes=codes_of(*shape), top=case["top"], T=case["T"])
        if case["train"]:
            s["g_logp"], s["g_entropy"] = normal(*shape), normal(*shape)
            s["g_top"] = normal(*shape, case["top"]) if case["top"] else None
    else:
        s["codes"] = codes_of(*shape, case["S"]) if case["S"] > 1 else codes_of(*shape)
        if case["train"]:
            s["g_loss"] = 0.5 + torch.rand(shape[:-1], device=dev, generator=gen)
            s["g_mean"] = normal(*shape[:-1], K)
            if dtype is torch.float16:  # a program with 16-bit gradients scales its loss, here by the rows that share it
                s["g_loss"].mul_(case["G"])
                s["g_mean"].mul_(case["G"])
    return s


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    gs = _package()
    train = s["train"]
    with torch.set_grad_enabled(train):
        if s["op"] == "lookup":
            out = gs.lookup_codes(s["codes"], s["codebook"], s["scales"])
            r = {"out": out}
            if train:
                inputs = [s["codebook"]] + ([s["scales"]] if s["scales"] is not None else [])
                r["grads"] = torch.autograd.grad(out, inputs, s["grad"])
            return _detached(r)
        if s["op"] == "probs":
            o = gs.code_log_probs(s["logits"], s["codes"], top=s["top"], temperature=s["T"])
            r = {"logp": o.log_probs, "entropy": o.entropy}
            if s["top"]:
                r.update(top=o.top_log_probs, best=o.top_codes)
            if train:
                outs, gs_ = [o.log_probs, o.entropy], [s["g_logp"], s["g_entropy"]]
                if s["top"]:
                    outs.append(o.top_log_probs)
                    gs_.append(s["g_top"])
                r["grad"] = torch.autograd.grad(outs, s["logits"], gs_)[0]
            return _detached(r)
        o = gs.code_balance(s["logits"], s["codes"])
        r = {"loss": o.loss, "counts": o.counts, "mean": o.mean_probs}
        if train:
            r["grad"] = torch.autograd.grad([o.loss, o.mean_probs], s["logits"], [s["g_loss"], s["g_mean"]])[0]
        return _detached(r)


def _detached(r):
    return {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in r.items()}


@torch.no_grad()
def _plain(s):
    if s["op"] == "lookup":
        return _plain_lookup(s)
    return _plain_probs(s) if s["op"] == "probs" else _plain_balance(s)


def _plain_lookup(s):
    table, codes, scales = s["codebook"].detach(), s["codes"], s["scales"]
    K, D = table.shape
    factor = (codes >= 0).float() if scales is None else scales * (codes >= 0)
    at = codes.clamp(min=0).long()
    rows = table.float()[at]
    r = {"out": (rows * factor.unsqueeze(-1)).to(table.dtype)}
    if s["train"]:
        g = s["grad"].float()
        g_table = torch.zeros(K, D, device=table.device)
        g_table.index_add_(0, at.reshape(-1), (g * factor.unsqueeze(-1)).reshape(-1, D))
        grads = [g_table.to(table.dtype)]
        if scales is not None:
            grads.append((g * rows).sum(-1) * (codes >= 0))
        r["grads"] = tuple(grads)
    return r


def _softmax(x, T):
    """(z - log sum, probabilities, sum, whether a row has any logit) of 32-bit logits; rows with none have probabilities of 0."""
    m = x.amax(-1, keepdim=True)
    some = m > -math.inf
    z = (x - torch.where(some, m, torch.zeros_like(m))) / T
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    return z - torch.log(total.clamp(min=1e-30)), e / total.clamp(min=1e-30), some


def _plain_probs(s):
    x, codes, k, T = s["logits"].detach().float(), s["codes"].long(), s["top"], s["T"]
    K = x.shape[-1]
    logp, p, some = _softmax(x, T)
    given = codes >= 0
    at = codes.clamp(min=0).unsqueeze(-1)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(-1)
    r = {"logp": torch.where(given, logp.gather(-1, at).squeeze(-1), torch.zeros_like(entropy)), "entropy": entropy}
    if k:
        bits = (x + 0.0).view(torch.int32)
        order = bits ^ ((bits >> 31) & 0x7FFFFFFF)  # ascending with the logit
        keys = (order.long() << 32) | (K - 1 - torch.arange(K, device=x.device))  # of equal ones the lowest index first
        best = K - 1 - (torch.topk(keys, k, dim=-1).values & 0xFFFFFFFF)
        r.update(top=logp.gather(-1, best), best=best.to(torch.int32))
    if s["train"]:
        gl = (s["g_logp"] * given).unsqueeze(-1) * some
        total = gl
        if k:
            gt = s["g_top"] * some
            total = total + gt.sum(-1, keepdim=True)
        g = -p * total - s["g_entropy"].unsqueeze(-1) * (plogp + p * entropy.unsqueeze(-1))
        g.scatter_add_(-1, at, gl)
        if k:
            g.scatter_add_(-1, best, gt)
        r["grad"] = (g / T).to(s["logits"].dtype)
    return r


def _plain_balance(s):
    x, codes = s["logits"].detach().float(), s["codes"].long()
    K, B = x.shape[-1], max(1, s["case"]["B"])
    _, p, _ = _softmax(x, 1.0)
    codes = codes.reshape(*x.shape[:-1], -1)
    given = codes >= 0
    takes_part = given.any(-1).float()
    p = p * takes_part.unsqueeze(-1)
    counts = torch.zeros(B, K, dtype=torch.int32, device=x.device)
    counts.scatter_add_(-1, codes.clamp(min=0).reshape(B, -1), given.reshape(B, -1).to(torch.int32))
    counts = counts.reshape(*x.shape[:-2], K)
    rows = takes_part.sum(-1, keepdim=True).clamp(min=1)
    share = counts.float() / counts.sum(-1, keepdim=True).clamp(min=1).float()
    mean = p.sum(-2) / rows
    r = {"loss": K * (share * mean).sum(-1), "counts": counts, "mean": mean}
    if s["train"]:
        a = (K * share * s["g_loss"].unsqueeze(-1) + s["g_mean"]).unsqueeze(-2)
        g = p * (a - (a * p).sum(-1, keepdim=True)) / rows.unsqueeze(-1)
        r["grad"] = g.to(s["logits"].dtype)
    return r


def work(case):
    N, K, b = max(1, case["B"]) * case["G"], case["K"], SIZE[case["dtype"]]
    code = 8 if case["long"] else 4
    if case["op"] == "lookup":
        D, scale = case["D"], 4 if case["scales"] else 0
        n = N * (code + scale + D * b) + min(N, K) * D * b
        flops = N * D
        if case["train"]:
            n += N * D * b + K * D * b + N * scale
            flops += N * D * (4 if scale else 1)
        return {"bytes": n, "flops": flops}
    if case["op"] == "probs":
        n = N * (K * b + code + 8 + 8 * case["top"])
        flops = 7 * N * K
        if case["train"]:
            n += N * (2 * K * b + 8 + 4 * case["top"])
            flops += 7 * N * K
        return {"bytes": n, "flops": flops}
    B = max(1, case["B"])
    n = N * (K * b + code * case["S"]) + B * (8 * K + 4)
    flops = 6 * N * K
    if case["train"]:
        n += N * 2 * K * b + B * (8 * K + 4)
        flops += 7 * N * K
    return {"bytes": n, "flops": flops}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "lookup":
        table, codes = s["codebook"].detach().to(f64), s["codes"].reshape(-1).long()
        K, D = table.shape
        scale = torch.ones(codes.numel(), dtype=f64, device=table.device) if s["scales"] is None \
            else s["scales"].detach().reshape(-1).to(f64)
        padded = torch.cat([table, torch.zeros(1, D, dtype=f64, device=table.device)])  # row K (and -1): no code
        r = {"out": (padded[codes] * scale[:, None]).reshape(*s["codes"].shape, D)}
        if case["train"]:
            g = s["grad"].reshape(-1, D).to(f64)
            order = torch.argsort(codes)
            edges = torch.searchsorted(codes[order], torch.arange(K + 1, device=codes.device))
            sums = torch.cat([torch.zeros(1, D, dtype=f64, device=table.device), (g * scale[:, None])[order].cumsum(0)])
            grads = [sums[edges[1:]] - sums[edges[:-1]]]
            if s["scales"] is not None:
                grads.append(torch.linalg.vecdot(g, padded[codes]).reshape(s["codes"].shape))
            r["grads"] = tuple(grads)
        return r
    K = case["K"]
    logits = s["logits"].detach().reshape(-1, K)
    N = logits.shape[0]
    step = max(1, (1 << 26) // K)
    dev = logits.device
    if case["op"] == "probs":
        T, k = case["T"], case["top"]
        codes = s["codes"].reshape(-1).long()
        logp, entropy = torch.empty(N, dtype=f64, device=dev), torch.empty(N, dtype=f64, device=dev)
        top = torch.empty(N, k, dtype=f64, device=dev)
        grad = torch.empty(N, K, dtype=f64, device=dev) if case["train"] else None
        for a in range(0, N, step):
            b = min(N, a + step)
            i = torch.arange(b - a, device=dev)
            y = logits[a:b].to(f64) / T
            lse = torch.logsumexp(y, -1, keepdim=True)
            empty = torch.isneginf(lse)
            lp = torch.where(empty, torch.full_like(y, -math.inf), y - lse)
            p = lp.exp()
            c = codes[a:b]
            logp[a:b] = torch.where(c < 0, torch.zeros_like(lse[:, 0]), lp[i, c.clamp(min=0)])
            entropy[a:b] = torch.special.entr(p).sum(-1)
            if k:
                # (64-bit values are equal where the logits are: the values of the best need no order among equals)
                top[a:b] = lp.topk(k, dim=-1).values
                best = torch.sort(logits[a:b].float(), dim=-1, descending=True, stable=True).indices[:, :k]
            if case["train"]:
                w = torch.zeros_like(p)  # d loss / d lp of single entries
                w[i, c.clamp(min=0)] += torch.where(c < 0, 0.0, s["g_logp"].reshape(-1)[a:b].to(f64))
                if k:
                    w.scatter_add_(1, best, s["g_top"].reshape(-1, k)[a:b].to(f64))
                ge = s["g_entropy"].reshape(-1)[a:b, None].to(f64)
                g = (w - p * w.sum(-1, keepdim=True) + ge * (torch.special.entr(p) - p * entropy[a:b, None])) / T
                grad[a:b] = torch.where(empty, torch.zeros_like(g), g)
        shape = s["codes"].shape
        r = {"logp": logp.reshape(shape), "entropy": entropy.reshape(shape)}
        if k:
            r.update(top=top.reshape(*shape, k), best=None)
        if case["train"]:
            r["grad"] = grad.reshape(*shape, K)
        return r
    B, S = max(1, case["B"]), case["S"]
    G = N // B
    codes = s["codes"].reshape(B, G, S).long()
    losses, means = [], []
    grad = torch.empty(N, K, dtype=f64, device=dev) if case["train"] else None
    for b in range(B):
        c = codes[b].reshape(-1)
        counts = torch.bincount(c[c >= 0], minlength=K).to(f64)
        share = counts / counts.sum().clamp(min=1)
        part = (codes[b] >= 0).sum(-1) > 0
        n = part.sum().clamp(min=1)
        acc = torch.zeros(K, dtype=f64, device=dev)

        def probs(lo, hi):
            p = torch.softmax(logits[b * G + lo:b * G + hi].to(f64), -1)
            return torch.where(part[lo:hi, None], p.nan_to_num(0.0), 0.0)

        for lo in range(0, G, step):
            acc += probs(lo, min(G, lo + step)).sum(0)
        means.append(acc / n)
        losses.append(K * torch.dot(share, means[-1]))
        if case["train"]:
            a = K * share * s["g_loss"].reshape(B)[b].to(f64) + s["g_mean"].reshape(B, K)[b].to(f64)
            for lo in range(0, G, step):
                hi = min(G, lo + step)
                p = probs(lo, hi)
                grad[b * G + lo:b * G + hi] = (p * a - p * (p @ a)[:, None]) / n
    shape = s["logits"].shape
    r = {"loss": torch.stack(losses).reshape(shape[:-2]), "counts": None, "mean": torch.stack(means).reshape(*shape[:-2], K)}
    if case["train"]:
        r["grad"] = grad.reshape(shape)
    return r
