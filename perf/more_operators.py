"""The operators of decoders by code (splats whose code names a small map of their features), and of the gradients of a
training step over many tensors, each as a user's program calls it.

A case is a plain dict:

  op       "group"     group_codes and rows_by_code: splats' rows sorted by code
           "back"      rows_from_codes: rows in the order of the codes brought back, weighted, summed per splat
           "adapt"     group_codes and code_adapters: a low-rank map of each splat's row by its code, beside a shared one
           "clip"      clip_gradients: the norm of many tensors together, and their clipping
  train    forward and backward (every gradient comes back), or the forward under no_grad
  B, G     images (0: inputs without a batch axis) and splats per image
  S        codes per splat
  K        codes
  D        values per row; "adapt": D of the rows and E of the results
  r        rank of the maps ("adapt")
  dtype    "f32", "bf16" or "f16": of the rows, the maps and their results; "clip": of the decoders' tensors
  long     codes of 64 bits instead of 32
  skew     80% of the choices are of eight codes
  weights  a weight per choice ("back")
  base     the shared map's results are added to ("adapt")
  decoders tensors beside the scene's own ("clip"), of `size` values on average
  limit    the largest norm, as a share of the norm there is ("clip")
  into     clipped gradients go to tensors of their own instead of in place

About one choice in fifty is no code (-1): a splat that was pruned.
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


def _group(name, train, B, G, K, D, S=1, dtype="f32", long=False, skew=False):
    return dict(name=name, op="group", train=train, B=B, G=G, K=K, D=D, S=S, dtype=dtype, long=long, skew=skew)


def _back(name, train, B, G, K, D, S=1, dtype="f32", weights=True, skew=False):
    return dict(name=name, op="back", train=train, B=B, G=G, K=K, D=D, S=S, dtype=dtype, weights=weights, skew=skew, long=False)


def _adapt(name, train, B, G, K, D, E, r, dtype="bf16", base=True, skew=False, long=False):
    return dict(name=name, op="adapt", train=train, B=B, G=G, K=K, D=D, E=E, r=r, S=1, dtype=dtype, base=base, skew=skew, long=long)


def _clip(name, G, degree, decoders, size, dtype="f32", limit=0.25, into=True):
    return dict(name=name, op="clip", train=False, G=G, degree=degree, decoders=decoders, size=size, dtype=dtype, limit=limit,
                into=into)


def listed():
    return [
        # fitting a small image: a few hundred splats, thousands of steps; the calls' own cost
        _group("group_train_512", True, 0, 512, 64, 11),
        # four images in a batch, two codes per splat, most of them on a few codes
        _group("group_train_b4", True, 4, 65536, 256, 48, S=2, dtype="bf16", long=True, skew=True),
        # a million splats with wide features, taken to the decoders of a stored scene
        _group("group_eval_1m", False, 0, 1 << 20, 16384, 128),
        # the way back of the small image
        _back("back_train_512", True, 0, 512, 64, 11, S=2),
        # the way back of the batch, in the other 16-bit type
        _back("back_train_b4", True, 4, 65536, 256, 48, S=2, dtype="f16", skew=True),
        # the way back with four codes per splat and wide features
        _back("back_train_256k", True, 0, 262144, 1024, 128, S=4, dtype="bf16"),
        # one splat edited: a single row through its code's map
        _adapt("adapt_one", False, 0, 1, 64, 1024, 1024, 16),
        # rows of many scenes at once, each with its own map of wide features, beside the shared one
        _adapt("adapt_requests_61", False, 0, 61, 32, 4096, 4096, 16, dtype="f16", long=True),
        # splats' features to all attributes (59 values: position, scales, rotation, opacity, colours), in 32 bits
        _adapt("adapt_train_64k", True, 0, 65536, 64, 128, 59, 8, dtype="f32", base=False),
        # the largest: a training step with wide features and maps of a higher rank
        _adapt("adapt_train_128k", True, 2, 65536, 256, 1024, 1024, 32),
        # a small scene's gradients, clipped in every step
        _clip("clip_small", 4096, 0, 2, 192),
        # a million splats with colours that depend on the view and decoders in 16 bits; most steps clip nothing
        _clip("clip_1m", 1 << 20, 3, 300, 20011, dtype="bf16", limit=4.0, into=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("group", "back", "adapt", "clip"))
    dtype = rng.choice(("f32", "bf16", "f16"))
    train = rng.random() < 0.7
    B = rng.choice((0, 0, 1, 2, 5))
    skew, long = rng.random() < 0.3, rng.random() < 0.3
    if op == "clip":
        into = rng.random() < 0.5
        limit = rng.choice((0.1, 0.5, 2.0)) if into else rng.choice((1.5, 4.0))
        decoders = _log(rng, 1, 400)
        c = _clip("", _log(rng, 100, 1 << 20), rng.choice((0, 0, 1, 2, 3)), decoders,
                  _log(rng, 1, min(1 << 20, 6000000 // decoders)), dtype, limit, into)
    elif op == "adapt":
        D, E = (rng.choice((11, 59, 64, 128, 256, 1024, _log(rng, 8, 4096))) for _ in range(2))
        r = rng.choice((1, 4, 8, 16, 16, 32, 64, rng.randint(2, 128)))
        rows = _log(rng, 1, min(131072, (1 << 28) // (D + E), (1 << 33) // (r * (D + E))))
        K = _log(rng, 1, min(4096, max(1, (1 << 25) // (r * (D + E)))))
        c = _adapt("", train, B, max(1, rows // max(B, 1)), K, D, E, r, dtype, rng.random() < 0.6, skew, long)
    else:
        S = rng.choice((1, 1, 2, 3, 4, 8))
        D = rng.choice((1, 3, 11, 48, 64, 128, _log(rng, 1, 1024)))
        rows = max(1, min(_log(rng, 1, 1 << 20), (1 << 27) // (D * S)))
        G, K = max(1, rows // max(B, 1)), _log(rng, 1, 65536)
        if op == "group":
            c = _group("", train, B, G, K, D, S, dtype, long, skew)
        else:
            c = _back("", train, B, G, K, D, S, dtype, rng.random() < 0.7, skew)
    del c["name"]
    return c


def _shape(case):
    return ((case["B"],) if case["B"] else ()) + (case["G"],)


def _sorted(codes, K, S):
    """(order, places, starts): choices by code, those without one last; where each choice went; where codes begin."""
    flat = codes.reshape(-1).long()
    keys = torch.where(flat >= 0, flat, torch.full_like(flat, K))
    order = torch.sort(keys, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(order.numel(), device=order.device)
    places = torch.where(flat >= 0, places, torch.full_like(places, -1)).reshape(*(codes.shape if S > 1 else (*codes.shape, 1)))
    counts = torch.zeros(K + 1, dtype=torch.int64, device=codes.device)
    counts.scatter_add_(0, keys, torch.ones_like(keys))
    starts = torch.cat([counts.new_zeros(1), counts[:K].cumsum(0)])
    return order.int(), places.int(), starts.int()


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, device=dev, generator=gen)

    s = dict(case=case, op=case["op"], train=case["train"])
    dtype, train = DTYPES[case["dtype"]], case["train"]
    if case["op"] == "clip":
        G = case["G"]
        # positions, scales, rotations, opacities and colours of the splats
        shapes = [(G, 3), (G, 3), (G, 4), (G,), (G, (case["degree"] + 1) ** 2, 3)]
        sizes = [(1 << (k * 7919 % 5)) * case["size"] // 6 + 1 for k in range(case["decoders"])]
        # (the parts of a scene have gradients of quite different sizes)
        grads = [normal(*sh) * 10.0 ** -k for k, sh in enumerate(shapes)]
        # the decoders' are parts of one buffer, as a program that exchanges gradients between processes keeps them
        flat = torch.cat([normal(n) * (1 + k % 3) for k, n in enumerate(sizes)] + [normal(0)]).to(dtype)
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in [*grads, flat]))
        whole = [*grads, flat]
        out = [torch.empty_like(g) for g in whole] if case["into"] else None
        s.update(scene=len(grads), sizes=sizes, whole=whole, max_norm=norm * case["limit"], whole_out=out)
        return s
    shape, K, S, D = _shape(case), case["K"], case["S"], case["D"]
    many = (*shape, S) if S > 1 else shape
    c = torch.randint(0, K, many, device=dev, generator=gen)
    if case["skew"]:
        few = torch.randint(0, K, (8,), device=dev, generator=gen)
        pick = torch.randint(0, 8, many, device=dev, generator=gen)
        c = torch.where(torch.rand(many, device=dev, generator=gen) < 0.8, few[pick], c)
    c = torch.where(torch.rand(many, device=dev, generator=gen) < 0.02, torch.full_like(c, -1), c)
    c = c if case["long"] else c.to(torch.int32)
    if case["op"] == "back":
        s["groups"] = _sorted(c, K, S)  # (as the way there left it)
        s["rows"] = normal(c.numel(), D).to(dtype).requires_grad_(train)
        s["weights"] = torch.rand(many, device=dev, generator=gen).requires_grad_(train) if case["weights"] else None
        s["grad"] = normal(*shape, D).to(dtype) if train else None
        return s
    s["codes"] = c
    s["rows"] = normal(*shape, D).to(dtype).requires_grad_(train)
    if case["op"] == "group":
        s["grad"] = normal(c.numel(), D).to(dtype) if train else None
        return s
    E, r = case["E"], case["r"]
    s["down"] = (normal(K, r, D) / math.sqrt(D)).to(dtype).requires_grad_(train)
    s["up"] = (normal(K, E, r) / math.sqrt(r)).to(dtype).requires_grad_(train)
    s["base"] = normal(*shape, E).to(dtype).requires_grad_(train) if case["base"] else None
    s["scale"] = 0.5
    s["grad"] = normal(*shape, E).to(dtype) if train else None
    return s


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    gs = _package()
    if s["op"] == "clip":
        grads, out = _tensors(s, s["whole"]), _tensors(s, s["whole_out"])
        norm = gs.clip_gradients(grads, s["max_norm"], out=out)
        return {"norm": norm, "out": s["whole"] if out is None else s["whole_out"]}
    with torch.set_grad_enabled(s["train"]):
        if s["op"] == "group":
            groups = gs.group_codes(s["codes"], s["case"]["K"], several=s["case"]["S"] > 1)
            out = gs.rows_by_code(s["rows"], groups)
            r = {"out": out.detach(), "order": groups.order, "places": groups.places, "starts": groups.starts}
            inputs = [s["rows"]]
        elif s["op"] == "back":
            out = gs.rows_from_codes(s["rows"], gs.CodeGroups(*s["groups"]), s["weights"])
            r = {"out": out.detach()}
            inputs = [s["rows"], s["weights"]]
        else:
            groups = gs.group_codes(s["codes"], s["case"]["K"])
            out = gs.code_adapters(s["rows"], groups, s["down"], s["up"], base=s["base"], scale=s["scale"])
            r = {"out": out.detach()}
            inputs = [s["rows"], s["down"], s["up"], s["base"]]
        if s["train"]:
            r["grads"] = torch.autograd.grad(out, [t for t in inputs if t is not None], s["grad"])
        return r


def _tensors(s, whole):
    """The gradients, one of each tensor."""
    return None if whole is None else [*whole[:-1], *whole[-1].split(s["sizes"])]


@torch.no_grad()
def _plain(s):
    return {"group": _plain_group, "back": _plain_back, "adapt": _plain_adapt, "clip": _plain_clip}[s["op"]](s)


def _plain_group(s):
    codes, x, S = s["codes"], s["rows"].detach(), s["case"]["S"]
    order, places, starts = _sorted(codes, s["case"]["K"], S)
    flat = x.reshape(-1, x.shape[-1])
    named = (torch.arange(order.numel(), device=x.device) < starts[-1]).unsqueeze(-1)
    out = torch.where(named, flat[order.long() // S], torch.zeros_like(flat[:1]))
    r = {"out": out, "order": order, "places": places, "starts": starts}
    if s["train"]:
        at = places.reshape(-1, S)
        g = s["grad"].float()[at.clamp(min=0).long()] * (at >= 0).unsqueeze(-1)
        r["grads"] = (g.sum(1).to(x.dtype).reshape(x.shape),)
    return r


def _plain_back(s):
    (order, places, starts), y, S = s["groups"], s["rows"].detach(), s["case"]["S"]
    shape = _shape(s["case"])
    at = places.reshape(-1, S)
    w = torch.ones(at.shape, device=y.device) if s["weights"] is None else s["weights"].detach().reshape(-1, S)
    w = w * (at >= 0)
    rows = y[at.clamp(min=0).long()].float()
    r = {"out": (rows * w.unsqueeze(-1)).sum(1).to(y.dtype).reshape(*shape, -1)}
    if s["train"]:
        g = s["grad"].float().reshape(-1, 1, y.shape[-1])
        of_rows = (g[order.long() // S, 0] * w.reshape(-1)[order.long()].unsqueeze(-1)).to(y.dtype)
        grads = [of_rows]
        if s["weights"] is not None:
            grads.append(((g * rows).sum(-1) * (at >= 0)).reshape(s["weights"].shape))
        r["grads"] = tuple(grads)
    return r


def _plain_adapt(s):
    x, down, up, base = (None if s[k] is None else s[k].detach() for k in ("rows", "down", "up", "base"))
    K, r, D = down.shape
    E, f = up.shape[1], s["scale"]
    codes = s["codes"].reshape(-1).long()
    flat = x.reshape(-1, D)
    N = flat.shape[0]
    train = s["train"]
    out = torch.empty(N, E, dtype=x.dtype, device=x.device)
    if train:
        g = s["grad"].reshape(-1, E)
        gx = torch.empty_like(flat)
        g_down = torch.zeros(K, r, D, device=x.device)
        g_up = torch.zeros(K, E, r, device=x.device)
    step = max(1, (1 << 26) // (r * max(D, E)))  # rows whose own copies of the maps take 256 MB
    for a in range(0, N, step):
        c = codes[a:a + step]
        named = (c >= 0).float().unsqueeze(-1)
        c = c.clamp(min=0)
        xs, dn, u = flat[a:a + step].float(), down[c].float(), up[c].float()
        h = torch.matmul(dn, xs.unsqueeze(-1)).squeeze(-1) * named
        y = torch.matmul(u, h.unsqueeze(-1)).squeeze(-1) * f
        out[a:a + step] = y if base is None else base.reshape(-1, E)[a:a + step].float() + y
        if train:
            gs = g[a:a + step].float()
            dh = torch.matmul(gs.unsqueeze(-2), u).squeeze(-2) * (named * f)
            gx[a:a + step] = torch.matmul(dh.unsqueeze(-2), dn).squeeze(-2)
            g_down.index_add_(0, c, dh.unsqueeze(-1) * xs.unsqueeze(-2))
            g_up.index_add_(0, c, (gs * f).unsqueeze(-1) * h.unsqueeze(-2))
    res = {"out": out.reshape(*x.shape[:-1], E)}
    if train:
        grads = [gx.reshape(x.shape), g_down.to(x.dtype), g_up.to(x.dtype)]
        res["grads"] = tuple(grads + ([s["grad"]] if base is not None else []))
    return res


def _plain_clip(s):
    grads, out = _tensors(s, s["whole"]), _tensors(s, s["whole_out"])
    total = torch.zeros((), dtype=torch.float64, device=grads[0].device)
    for g in grads:
        total += g.float().square().sum()
    norm = total.sqrt().float()
    factor = (s["max_norm"] / norm).clamp(max=1.0)
    for g, o in zip(grads, grads if out is None else out):
        o.copy_(g.float() * factor)
    return {"norm": norm, "out": s["whole"] if out is None else s["whole_out"]}


def _values(case):
    """Values of a scene's and its decoders' gradients: of 32 bits, and of the decoders' type."""
    return case["G"] * (11 + 3 * (case["degree"] + 1) ** 2), \
        sum((1 << (k * 7919 % 5)) * case["size"] // 6 + 1 for k in range(case["decoders"]))


def work(case):
    b = SIZE[case["dtype"]]
    if case["op"] == "clip":
        scene, decoders = _values(case)
        n = 4 * scene + b * decoders
        return {"bytes": n * (2 if case["limit"] < 1 else 1) + 4, "flops": (scene + decoders) * (3 if case["limit"] < 1 else 2)}
    N, S, K, D = max(1, case["B"]) * case["G"], case["S"], case["K"], case["D"]
    P, code = N * S, 8 if case["long"] else 4
    train = 2 if case["train"] else 1
    if case["op"] == "group":
        return {"bytes": P * (code + 8) + 4 * (K + 1) + train * (N + P) * D * b + (4 * P if train == 2 else 0),
                "flops": P * D if train == 2 else P}
    if case["op"] == "back":
        w = 4 * P if case["weights"] else 0
        n = 4 * P + w + (N + P) * D * b
        if train == 2:
            n += 2 * w + 4 * P + (N + P + (P if w else 0)) * D * b
        return {"bytes": n, "flops": P * D * (2 if train == 1 else 5)}
    E, r = case["E"], case["r"]
    n = N * (code + (D + E + (E if case["base"] else 0)) * b) + min(K, N) * r * (D + E) * b
    if train == 2:
        n += N * (2 * D + E) * b + min(K, N) * r * (D + E) * b + K * r * (D + E) * b
    return {"bytes": n, "flops": 2 * N * r * (D + E) * (3 if train == 2 else 1)}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "clip":
        norm = math.sqrt(sum(float(torch.dot(g.reshape(-1).to(f64), g.reshape(-1).to(f64))) for g in s["whole"]))
        factor = min(1.0, s["max_norm"] / norm)
        return {"norm": torch.tensor(norm, dtype=f64, device="cuda:0"), "out": [g.to(f64) * factor for g in s["whole"]]}
    shape, S, D = _shape(case), case["S"], case["D"]
    if case["op"] == "group":
        x = s["rows"].detach().reshape(-1, D)
        codes = s["codes"].reshape(-1)
        named = torch.nonzero(codes >= 0).squeeze(-1)
        by_code = named[torch.argsort(codes[named], stable=True)]
        out = torch.zeros(codes.numel(), D, dtype=f64, device=x.device)
        out[:by_code.numel()] = x.index_select(0, by_code // S).to(f64)
        r = {"out": out, "order": None, "places": None, "starts": None}
        if case["train"]:
            g = torch.zeros(codes.numel(), D, dtype=f64, device=x.device)
            g[by_code] = s["grad"][:by_code.numel()].to(f64)
            r["grads"] = (torch.einsum("nsd->nd", g.reshape(-1, S, D)).reshape(*shape, D),)
        return r
    if case["op"] == "back":
        order, places, starts = s["groups"]
        n = int(starts[-1])
        splat, choice = order[:n].long() // S, order[:n].long()
        y = s["rows"].detach()[:n].to(f64)
        w = torch.ones(n, dtype=f64, device=y.device) if s["weights"] is None \
            else s["weights"].detach().reshape(-1)[choice].to(f64)
        lone = torch.zeros(places.numel(), D, dtype=f64, device=y.device)
        lone[choice] = y * w[:, None]
        r = {"out": lone.reshape(-1, S, D).sum(1).reshape(*shape, D)}
        del lone
        if case["train"]:
            g = s["grad"].reshape(-1, D)[splat].to(f64)
            g_rows = torch.zeros(places.numel(), D, dtype=f64, device=y.device)
            g_rows[:n] = g * w[:, None]
            grads = [g_rows]
            if s["weights"] is not None:
                g_w = torch.zeros(places.numel(), dtype=f64, device=y.device)
                g_w[choice] = torch.linalg.vecdot(g, y)
                grads.append(g_w.reshape(s["weights"].shape))
            r["grads"] = tuple(grads)
        return r
    x, codes = s["rows"].detach().reshape(-1, D), s["codes"].reshape(-1)
    K, r, _ = s["down"].shape
    E, f, train = case["E"], s["scale"], case["train"]
    zeros = dict(dtype=f64, device=x.device)
    out = torch.zeros(x.shape[0], E, **zeros) if s["base"] is None else s["base"].detach().reshape(-1, E).to(f64)
    if train:
        gx, g_down, g_up = torch.zeros(x.shape[0], D, **zeros), torch.zeros(K, r, D, **zeros), torch.zeros(K, E, r, **zeros)
        g = s["grad"].reshape(-1, E)
    ids, counts = torch.unique(codes, return_counts=True)
    by_code = torch.argsort(codes, stable=True).split(counts.tolist())
    for k, rows in zip(ids.tolist(), by_code):
        if k < 0:
            continue
        dn, u, xs = s["down"].detach()[k].to(f64), s["up"].detach()[k].to(f64), x[rows].to(f64)
        h = xs @ dn.t()
        out[rows] += f * (h @ u.t())
        if train:
            gk = g[rows].to(f64)
            dh = f * (gk @ u)
            gx[rows] = dh @ dn
            g_down[k] = dh.t() @ xs
            g_up[k] = f * (gk.t() @ h)
    res = {"out": out.reshape(*shape, E)}
    if train:
        grads = [gx.reshape(*shape, D), g_down, g_up]
        res["grads"] = tuple(grads + ([s["grad"].to(f64)] if s["base"] is not None else []))
    return res
