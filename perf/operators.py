"""The transformer operators of the framework, as a user's program calls them, beside their plain forms.

Three operators: the root-mean-square norm with the residual's addition, rotary positions, and attention whose scores
may be capped, biased by distance and masked by documents, a shared prefix or the length of a cache.  `own` chooses
who computes: False, elementary torch operations; True, a traced program on the framework's device.
"""
import importlib
import math

import numpy as np
import torch

own = False

EPS = 1e-6
BASE = 10000.0


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of a decoding step through the norm of a 4096-wide network: latency
        dict(name="norm-token", op="norm", rows=1, width=4096, grad=False),
        # the training step of a 1024-wide network over 65536 tokens: bandwidth, both directions
        dict(name="norm-train", op="norm", rows=65536, width=1024, grad=True),
        # an odd width and an odd count of rows: no vector access fits
        dict(name="norm-odd", op="norm", rows=2001, width=5003, grad=True),
        # queries of a training batch, the two halves of a head turned against each other
        dict(name="rotary-train", op="rotary", batch=4, tokens=4096, heads=32, dim=128, rot=128, interleaved=False,
             far=0, stretch=1.0, grad=True),
        # part of a head, neighbouring pairs, positions of its own for every token, far out in a stretched context
        dict(name="rotary-far", op="rotary", batch=3, tokens=777, heads=5, dim=96, rot=64, interleaved=True,
             far=1000000, stretch=8.0, grad=True),
        # a training step over many short sequences
        dict(name="attend-short", op="attend", batch=16, tq=64, tk=64, heads=8, kv_heads=8, dim=64, causal=True,
             cap=0.0, slopes=False, docs=0, prefix=0, lengths=False, grad=True),
        # the ordinary training step
        dict(name="attend-train", op="attend", batch=2, tq=4096, tk=4096, heads=16, kv_heads=16, dim=128, causal=True,
             cap=0.0, slopes=False, docs=0, prefix=0, lengths=False, grad=True),
        # a long sequence, four query heads to a head of keys
        dict(name="attend-long", op="attend", batch=1, tq=8192, tk=8192, heads=16, kv_heads=4, dim=128, causal=True,
             cap=0.0, slopes=False, docs=0, prefix=0, lengths=False, grad=True),
        # documents packed into rows of odd length with padding behind them, capped scores, an odd head size
        dict(name="attend-packed", op="attend", batch=2, tq=4001, tk=4001, heads=12, kv_heads=4, dim=80, causal=True,
             cap=30.0, slopes=False, docs=700, prefix=0, lengths=False, grad=True),
        # reading prompts: a prefix that sees itself whole, scores that fall with distance, forward only
        dict(name="attend-prompt", op="attend", batch=4, tq=2048, tk=2048, heads=32, kv_heads=8, dim=128, causal=True,
             cap=0.0, slopes=True, docs=0, prefix=300, lengths=False, grad=False),
        # one new token for each of 32 sequences against a cache with room for 16384
        dict(name="decode-batch", op="attend", batch=32, tq=1, tk=16384, heads=32, kv_heads=8, dim=128, causal=True,
             cap=0.0, slopes=False, docs=0, prefix=0, lengths=True, grad=False),
        # one token of one sequence against a short cache: latency
        dict(name="decode-one", op="attend", batch=1, tq=1, tk=1025, heads=8, kv_heads=2, dim=64, causal=True,
             cap=0.0, slopes=True, docs=0, prefix=0, lengths=False, grad=False),
    ]


def _spread(rng, lo, hi):
    """a whole number between lo and hi, even over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "attend", "attend", "decode"])
    if op == "norm":
        width = _spread(rng, 1, 16384)
        return dict(op="norm", rows=_spread(rng, 1, max(1, min(100000, (1 << 26) // width))), width=width,
                    grad=rng.random() < 0.6)
    if op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        batch, heads = _spread(rng, 1, 8), _spread(rng, 1, 40)
        tokens = _spread(rng, 1, max(1, min(20000, (1 << 26) // (batch * heads * dim))))
        return dict(op="rotary", batch=batch, tokens=tokens, heads=heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                    interleaved=rng.random() < 0.5, far=rng.choice([0, 0, 5000, 2000000]),
                    stretch=rng.choice([1.0, 4.0, 32.0]), grad=rng.random() < 0.6)
    kv_heads = _spread(rng, 1, 8)
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    masks = dict(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3)
    if op == "decode":
        batch = _spread(rng, 1, 32)
        tk = _spread(rng, 1, max(1, min(60000, (1 << 28) // (batch * kv_heads * dim))))
        return dict(op="attend", batch=batch, tq=min(tk, rng.choice([1, 1, 1, 2, 5])), tk=tk, heads=heads,
                    kv_heads=kv_heads, dim=dim, causal=True, docs=0, prefix=0, lengths=rng.random() < 0.5, grad=False,
                    **masks)
    batch = _spread(rng, 1, 8)
    # no more pairs of tokens than the longest listed case has
    most = math.isqrt(8192 * 8192 * 16 // (batch * heads))
    tk = _spread(rng, 1, max(1, min(8192, most)))
    tq = tk if rng.random() < 0.7 else _spread(rng, 1, tk)
    causal = rng.random() < 0.8
    return dict(op="attend", batch=batch, tq=tq, tk=tk, heads=heads, kv_heads=kv_heads, dim=dim, causal=causal,
                docs=rng.choice([0, 0, max(1, tk // 3), 100]),
                prefix=rng.choice([0, 0, max(1, tk // 4)]) if causal else 0, lengths=False,
                grad=rng.random() < 0.6, **masks)


# ---------------------------------------------------------------------------------------------------- inputs
def _docs(case, gen):
    """document numbers [batch, tk]: lengths near `docs`, the first one cut; the last tokens of a row are padding (-1)"""
    b, t, n = case["batch"], case["tk"], case["docs"]
    cut = torch.randint(0, n, (b, 1), generator=gen, device="cuda")
    at = torch.arange(t, device="cuda")[None, :]
    ids = torch.div(at + cut, n, rounding_mode="floor").float()
    pad = torch.randint(0, max(1, t // 16), (b, 1), generator=gen, device="cuda")
    return torch.where(at >= t - pad, -torch.ones_like(ids), ids)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale

    x = {}
    if case["op"] == "norm":
        r, w = case["rows"], case["width"]
        x["x"], x["residual"] = normal(r, w, scale=0.7), normal(r, w, scale=2.0)
        x["scale"] = 1.0 + normal(w, scale=0.2)
        if case["grad"]:
            x["dy"], x["dh"] = normal(r, w, scale=1e-2), normal(r, w, scale=1e-2)
    elif case["op"] == "rotary":
        shape = (case["batch"], case["tokens"], case["heads"], case["dim"])
        x["x"] = normal(*shape)
        if case["far"]:
            x["positions"] = torch.randint(0, case["far"], shape[:2], generator=gen, device="cuda").float()
        if case["grad"]:
            x["dy"] = normal(*shape, scale=1e-2)
    else:
        b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        # some channels of queries and keys are louder than the others, as projections of trained networks are
        loud = torch.where(torch.arange(d, device="cuda") % 17 == 3, 2.5, 1.0)
        x["q"] = normal(b, case["tq"], h, d) * loud
        x["k"] = normal(b, case["tk"], g, d) * loud
        x["v"] = normal(b, case["tk"], g, d)
        if case["slopes"]:
            x["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h).float()
        if case["docs"]:
            x["docs"] = _docs(case, gen)
        if case["prefix"]:
            x["prefix"] = torch.randint(0, 2 * case["prefix"], (b,), generator=gen, device="cuda").float()
        if case["lengths"]:
            lo = max(1, case["tk"] // 2)
            x["lengths"] = torch.randint(lo, case["tk"] + 1, (b,), generator=gen, device="cuda").float()
        if case["grad"]:
            x["dout"] = normal(b, case["tq"], h, d, scale=1e-2)
    return x


class _DeviceArray:
    """a kept tensor of the framework's device, left where it is; the memory belongs to the device's handle"""

    def __init__(self, device, address, shape):
        self.device = device
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr="<f4", data=(address, False), version=2)


def _program(case, x):
    """traces the case's program once; what a user's program keeps is the device handle and the serialised program"""
    adb = importlib.import_module("autodiff-ir-rust_b200")
    ad, ir, nn = adb.autodiff, adb.ir, adb.nn
    dev = adb.devices.B200(torch.cuda.current_device(), flags=adb.devices.FLAG_DEVICE_RESULTS)
    ad.set_device(dev)
    ad.eager_dep_opt()

    def leaf(name):
        t = x.get(name)
        return None if t is None else ad.tensor(ir.DevicePayload(t.data_ptr(), t.numel(), t), list(t.shape))

    def data(name):
        return leaf(name).val().to_node()

    def backward(loss):
        """a loss is one number: the sum over every axis"""
        for _ in loss.dim():
            loss = loss.sum(len(loss.dim()) - 1)
        loss.forward()
        loss.backward()

    if case["op"] == "norm":
        a, scale = leaf("x"), leaf("scale")
        y, h = ad.rms_norm(a, scale, residual=leaf("residual"), eps=EPS)
        outs = [y.forward(), h.forward()]
        if case["grad"]:
            backward(y * data("dy") + h * data("dh"))
            outs += [a.grad(), scale.grad()]
    elif case["op"] == "rotary":
        a = leaf("x")
        turn = nn.Rotary(case["rot"], base=BASE, stretch=case["stretch"], interleaved=case["interleaved"])
        y = turn.f(a, positions=leaf("positions"))
        outs = [y.forward()]
        if case["grad"]:
            backward(y * data("dy"))
            outs.append(a.grad())
    else:
        q, k, v = leaf("q"), leaf("k"), leaf("v")
        out = ad.attention(q, k, v, causal=case["causal"], cap=case["cap"], slopes=leaf("slopes"), docs=leaf("docs"),
                           prefix=leaf("prefix"), lengths=leaf("lengths"))
        outs = [out.forward()]
        if case["grad"]:
            backward(out * data("dout"))
            outs += [q.grad(), k.grad(), v.grad()]
    for o in outs:
        o.keep()
    blob, alive = ir.serialize(ad.current_ir(), ad.ret_dep_list())
    return dict(device=dev, blob=blob, alive=alive, ids=[o.id for o in outs], views={})


def _view(p, id_):
    """the kept tensor as a torch tensor; made anew when the device has moved it"""
    address, shape = p["device"].get_tensor_device(id_)
    if p["views"].get(id_, (None, None))[0] != address:
        p["views"][id_] = address, torch.as_tensor(_DeviceArray(p["device"], address, shape), device="cuda")
    return p["views"][id_][1]


def prepare(case, seed):
    x = _inputs(case, seed)
    state = dict(case=case, x=x)
    if case["op"] == "rotary":
        state["freq"] = _frequencies(case)
    if own:
        state["program"] = _program(case, x)
    torch.cuda.synchronize()   # the framework's device works on streams of its own
    return state


def run(state):
    if own:
        p = state["program"]
        p["device"].execute_blob(p["blob"])
        return [_view(p, i) for i in p["ids"]]
    case, x = state["case"], state["x"]
    if case["op"] == "norm":
        return _norm(case, x)
    if case["op"] == "rotary":
        return _rotary(case, x, state["freq"])
    return _attend(case, x)


# ---------------------------------------------------------------------------------------------------- plain forms
def _norm(case, x):
    h = x["x"] + x["residual"]
    inv = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    n = h * inv
    y = n * x["scale"]
    if not case["grad"]:
        return [y, h]
    dn = x["dy"] * x["scale"]
    dx = x["dh"] + inv * (dn - n * (dn * n).mean(-1, keepdim=True))
    return [y, h, dx, (x["dy"] * n).sum(0)]


def _frequencies(case):
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda")
    return BASE ** (-2.0 * i / case["rot"]) / case["stretch"]


def _rotary(case, x, freq):
    rot, inter = case["rot"], case["interleaved"]
    at = x["positions"].double() if "positions" in x else torch.arange(case["tokens"], device="cuda").double()[None, :]
    angle = at[:, :, None, None] * freq      # far positions: 32 bits would lose the fraction of a turn
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(t, sin):
        if inter:
            a, b = t[..., 0:rot:2], t[..., 1:rot:2]
        else:
            a, b = t[..., : rot // 2], t[..., rot // 2: rot]
        c, d = a * cos - b * sin, b * cos + a * sin
        head = torch.stack((c, d), -1).flatten(-2) if inter else torch.cat((c, d), -1)
        return torch.cat((head, t[..., rot:]), -1)

    outs = [turn(x["x"], sin)]
    if case["grad"]:
        outs.append(turn(x["dy"], -sin))
    return outs


def _allowed(case, x, rows):
    """which keys the queries of some sequences may see [rows, tq, tk], and how far away they are"""
    tq, tk = case["tq"], case["tk"]
    n = x["lengths"][rows].view(-1, 1, 1) if case["lengths"] else torch.full((1, 1, 1), float(tk), device="cuda")
    pos = torch.arange(tq, device="cuda").view(1, -1, 1) + (n - tq)
    key = torch.arange(tk, device="cuda").float().view(1, 1, -1)
    see = (key < n) & (pos >= 0)
    if case["causal"]:
        back = key <= pos
        see = see & (back | (key < x["prefix"][rows].view(-1, 1, 1)) if case["prefix"] else back)
    if case["docs"]:
        ids = x["docs"][rows]
        mine = ids.gather(1, pos[..., 0].clamp(min=0).long().expand(ids.shape[0], -1))
        see = see & (mine[:, :, None] == ids[:, None, :]) & (ids[:, None, :] >= 0)
    return see[:, None, None], (pos - key).abs()[:, None, None]


def _attend(case, x):
    h, g, d, tq = case["heads"], case["kv_heads"], case["dim"], case["tq"]
    scale, cap = 1.0 / math.sqrt(d), case["cap"]
    outs = [[], [], [], []]
    step = max(1, (1 << 29) // (h * tq * case["tk"]))    # sequences whose scores are held at once
    for b in range(0, case["batch"], step):
        rows = slice(b, min(b + step, case["batch"]))

        def heads(name):      # [rows, kv heads, query heads that share them, tokens, dim]
            return x[name][rows].transpose(1, 2).unflatten(1, (g, -1))

        def back(t):
            return t.flatten(1, 2).transpose(1, 2)

        q, k, v = heads("q"), heads("k"), heads("v")
        see, dist = _allowed(case, x, rows)
        s = (q @ k.transpose(-1, -2)) * scale
        if cap:
            t = torch.tanh(s / cap)
            s = cap * t
        if case["slopes"]:
            s = s - x["slopes"].view(g, h // g, 1, 1) * dist
        s = torch.where(see, s, -math.inf)
        top = s.amax(-1, keepdim=True).clamp(min=-3e38)
        e = torch.exp(s - top)
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total > 0, total, 1.0)
        o = p @ v
        outs[0].append(back(o))
        if case["grad"]:
            do = heads("dout")
            ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
            if cap:
                ds = ds * (1.0 - t * t)
            ds = ds * scale
            outs[1].append(back(ds @ k))
            outs[2].append(back((ds.transpose(-1, -2) @ q).sum(2, keepdim=True)))
            outs[3].append(back((p.transpose(-1, -2) @ do).sum(2, keepdim=True)))
    return [torch.cat(o) for o in outs if o]


# ---------------------------------------------------------------------------------------------------- what a pass has to do
def _pairs(case):
    """pairs of a query and a key that it sees, over the whole batch (documents at half their first cut, no padding;
    prefixes and cache lengths at the middle of what is drawn)"""
    tq, tk = case["tq"], case["tk"]
    n = (max(1, tk // 2) + tk) // 2 if case["lengths"] else tk
    pos = np.arange(tq, dtype=np.int64) + n - tq
    pos = pos[pos >= 0]
    if not case["docs"]:
        last = np.minimum(pos + 1, n) if case["causal"] else np.full_like(pos, n)
        if case["prefix"]:
            last = np.maximum(last, min(case["prefix"], n))
        return int(last.sum()) * case["batch"]
    size, cut = case["docs"], case["docs"] // 2
    first = np.maximum(0, (pos + cut) // size * size - cut)
    end = np.minimum(n, ((pos + cut) // size + 1) * size - cut)
    if case["causal"]:
        end = np.maximum(pos + 1, np.minimum(end, case["prefix"]))
    return int((end - first).sum()) * case["batch"]


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        return dict(bytes=4 * (n * (8 if case["grad"] else 4) + case["width"] * (2 if case["grad"] else 1)),
                    flops=n * (12 if case["grad"] else 5))
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
        turned = n // case["dim"] * case["rot"]
        both = 2 if case["grad"] else 1
        at = case["batch"] * case["tokens"] if case["far"] else 0
        return dict(bytes=4 * (2 * n * both + at + case["rot"]), flops=3 * turned * both)
    b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    n = (max(1, case["tk"] // 2) + case["tk"]) // 2 if case["lengths"] else case["tk"]
    q, kv = b * case["tq"] * h * d, b * n * g * d
    small = (h if case["slopes"] else 0) + (b * case["tk"] if case["docs"] else 0) + (b if case["prefix"] else 0)
    # forward: two products over every pair; backward: the scores again and the four gradients' products
    return dict(bytes=4 * ((q + kv + kv + q) + (q + q + 2 * kv if case["grad"] else 0) + small),
                flops=_pairs(case) * h * d * (14 if case["grad"] else 4))


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    x = {k: v.double() for k, v in _inputs(case, seed).items()}
    if case["op"] == "norm":
        h = x["x"] + x["residual"]
        length = h.square().mean(-1, keepdim=True).add(EPS).sqrt()
        y = h / length * x["scale"]
        if not case["grad"]:
            return [y, h]
        w = x["dy"] * x["scale"]
        along = (w * h).sum(-1, keepdim=True) / case["width"]
        return [y, h, x["dh"] + w / length - h * along / length ** 3, (x["dy"] * h / length).sum(0)]
    if case["op"] == "rotary":
        pairs = case["rot"] // 2
        i = torch.arange(pairs, dtype=torch.float64, device="cuda")
        turn = torch.exp(-math.log(BASE) * i / pairs) / case["stretch"]
        at = x["positions"] if "positions" in x else torch.arange(case["tokens"], device="cuda").double().expand(case["batch"], -1)
        unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at[..., None, None] * turn)
        first = 2 * torch.arange(pairs, device="cuda") if case["interleaved"] else torch.arange(pairs, device="cuda")
        second = first + (1 if case["interleaved"] else pairs)
        outs = []
        for name, u in (("x", unit), ("dy", unit.conj())):
            if name in x:
                z = torch.complex(x[name][..., first], x[name][..., second]) * u
                t = x[name].clone()
                t[..., first], t[..., second] = z.real, z.imag
                outs.append(t)
        return outs
    b, h, g, d, tq, tk = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "tq", "tk"))
    outs = [torch.zeros_like(x["q"])]
    if case["grad"]:
        outs += [torch.zeros_like(x["q"]), torch.zeros_like(x["k"]), torch.zeros_like(x["v"])]
    j = torch.arange(tk, device="cuda", dtype=torch.float64)
    for n in range(b):
        length = x["lengths"][n] if case["lengths"] else float(tk)
        at = (torch.arange(tq, device="cuda", dtype=torch.float64) + length - tq)[:, None]
        hidden = (j >= length) | (at < 0)
        if case["causal"]:
            ahead = j > at
            hidden = hidden | (ahead & (j >= x["prefix"][n]) if case["prefix"] else ahead)
        if case["docs"]:
            doc = x["docs"][n]
            hidden = hidden | (doc[at[:, 0].clamp(min=0).long()][:, None] != doc) | (doc < 0)
        for m in range(h):
            q, k, v = x["q"][n, :, m], x["k"][n, :, m // (h // g)], x["v"][n, :, m // (h // g)]
            z = torch.einsum("id,jd->ij", q, k) / math.sqrt(d)
            bend = torch.ones((), dtype=torch.float64, device="cuda")
            if case["cap"]:
                z = torch.tanh(z / case["cap"])
                bend = 1 - z.square()
                z = z * case["cap"]
            if case["slopes"]:
                z = z - x["slopes"][m] * (at - j).abs()
            p = torch.softmax(z.masked_fill(hidden, -math.inf), -1).masked_fill(hidden, 0.0)
            outs[0][n, :, m] = torch.einsum("ij,jd->id", p, v)
            if case["grad"]:
                do = x["dout"][n, :, m]
                dp = torch.einsum("id,jd->ij", do, v)
                dz = p * (dp - (dp * p).sum(-1, keepdim=True)) * bend / math.sqrt(d)
                outs[1][n, :, m] = torch.einsum("ij,jd->id", dz, k)
                outs[2][n, :, m // (h // g)] += torch.einsum("ij,id->jd", dz, q)
                outs[3][n, :, m // (h // g)] += torch.einsum("ij,id->jd", p, do)
    return outs
