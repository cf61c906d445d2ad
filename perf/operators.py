"""The serving and packed-training operators as measurable cases.

Each case is one pass through an operator on inputs of the distributions the model meets: QK
RMS-normalised scores, a learned per-head sink, the algebraic preset's exponents (n = 16,
c = 8). With ``own`` false ``run`` computes the plain form in elementary torch operations of 32
bits; with ``own`` true it makes the calls a user makes. ``listed`` names the sizes that stand
for the range, ``draw`` gives others of the same range, ``exact`` states the maths in float64.

Attention: scores x = q.k / (sqrt(D) c), weights w = (x + sqrt(1 + x^2))^n over the keys at or
before the query's position, normalised together with the sink's weight; H query heads share
Hkv key and value heads in groups of H / Hkv.
"""

import math
import sys
from pathlib import Path

import torch

own = False

N_EXP, C = 16, 8.0
EPS = 1e-5
E4M3_MAX = 448.0


def listed():
    return [
        # One training microbatch of packed documents, 1B heads (D = 128) with four queries to a key head.
        dict(name="packed_1b_train", kind="packed", N=16384, S=9, spread=6.0, H=16, Hkv=4, D=128, train=True),
        # The same at the 350M shape, every query head with a key head of its own, odd lengths.
        dict(name="packed_350m_train", kind="packed", N=8161, S=13, spread=5.0, H=16, Hkv=16, D=64, train=True),
        # A few short documents: launches and latency count.
        dict(name="packed_short_train", kind="packed", N=403, S=3, spread=3.0, H=12, Hkv=4, D=64, train=True),
        # Prefill of a few long prompts, forward only.
        dict(name="packed_prefill", kind="packed", N=16384, S=3, spread=2.0, H=32, Hkv=8, D=128, train=False),
        # One token for each of a few requests: the smallest serving step.
        dict(name="decode_small", kind="paged", S=4, spread=2.0, kv=3600, chunk=1, H=16, Hkv=4, D=128, page=16),
        # One token for each of a full batch.
        dict(name="decode_batch", kind="paged", S=64, spread=4.0, kv=200000, chunk=1, H=32, Hkv=8, D=128, page=64),
        # One token of one request over a very long cache: the work has to be split over the keys.
        dict(name="decode_long", kind="paged", S=1, spread=1.0, kv=131001, chunk=1, H=16, Hkv=4, D=128, page=128),
        # A chunk of a prompt for each of three requests whose earlier part is in the cache.
        dict(name="chunk_prefill", kind="paged", S=3, spread=2.0, kv=24000, chunk=701, H=16, Hkv=4, D=128, page=48),
        # The new tokens' norm, rotation and place in the cache, one token a request.
        dict(name="append_decode", kind="append", S=64, spread=4.0, kv=40000, chunk=1, H=32, Hkv=8, D=128, page=64),
        # The same for whole prompts.
        dict(name="append_prompts", kind="append", S=5, spread=3.0, kv=12000, chunk=1600, H=16, Hkv=16, D=64, page=32),
        # The residual stream's addition and norm between two blocks, one training microbatch of the 1B shape.
        dict(name="add_norm_train", kind="norm", rows=16384, d=2048, out="bf16"),
        # The same ahead of an 8-bit product, one serving step.
        dict(name="add_norm_fp8", kind="norm", rows=509, d=2048, out="fp8"),
    ]


# --- drawn cases ---------------------------------------------------------------------------

def _logint(rng, lo, hi, step=1):
    """A whole number of [lo, hi], uniform over its logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def _heads(rng):
    G = rng.choice([1, 2, 3, 4, 8])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    while G * Hkv > 32:
        Hkv //= 2
    return G * Hkv, Hkv


def draw(rng):
    kind = rng.choice(["packed", "packed", "packed", "paged", "paged", "paged", "append", "norm"])
    spread = round(math.exp(rng.uniform(0.0, math.log(8.0))), 2)
    H, Hkv = _heads(rng)
    D = rng.choice([64, 128])
    if kind == "packed":
        S = _logint(rng, 1, 32)
        N = _logint(rng, max(64, 4 * S), 16384)
        case = dict(kind=kind, N=N, S=S, spread=spread, H=H, Hkv=Hkv, D=D, train=rng.random() < 0.7)
        # The plain form holds S H L^2 scores, L the longest sequence.
        while case["N"] > 64 and S * H * max(lens(case["N"], S, spread)) ** 2 > 2.3e9:
            case["N"] = int(case["N"] * 0.8)
        return case
    if kind == "norm":
        rows, d = _logint(rng, 1, 16384), _logint(rng, 256, 4096, 8)
        while rows * d > 16384 * 2048:
            rows = int(rows * 0.8)
        return dict(kind=kind, rows=rows, d=d, out=rng.choice(["bf16", "fp8"]))
    S = _logint(rng, 1, 64)
    page = rng.choice([16, 32, 48, 64, 128])
    chunk = 1 if kind == "paged" and rng.random() < 0.5 else _logint(rng, 1, 900 if kind == "paged" else 1600)
    while S * chunk > 8000:
        S = max(1, S // 2)
    kv = _logint(rng, S * (chunk + 8) * 4, max(S * (chunk + 8) * 4 + 1, 200000 if kind == "paged" else 40000))
    if kind == "paged":
        while kv > S * (chunk + 8) * 4 and (S * H * chunk * max(lens(kv, S, spread)) > 1.2e9 or
                                            S * Hkv * D * max(lens(kv, S, spread)) > 3e8):
            kv = int(kv * 0.8)
    return dict(kind=kind, S=S, spread=spread, kv=kv, chunk=chunk, H=H, Hkv=Hkv, D=D, page=page)


def lens(total, S, spread):
    """`total` in S parts, the largest about `spread` times the smallest, large and small in turn."""
    w = [spread ** (i / max(1, S - 1)) for i in range(S)]
    w = w[::2] + w[1::2][::-1]
    got = [max(1, int(total * x / sum(w))) for x in w]
    got[0] += max(0, total - sum(got))
    return got


# --- inputs ---------------------------------------------------------------------------------

def _normed(x):
    return x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))

    def rn(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32)

    bf = torch.bfloat16
    s = {"case": case}
    if case["kind"] == "norm":
        rows, d = case["rows"], case["d"]
        train = case["out"] == "bf16"
        s["x"] = rn(rows, d).to(bf).requires_grad_(train)
        s["r"] = (2 * rn(rows, d)).to(bf).requires_grad_(train)
        s["gain"] = (1 + 0.1 * rn(d)).to(bf).requires_grad_(train)
        if train:
            s["dy"], s["ds"] = rn(rows, d).to(bf), rn(rows, d).to(bf)
        return s
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if case["kind"] == "packed":
        N, train = case["N"], case["train"]
        ls = lens(N, case["S"], case["spread"])
        s["longest"] = max(ls)
        s["cu"] = _i32([sum(ls[:i]) for i in range(len(ls) + 1)], dev)
        for name, heads in (("q", H), ("k", Hkv), ("v", Hkv)):
            t = rn(N, heads, D)
            s[name] = (t if name == "v" else _normed(t)).to(bf).requires_grad_(train)
        s["sink"] = (0.1 * rn(H)).to(bf).requires_grad_(train)
        if train:
            s["do"] = rn(N, H, D).to(bf)
        return s
    # A cache of pages in a shuffled order, more of them than the requests use; the requests'
    # last `chunk` tokens (an eighth fewer or more) are the new ones.
    S, page = case["S"], case["page"]
    kv = lens(case["kv"], S, case["spread"])
    new = [1 if case["chunk"] == 1 else min(n, max(1, case["chunk"] + (i % 3 - 1) * (case["chunk"] // 8)))
           for i, n in enumerate(kv)]
    need = [-(-n // page) for n in kv]
    width, pages = max(need), sum(need) + 5
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    table = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    N = sum(new)
    s.update(longest=max(kv), chunk=max(new), table=table, cu=_i32([sum(new[:i]) for i in range(S + 1)], dev), kv=_i32(kv, dev))
    if case["kind"] == "paged":
        s["q"] = _normed(rn(N, H, D)).to(bf)
        s["kp"] = _normed(rn(pages, Hkv, page, D)).to(bf)
        s["vp"] = rn(pages, Hkv, page, D).to(bf)
        s["sink"] = 0.1 * rn(H)
        return s
    s["kp"] = torch.zeros(pages, Hkv, page, D, dtype=bf, device=dev)
    s["vp"] = torch.zeros(pages, Hkv, page, D, dtype=bf, device=dev)
    for name, heads in (("q", H), ("k", Hkv), ("v", Hkv)):
        s[name] = (1.5 * rn(N, heads, D)).to(bf)
    s["gq"], s["gk"] = 1 + 0.1 * rn(D), 1 + 0.1 * rn(D)
    half = D // 2
    w = 0.5 * 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
    angle = 2 * torch.arange(width * page, device=dev, dtype=torch.float64)[:, None] * torch.atan(w)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# --- one pass --------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    pkg = str(Path.cwd() / "algebraic-transformer_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from algebraic_amd.kernels.norm import add_rms_norm, add_rms_norm_fp8
    from algebraic_amd.kernels.packed import packed_flash_attention
    from algebraic_amd.kernels.paged import paged_append, paged_flash_attention

    case, kind = s["case"], s["case"]["kind"]
    if kind == "packed":
        o = packed_flash_attention(s["q"], s["k"], s["v"], s["cu"], s["sink"], n=N_EXP, c=C)
        if not case["train"]:
            return [o]
        return [o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"], s["sink"]), s["do"])]
    if kind == "paged":
        return [paged_flash_attention(s["q"], s["kp"], s["vp"], s["table"], s["cu"], s["kv"], s["sink"], n=N_EXP, c=C)]
    if kind == "append":
        q = paged_append(s["q"], s["k"], s["v"], s["kp"], s["vp"], s["table"], s["cu"], s["kv"], s["gq"], s["gk"],
                         s["cos"], s["sin"], eps=EPS)
        return [q, s["kp"], s["vp"]]
    if case["out"] == "fp8":
        y8, scale, h = add_rms_norm_fp8(s["x"], s["r"], s["gain"], EPS)
        return [(y8.to(torch.float32) * scale).to(torch.bfloat16), scale, h]
    y, h = add_rms_norm(s["x"], s["r"], s["gain"], EPS)
    return [y, h, *torch.autograd.grad((y, h), (s["x"], s["r"], s["gain"]), (s["dy"], s["ds"]))]


# The plain forms: sequences padded to the longest, everything in 32 bits, rounded at the end.

def _padded(rows, cu, longest):
    """(S, longest, ...) of packed rows, and which of its places hold a row."""
    t = torch.arange(longest, device=cu.device)
    live = t < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + t).clamp(max=rows.shape[0] - 1).long()
    return torch.where(live[..., None, None], rows[at].float(), 0.0), live


def _weights(q, k, sink, dead):
    """Scores and normalised weights of q (S, Hkv, G, L, D) over k (S, Hkv, 1, K, D), and the sink's weight."""
    x = (q @ k.transpose(-1, -2)) * (1.0 / (math.sqrt(q.shape[-1]) * C))
    a = (N_EXP * torch.asinh(x)).masked_fill_(dead, -math.inf)
    ab = N_EXP * torch.asinh(sink / C)
    m = torch.maximum(a.amax(-1, keepdim=True), ab)
    w = a.sub_(m).exp_()
    wb = (ab - m).exp()
    z = w.sum(-1, keepdim=True) + wb
    return x, w.div_(z), wb / z


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    bf = torch.bfloat16
    if kind == "norm":
        return _plain_norm(s, case["out"])
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    G = H // Hkv
    if kind == "append":
        return _plain_append(s, H, Hkv, D, case["page"])
    cu = s["cu"].long()

    def query_heads(t):  # (S, L, H, D) -> (S, Hkv, G, L, D)
        return t.unflatten(2, (Hkv, G)).permute(0, 2, 3, 1, 4)

    def key_heads(t):
        return t.permute(0, 2, 1, 3).unsqueeze(2)

    sink = s["sink"].detach().float().view(Hkv, G, 1, 1)
    longest = s["longest"] if kind == "packed" else s["chunk"]
    qp, live = _padded(s["q"].detach(), cu, longest)
    q = query_heads(qp)
    if kind == "packed":
        k, v = (key_heads(_padded(s[n].detach(), cu, longest)[0]) for n in "kv")
        pos = torch.arange(longest, device=cu.device).expand(len(cu) - 1, -1)
    else:
        t = torch.arange(s["longest"], device=cu.device)
        kv = s["kv"].long()
        page = s["table"].long()[:, t // case["page"]].clamp(min=0)
        held = (t < kv[:, None])[:, :, None, None]
        k, v = (key_heads(torch.where(held, s[n][page, :, t % case["page"]].float(), 0.0)) for n in ("kp", "vp"))
        pos = (kv - (cu[1:] - cu[:-1]))[:, None] + torch.arange(longest, device=cu.device)
    dead = (torch.arange(k.shape[3], device=cu.device) > pos[..., None])[:, None, None]
    x, p, pb = _weights(q, k, sink, dead)
    o = p @ v

    def packed(t):  # (S, Hkv, G, L, D) back to rows
        return t.permute(0, 3, 1, 2, 4).flatten(2, 3)[live]

    out = packed(o).to(bf)
    if kind == "paged" or not case["train"]:
        return [out]
    do = query_heads(_padded(s["do"], cu, longest)[0])
    di = (do * o).sum(-1, keepdim=True)
    dsink = -(pb * di).sum((0, 3, 4)) * N_EXP * torch.rsqrt(1 + (sink / C).square())[..., 0, 0] / C
    ds = (do @ v.transpose(-1, -2)).sub_(di).mul_(p).mul_(x.square_().add_(1).rsqrt_())
    ds *= N_EXP / (math.sqrt(D) * C)
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    dv = (p.transpose(-1, -2) @ do).sum(2, keepdim=True)
    return [out, packed(dq).to(bf), packed(dk).to(bf), packed(dv).to(bf), dsink.flatten().to(bf)]


def _plain_append(s, H, Hkv, D, page):
    bf = torch.bfloat16
    cu, kv = s["cu"].long(), s["kv"].long()
    new = cu[1:] - cu[:-1]
    N = s["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(kv), device=cu.device), new, output_size=N)
    pos = torch.arange(N, device=cu.device) - cu[seq] + (kv - new)[seq]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(x, gain):
        a, b = (_normed(x.float()) * gain).chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(bf)

    at = s["table"].long()[seq, pos // page]
    s["kp"][at, :, pos % page] = turned(s["k"], s["gk"])
    s["vp"][at, :, pos % page] = s["v"]
    return [turned(s["q"], s["gq"]), s["kp"], s["vp"]]


def _plain_norm(s, out):
    bf = torch.bfloat16
    h = (s["x"].detach().float() + s["r"].detach().float()).to(bf)
    h32, gain = h.float(), s["gain"].detach().float()
    tau = (h32.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = h32 * tau * gain
    if out == "fp8":
        scale = y.abs().amax(-1, keepdim=True) / E4M3_MAX
        scale = torch.where(scale > 0, scale, 1.0)
        return [((y / scale).to(torch.float8_e4m3fn).float() * scale).to(bf), scale, h]
    dy = s["dy"].float()
    a = dy * gain
    dh = a * tau - h32 * tau ** 3 * (a * h32).mean(-1, keepdim=True) + s["ds"].float()
    dh = dh.to(bf)
    return [y.to(bf), h, dh, dh, (dy * h32 * tau).sum(0).to(bf)]


# --- what a pass cannot do without ----------------------------------------------------------

def work(case):
    if case["kind"] == "norm":
        n, d = case["rows"], case["d"]
        if case["out"] == "fp8":  # x, r in; the sum, the bytes and the scales out
            return {"bytes": n * d * 7 + n * 4 + d * 2, "flops": 8.0 * n * d}
        # x, r in, y and the sum out; dy, ds and the sum in, the one gradient of both out.
        return {"bytes": n * d * 16 + d * 4, "flops": 20.0 * n * d}
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    if case["kind"] == "packed":
        ls = lens(case["N"], case["S"], case["spread"])
        scores = sum(n * (n + 1) // 2 for n in ls) * H
        tensors = case["N"] * D * 2 * (2 * H + 2 * Hkv)  # q, o, k, v
        if not case["train"]:
            return {"bytes": tensors, "flops": 4.0 * scores * D}
        # backward: dO in, dq, dk, dv out (q, k, v and o counted once).
        return {"bytes": 2 * tensors, "flops": 14.0 * scores * D}
    S, chunk, page = case["S"], case["chunk"], case["page"]
    kv = lens(case["kv"], S, case["spread"])
    new = [1 if chunk == 1 else min(n, max(1, chunk + (i % 3 - 1) * (chunk // 8))) for i, n in enumerate(kv)]
    if case["kind"] == "append":  # q, k, v in and out, a row of each table
        return {"bytes": sum(new) * (2 * (H + 2 * Hkv) * D * 2 + D * 4), "flops": 10.0 * sum(new) * (H + Hkv) * D}
    scores = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(new, kv)) * H
    return {"bytes": sum(kv) * Hkv * D * 4 + sum(new) * H * D * 4 + sum(-(-n // page) for n in kv) * 4,
            "flops": 4.0 * scores * D}


# --- the same maths in 64 bits ---------------------------------------------------------------

def _attend64(q, k, v, sink, do=None, rows=2048):
    """One head's queries, the last of q.shape[0] positions of k: outputs, and gradients for `do`."""
    D = q.shape[1]
    first = k.shape[0] - q.shape[0]
    alpha = 1.0 / (math.sqrt(D) * C)
    o, dq, dk, dv, dsink = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v), 0.0
    for a in range(0, q.shape[0], rows):
        b = min(a + rows, q.shape[0])
        e = first + b
        x = alpha * (q[a:b] @ k[:e].T)
        logw = torch.log(torch.hypot(x, torch.ones_like(x)) + x.abs()) * x.sign() * N_EXP
        pos = torch.arange(first + a, e, device=q.device)[:, None]
        logw[torch.arange(e, device=q.device)[None] > pos] = -math.inf
        beta = sink / C
        p = torch.softmax(torch.cat([logw, (N_EXP * torch.asinh(beta)).expand(b - a, 1)], 1), 1)
        pb, p = p[:, -1], p[:, :-1]
        o[a:b] = p @ v[:e]
        if do is None:
            continue
        di = (do[a:b] * o[a:b]).sum(1)
        ds = p * (do[a:b] @ v[:e].T - di[:, None]) * N_EXP / torch.hypot(x, torch.ones_like(x))
        dq[a:b] = alpha * (ds @ k[:e])
        dk[:e] += alpha * (ds.T @ q[a:b])
        dv[:e] += p.T @ do[a:b]
        dsink = dsink - (pb * di).sum() * N_EXP / torch.sqrt(1 + beta * beta) / C
    return o, dq, dk, dv, dsink


def exact(case, seed):
    s = prepare(case, seed)
    d64 = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if case["kind"] == "norm":
        h = (s["x"].detach() + s["r"].detach()).double()  # the stream as it is stored
        gain = d64["gain"]
        rms = (h.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        y = h / rms * gain
        if case["out"] == "fp8":
            scale = y.abs().amax(-1, keepdim=True) / E4M3_MAX
            return [(y / scale).to(torch.float8_e4m3fn).double() * scale, scale, d64["x"] + d64["r"]]
        g = d64["dy"] * gain / rms
        dh = g - h * (g * h).sum(-1, keepdim=True) / (case["d"] * rms * rms) + d64["ds"]
        return [y, d64["x"] + d64["r"], dh, dh, (d64["dy"] * h / rms).sum(0)]
    H, Hkv = case["H"], case["Hkv"]
    cu = s["cu"].tolist()
    if case["kind"] == "packed":
        do = d64.get("do")
        o, dq = torch.zeros_like(d64["q"]), torch.zeros_like(d64["q"])
        dk, dv, dsink = torch.zeros_like(d64["k"]), torch.zeros_like(d64["v"]), torch.zeros_like(d64["sink"])
        for a, b in zip(cu, cu[1:]):
            for h in range(H):
                j = h // (H // Hkv)
                got = _attend64(d64["q"][a:b, h], d64["k"][a:b, j], d64["v"][a:b, j], d64["sink"][h],
                                None if do is None else do[a:b, h])
                o[a:b, h], dq[a:b, h] = got[0], got[1]
                dk[a:b, j] += got[2]
                dv[a:b, j] += got[3]
                dsink[h] += got[4]
        return [o, dq, dk, dv, dsink] if case["train"] else [o]
    table, kv = s["table"].long(), s["kv"].tolist()
    if case["kind"] == "paged":
        o = torch.zeros_like(d64["q"])
        for i, n in enumerate(kv):
            pages = table[i, :-(-n // case["page"])]
            k, v = (s[t][pages].double().transpose(1, 2).flatten(0, 1)[:n] for t in ("kp", "vp"))
            for h in range(H):
                j = h // (H // Hkv)
                o[cu[i]:cu[i + 1], h] = _attend64(d64["q"][cu[i]:cu[i + 1], h], k[:, j], v[:, j], d64["sink"][h])[0]
        return [o]
    q, kp, vp = torch.zeros_like(d64["q"]), d64["kp"].clone(), d64["vp"].clone()
    half = case["D"] // 2
    for i, n in enumerate(kv):
        rows = slice(cu[i], cu[i + 1])
        pos = torch.arange(n - (cu[i + 1] - cu[i]), n, device=q.device)
        turn = torch.complex(d64["cos"][pos], d64["sin"][pos])[:, None]
        made = []
        for t, gain in (("q", "gq"), ("k", "gk")):
            x = d64[t][rows]
            y = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * d64[gain]
            z = torch.complex(y[..., :half], y[..., half:]) * turn
            made.append(torch.cat([z.real, z.imag], -1))
        q[rows] = made[0]
        at = table[i, pos // case["page"]]
        kp[at, :, pos % case["page"]] = made[1]
        vp[at, :, pos % case["page"]] = d64["v"][rows]
    return [q, kp, vp]
