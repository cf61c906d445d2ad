"""The operators between one token and the next as measurable cases.

An 8-bit paged cache (append, read back, attention), the logits of a step's tokens, drawing
from the algebraic likelihood, and the embedding with its gradient. Each case is one pass on
inputs of the distributions that the model meets. With ``own`` false ``run`` computes the plain
form in elementary torch operations; with ``own`` true it makes the calls a user makes.
``listed`` names the sizes that stand for the range, ``draw`` gives others of the same range,
``exact`` states the maths in 64 bits.

The cache: a token's D values at a key head are stored as e4m3(x 2^-e), with one scale 2^e a
row, e the least whole number for which max |x| 2^-e <= 448.
Attention: scores x = q.k / (sqrt(D) c), weights w = (x + sqrt(1 + x^2))^n, n = 16, c = 8, over
the stored values at or before the query's position, with a sink's weight beside them.
Likelihood: weights (x + sqrt(1 + x^2))^(n / temperature) of x = min(z / c, X), n = 8, c = 2.
"""

import math
import sys
from pathlib import Path

import torch

own = False

N_EXP, C = 16, 8.0
HEAD_N, HEAD_C = 8, 2.0
EPS = 1e-5
E4M3_MAX = 448.0


def listed():
    return [
        # The new tokens' norm, rotation and 8-bit place in the cache, one token a request, and what was stored.
        dict(name="append8_decode", kind="append8", S=64, spread=4.0, kv=40000, chunk=1, H=32, Hkv=8, D=128, page=64),
        # The same for whole prompts.
        dict(name="append8_prompts", kind="append8", S=5, spread=3.0, kv=12000, chunk=1600, H=16, Hkv=16, D=64, page=32),
        # One token for each of a few requests: the smallest serving step.
        dict(name="decode8_small", kind="paged8", S=4, spread=2.0, kv=3600, chunk=1, H=16, Hkv=4, D=128, page=16),
        # One token for each of a full batch.
        dict(name="decode8_batch", kind="paged8", S=64, spread=4.0, kv=200000, chunk=1, H=32, Hkv=8, D=128, page=64),
        # One token of one request over a very long cache: the work has to be split over the keys.
        dict(name="decode8_long", kind="paged8", S=1, spread=1.0, kv=131001, chunk=1, H=16, Hkv=4, D=128, page=128),
        # A chunk of a prompt for each of three requests whose earlier part is in the cache.
        dict(name="chunk8_prefill", kind="paged8", S=3, spread=2.0, kv=24000, chunk=701, H=16, Hkv=4, D=128, page=48),
        # The logits of a small serving step, 1B shape: the table is read for five rows.
        dict(name="logits_step", kind="logits", N=5, d=2048, V=32000, dtype="bf16"),
        # The logits of many tokens, as for the likelihoods of a whole text, 125M shape.
        dict(name="logits_rows", kind="logits", N=509, d=768, V=50257, dtype="bf16"),
        # A token for each request of a full batch, each with settings of its own.
        dict(name="sample_batch", kind="sample", N=64, V=32000, mixed=True, temperature=0.8, top_k=50, top_p=0.95, min_p=0.02),
        # A token for a few requests by mass alone, the larger vocabulary.
        dict(name="sample_few", kind="sample", N=3, V=50257, mixed=False, temperature=0.7, top_k=0, top_p=0.9, min_p=0.0),
        # The embedding of one training microbatch, forward and backward, 1B shape, f32 master weights.
        dict(name="embed_1b_train", kind="embed", N=16384, d=2048, V=32000, table="f32", common=1.0),
        # The same at the 125M shape with bf16 weights and an odd number of tokens.
        dict(name="embed_125m_train", kind="embed", N=8161, d=768, V=50257, table="bf16", common=1.1),
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
    kind = rng.choice(["paged8", "paged8", "paged8", "append8", "logits", "sample", "sample", "embed"])
    if kind == "logits":
        d, V = rng.choice([512, 768, 1000, 1024, 2048]), _logint(rng, 500, 60000)
        dtype = rng.choice(["bf16", "bf16", "f32"])
        N = _logint(rng, 1, 1500 if dtype == "bf16" else 300)
        while N * d * V > 509 * 768 * 50257:
            N = max(1, int(N * 0.8))
            V = int(V * 0.9)
        return dict(kind=kind, N=N, d=d, V=V, dtype=dtype)
    if kind == "sample":
        N, V = _logint(rng, 1, 256), _logint(rng, 200, 130000)
        while N * V > 64 * 32000:
            N = int(N * 0.8)
        return dict(kind=kind, N=N, V=V, mixed=rng.random() < 0.5, temperature=rng.choice([0.0, 0.6, 1.0, 1.0, 1.3]),
                    top_k=rng.choice([0, 0, 1, _logint(rng, 2, 2000)]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]),
                    min_p=rng.choice([0.0, 0.0, 0.01, 0.2]))
    if kind == "embed":
        d, V = _logint(rng, 64, 4096, 8), _logint(rng, 100, 60000)
        N = _logint(rng, 1, 20000)
        while N * d + V * d > (16384 + 32000) * 2048 or N * d > 16384 * 2048:
            N, V = max(1, int(N * 0.8)), int(V * 0.8)
        return dict(kind=kind, N=N, d=d, V=V, table=rng.choice(["f32", "bf16"]), common=rng.choice([0.0, 0.8, 1.0, 1.2]))
    spread = round(math.exp(rng.uniform(0.0, math.log(8.0))), 2)
    H, Hkv = _heads(rng)
    D = rng.choice([64, 128])
    S = _logint(rng, 1, 64)
    page = rng.choice([16, 32, 48, 64, 128])
    chunk = 1 if kind == "paged8" and rng.random() < 0.5 else _logint(rng, 1, 900 if kind == "paged8" else 1600)
    while S * chunk > 8000:
        S = max(1, S // 2)
    least = S * (chunk + 8) * 4
    kv = _logint(rng, least, max(least + 1, 200000 if kind == "paged8" else 40000))
    if kind == "paged8":
        while kv > least and (S * H * chunk * max(lens(kv, S, spread)) > 1.2e9 or S * Hkv * D * max(lens(kv, S, spread)) > 3e8):
            kv = max(least, int(kv * 0.8))
    return dict(kind=kind, S=S, spread=spread, kv=kv, chunk=chunk, H=H, Hkv=Hkv, D=D, page=page)


def lens(total, S, spread):
    """`total` in S parts, the largest about `spread` times the smallest, large and small in turn."""
    w = [spread ** (i / max(1, S - 1)) for i in range(S)]
    w = w[::2] + w[1::2][::-1]
    got = [max(1, int(total * x / sum(w))) for x in w]
    got[0] += max(0, total - sum(got))
    return got


def _new(case):
    """The new tokens of each request: the last `chunk` of its keys, an eighth fewer or more."""
    kv, chunk = lens(case["kv"], case["S"], case["spread"]), case["chunk"]
    return kv, [1 if chunk == 1 else min(n, max(1, chunk + (i % 3 - 1) * (chunk // 8))) for i, n in enumerate(kv)]


# --- inputs ---------------------------------------------------------------------------------

def _normed(x):
    return x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()


def _scale_bits(x):
    """The exponent e of a row's scale, as a float's bits: (e + 127) << 23."""
    bits = x.abs().amax(-1).contiguous().view(torch.int32)
    over = (bits & 0x7FFFFF) > 0x600000  # the mantissa passes 1.75
    e = ((bits >> 23) - 8 + over.int()).clamp(min=1)
    return torch.where(bits == 0, 127, e) << 23


def _in_8_bits(x):
    """Rows of `x` (f32) as e4m3 bytes and e8m0 scales, both as uint8."""
    bits = _scale_bits(x)
    return (x / bits.view(torch.float32)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), (bits >> 23).to(torch.uint8)


def _values(x8, scale):
    """The f32 values that bytes and their rows' scales stand for."""
    return x8.view(torch.float8_e4m3fn).float() * (scale.int() << 23).view(torch.float32)[..., None]


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))

    def rn(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32)

    def ru(*shape):
        return torch.rand(*shape, device=dev, generator=g, dtype=torch.float32)

    bf, kind = torch.bfloat16, case["kind"]
    s = {"case": case}
    if kind == "logits":  # normed hidden states, a table whose logits spread over about +-2
        dtype = bf if case["dtype"] == "bf16" else torch.float32
        s["h"] = _normed(rn(case["N"], case["d"])).to(dtype)
        s["embed"] = (2.0 / math.sqrt(case["d"]) * rn(case["V"], case["d"])).to(dtype)
        return s
    if kind == "sample":  # a few dozen likely tokens over a broad tail
        N, V = case["N"], case["V"]
        s["z"] = 2.0 * rn(N, V) + 12.0 * ru(N, V).pow(400.0)
        s["u"] = ru(N)
        for name in ("temperature", "top_k", "top_p", "min_p"):
            s[name] = case[name]
        if case["mixed"]:  # settings of their own, every fourth row's switched off, row by row another one
            row = torch.arange(N, device=dev)
            s["temperature"] = torch.where(row % 4 == 0, 1.0, case["temperature"] * (0.75 + 0.5 * ru(N)))
            s["top_k"] = torch.where(row % 4 == 1, 0, case["top_k"] + (row % 7)).to(torch.int32)
            s["top_p"] = torch.where(row % 4 == 2, 1.0, case["top_p"] - 0.1 * ru(N))
            s["min_p"] = torch.where(row % 4 == 3, 0.0, case["min_p"] * (0.5 + ru(N)))
        return s
    if kind == "embed":  # tokens as common as words: the k-th at about k^-common
        N, d, V = case["N"], case["d"], case["V"]
        often = (torch.arange(V, device=dev, dtype=torch.float64) + 2.7).pow(-case["common"]).cumsum(0)
        rank = torch.searchsorted(often, ru(N).double() * often[-1]).clamp(max=V - 1)
        s["tokens"] = torch.randperm(V, device=dev, generator=g)[rank]
        s["embed"] = (0.02 * rn(V, d)).to(torch.float32 if case["table"] == "f32" else bf).requires_grad_(True)
        s["dy"] = rn(N, d).to(bf)
        s["scale"] = math.sqrt(d)
        return s
    # A cache of pages in a shuffled order, more of them than the requests use.
    S, page, H, Hkv, D = case["S"], case["page"], case["H"], case["Hkv"], case["D"]
    kv, new = _new(case)
    need = [-(-n // page) for n in kv]
    width, pages, N = max(need), sum(need) + 5, sum(new)
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    table = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s.update(longest=max(kv), chunk=max(new), table=table, cu=_i32([sum(new[:i]) for i in range(S + 1)], dev), kv=_i32(kv, dev), N=N)
    if kind == "paged8":
        s["q"] = _normed(rn(N, H, D)).to(bf)
        (k8, ks), (v8, vs) = _in_8_bits(_normed(rn(pages, Hkv, page, D))), _in_8_bits(rn(pages, Hkv, page, D))
        s["sink"] = 0.1 * rn(H)
    else:
        k8, v8 = (torch.zeros(pages, Hkv, page, D, dtype=torch.uint8, device=dev) for _ in range(2))
        ks, vs = (torch.full((pages, Hkv, page), 127, dtype=torch.uint8, device=dev) for _ in range(2))
        for name, heads in (("q", H), ("k", Hkv), ("v", Hkv)):
            s[name] = (1.5 * rn(N, heads, D)).to(bf)
        s["gq"], s["gk"] = 1 + 0.1 * rn(D), 1 + 0.1 * rn(D)
        half = D // 2
        w = 0.5 * 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        angle = 2 * torch.arange(width * page, device=dev, dtype=torch.float64)[:, None] * torch.atan(w)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["kp"], s["vp"] = k8.view(torch.float8_e4m3fn), v8.view(torch.float8_e4m3fn)
    s["ks"], s["vs"] = ks.view(torch.float8_e8m0fnu), vs.view(torch.float8_e8m0fnu)
    return s


# --- one pass --------------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    pkg = str(Path.cwd() / "algebraic-transformer_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import algebraic_amd as A

    kind = s["case"]["kind"]
    if kind == "logits":
        return [A.head_logits(s["h"], s["embed"])]
    if kind == "sample":
        return list(A.head_sample(s["z"], s["u"], n=HEAD_N, c=HEAD_C, temperature=s["temperature"], top_k=s["top_k"],
                                  top_p=s["top_p"], min_p=s["min_p"]))
    if kind == "embed":
        y = A.token_embedding(s["tokens"], s["embed"], scale=s["scale"], dtype=torch.bfloat16)
        return [y, torch.autograd.grad(y, s["embed"], s["dy"])[0]]
    cache = (s["kp"], s["vp"], s["ks"], s["vs"], s["table"], s["cu"], s["kv"])
    if kind == "paged8":
        return [A.paged_flash_attention_fp8(s["q"], *cache, s["sink"], n=N_EXP, c=C)]
    q = A.paged_append_fp8(s["q"], s["k"], s["v"], *cache, s["gq"], s["gk"], s["cos"], s["sin"], eps=EPS)
    return [q, *A.paged_read_fp8(*cache, tokens=s["N"])]


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "logits":
        return [s["h"].float() @ s["embed"].float().T]
    if kind == "sample":
        return _plain_sample(s)
    if kind == "embed":
        table = s["embed"].detach()
        y = (table[s["tokens"]].float() * s["scale"]).to(torch.bfloat16)
        grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
        grad.index_add_(0, s["tokens"], s["dy"].float())
        return [y, grad.mul_(s["scale"]).to(table.dtype)]
    return _plain_paged(s) if kind == "paged8" else _plain_append(s)


def _plain_sample(s):
    N, V = s["z"].shape
    z = s["z"]

    def per_row(x):
        return torch.as_tensor(x, device=z.device).double().expand(N)[:, None]

    T, k, top_p, min_p = (per_row(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    x = (z.double() / HEAD_C).clamp(max=0.25 * (1e38 / V) ** (1.0 / HEAD_N))
    x, order = x.sort(dim=-1, descending=True, stable=True)  # equal ones by their index
    a = HEAD_N * torch.asinh(x)
    w = torch.exp((a - a[:, :1]) / torch.where(T > 0, T, 1.0))
    rank = torch.arange(V, device=z.device)
    w = torch.where((rank < torch.where(k > 0, k, V)) & ((T > 0) | (rank == 0)), w, 0.0)
    mass = w.cumsum(-1)
    w = torch.where(((mass - w < top_p * mass[:, -1:]) | (top_p >= 1) | (rank == 0)) & (w >= min_p), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # back to the vocabulary's order
    mass = w.cumsum(-1)
    token = (mass <= s["u"].double()[:, None] * mass[:, -1:]).sum(-1)
    return [token, torch.log(w.gather(1, token[:, None])[:, 0] / mass[:, -1]).float()]


def _padded(rows, cu, longest):
    """(S, longest, ...) of packed rows, and which of its places hold a row."""
    t = torch.arange(longest, device=cu.device)
    live = t < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + t).clamp(max=rows.shape[0] - 1).long()
    return torch.where(live[..., None, None], rows[at].float(), 0.0), live


def _plain_paged(s):
    case = s["case"]
    H, Hkv, D, page = case["H"], case["Hkv"], case["D"], case["page"]
    G = H // Hkv
    cu, kv = s["cu"].long(), s["kv"].long()
    qp, live = _padded(s["q"], cu, s["chunk"])
    q = qp.unflatten(2, (Hkv, G)).permute(0, 2, 3, 1, 4)  # (S, Hkv, G, L, D)
    t = torch.arange(s["longest"], device=cu.device)
    at = s["table"].long()[:, t // page].clamp(min=0)
    held = (t < kv[:, None])[:, :, None, None]

    def key_heads(pages, scales):  # (S, Hkv, 1, K, D)
        x = _values(pages.view(torch.uint8)[at, :, t % page], scales.view(torch.uint8)[at, :, t % page])
        return torch.where(held, x, 0.0).permute(0, 2, 1, 3).unsqueeze(2)

    k, v = key_heads(s["kp"], s["ks"]), key_heads(s["vp"], s["vs"])
    pos = (kv - (cu[1:] - cu[:-1]))[:, None] + torch.arange(s["chunk"], device=cu.device)
    dead = (torch.arange(k.shape[3], device=cu.device) > pos[..., None])[:, None, None]
    x = (q @ k.transpose(-1, -2)) * (1.0 / (math.sqrt(D) * C))
    a = (N_EXP * torch.asinh(x)).masked_fill_(dead, -math.inf)
    ab = N_EXP * torch.asinh(s["sink"].float().view(Hkv, G, 1, 1) / C)
    m = torch.maximum(a.amax(-1, keepdim=True), ab)
    w = a.sub_(m).exp_()
    o = (w @ v) / (w.sum(-1, keepdim=True) + (ab - m).exp())
    return [o.permute(0, 3, 1, 2, 4).flatten(2, 3)[live].to(torch.bfloat16)]


def _plain_append(s):
    bf, page = torch.bfloat16, s["case"]["page"]
    cu, kv = s["cu"].long(), s["kv"].long()
    new = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(len(kv), device=cu.device), new, output_size=s["N"])
    pos = torch.arange(s["N"], device=cu.device) - cu[seq] + (kv - new)[seq]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(x, gain):
        a, b = (_normed(x.float()) * gain).chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    at = s["table"].long()[seq, pos // page]
    out = [turned(s["q"], s["gq"]).to(bf)]
    for pages, scales, x in (("kp", "ks", turned(s["k"], s["gk"])), ("vp", "vs", s["v"].float())):
        bytes_, scale = s[pages].view(torch.uint8), s[scales].view(torch.uint8)
        bytes_[at, :, pos % page], scale[at, :, pos % page] = _in_8_bits(x)
        out.append(_values(bytes_[at, :, pos % page], scale[at, :, pos % page]).to(bf))
    return out


# --- what a pass cannot do without ----------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "logits":
        N, d, V = case["N"], case["d"], case["V"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": (N * d + V * d) * size + N * V * 4, "flops": 2.0 * N * d * V}
    if kind == "sample":
        return {"bytes": case["N"] * (case["V"] * 4 + 16), "flops": 16.0 * case["N"] * case["V"]}
    if kind == "embed":  # the tokens' rows in and out, their gradients in, the table's gradient out
        N, d, V = case["N"], case["d"], case["V"]
        size = 4 if case["table"] == "f32" else 2
        return {"bytes": N * 8 + min(N, V) * d * size + 2 * N * d * 2 + V * d * size, "flops": 3.0 * N * d}
    H, Hkv, D, page = case["H"], case["Hkv"], case["D"], case["page"]
    kv, new = _new(case)
    if kind == "append8":  # q in and out, k and v in, their bytes out and in again, the values out
        return {"bytes": sum(new) * (2 * H * D * 2 + 2 * Hkv * (2 * D + 2 * (D + 1) + 2 * D) + D * 4), "flops": 14.0 * sum(new) * (H + Hkv) * D}
    scores = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(new, kv)) * H
    return {"bytes": sum(kv) * Hkv * (2 * D + 2) + sum(new) * H * D * 4 + sum(-(-n // page) for n in kv) * 4,
            "flops": 4.0 * scores * D}


# --- the same maths in 64 bits ---------------------------------------------------------------

def _stored64(x):
    """What an 8-bit row of float64 values stands for."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / E4M3_MAX)).clamp(min=-126)
    unit = torch.ldexp(torch.ones_like(top), e.int())
    return torch.where(top > 0, (x / unit).to(torch.float8_e4m3fn).double() * unit, 0.0)


def _attend64(q, k, v, sink):
    """One head's queries, the last of q.shape[0] positions of k."""
    o, D, first = torch.empty_like(q), q.shape[1], k.shape[0] - q.shape[0]
    for a in range(0, q.shape[0], 2048):
        b = min(a + 2048, q.shape[0])
        x = q[a:b] @ k[:first + b].T / (math.sqrt(D) * C)
        logw = torch.log(torch.hypot(x, torch.ones_like(x)) + x.abs()) * x.sign() * N_EXP
        pos = torch.arange(first + a, first + b, device=q.device)[:, None]
        logw[torch.arange(first + b, device=q.device)[None] > pos] = -math.inf
        logw = torch.cat([logw, (N_EXP * torch.asinh(sink / C)).expand(b - a, 1)], 1)
        o[a:b] = torch.softmax(logw, 1)[:, :-1] @ v[:first + b]
    return o


def _draw64(z, u, T, k, top_p, min_p):
    """One row's token and its log-probability, by its tokens in falling order."""
    V = z.shape[0]
    x = torch.minimum(z.double() / HEAD_C, torch.tensor(0.25 * (1e38 / V) ** (1.0 / HEAD_N), dtype=torch.float64))
    order = torch.argsort(-x, stable=True)
    if T == 0:
        return int(order[0]), 0.0
    logw = torch.log(torch.hypot(x, torch.ones_like(x)) + x.abs()) * x.sign() * HEAD_N / T
    w = torch.exp(logw - logw[order[0]])
    kept = order[:k] if 0 < k < V else order
    if top_p < 1:
        part = torch.cumsum(w[kept], 0) / w[kept].sum()
        kept = kept[:int((part < top_p).sum()) + 1]
    kept = kept[w[kept] >= min_p].sort().values
    part = torch.cumsum(w[kept], 0)
    i = min(int((part <= u * part[-1]).sum()), len(kept) - 1)
    return int(kept[i]), float(torch.log(w[kept[i]] / part[-1]))


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "logits":
        h, rows = s["h"].double(), []
        for a in range(0, case["V"], 8192):
            rows.append(h @ s["embed"][a:a + 8192].double().T)
        return [torch.cat(rows, 1)]
    if kind == "sample":
        N = case["N"]
        names = ("temperature", "top_k", "top_p", "min_p")
        T, k, top_p, min_p = ([float(y) for y in x.cpu()] if torch.is_tensor(x) else [x] * N for x in (s[m] for m in names))
        z, u = s["z"].cpu(), s["u"].cpu().double()
        got = [_draw64(z[i], float(u[i]), T[i], int(k[i]), top_p[i], min_p[i]) for i in range(N)]
        return [torch.tensor([t for t, _ in got]), torch.tensor([p for _, p in got], dtype=torch.float64)]
    if kind == "embed":
        table, tokens, dy = s["embed"].detach(), s["tokens"], s["dy"]
        y = table[tokens].double() * s["scale"]
        order = tokens.argsort(stable=True)
        ids, count = tokens[order].unique_consecutive(return_counts=True)
        total = torch.cat([torch.zeros(1, case["d"], dtype=torch.float64, device=dy.device), dy[order].double().cumsum(0)])
        end = count.cumsum(0)
        grad = torch.zeros(table.shape, dtype=torch.float64, device=dy.device)
        grad[ids] = (total[end] - total[end - count]) * s["scale"]
        return [y, grad]
    H, Hkv, D, page = case["H"], case["Hkv"], case["D"], case["page"]
    cu, kv, table = s["cu"].tolist(), s["kv"].tolist(), s["table"].long()
    if kind == "paged8":
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        for i, n in enumerate(kv):
            pages = table[i, :-(-n // page)]
            k, v = ((s[t].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
                     * torch.exp2(s[r].view(torch.uint8)[pages].double() - 127)[..., None]).transpose(1, 2).flatten(0, 1)[:n]
                    for t, r in (("kp", "ks"), ("vp", "vs")))
            for h in range(H):
                j = h // (H // Hkv)
                o[cu[i]:cu[i + 1], h] = _attend64(s["q"][cu[i]:cu[i + 1], h].double(), k[:, j], v[:, j], s["sink"][h].double())
        return [o]
    q, k, v = (s[t].double() for t in "qkv")
    half = D // 2
    for i, n in enumerate(kv):
        rows = slice(cu[i], cu[i + 1])
        pos = torch.arange(n - (cu[i + 1] - cu[i]), n, device=q.device)
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        for t, gain in ((q, "gq"), (k, "gk")):
            y = t[rows] / (t[rows].pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s[gain].double()
            z = torch.complex(y[..., :half], y[..., half:]) * turn
            t[rows] = torch.cat([z.real, z.imag], -1)
    return [q, _stored64(k), _stored64(v)]
