"""Timed cases of the long-context attention operators: heads normalised, rotated and appended to a cache
(``norm_rope_append``), rows appended to a cache held in 4 bits and read back (``Cache4.append`` / ``read``),
attention over such a cache (``Cache4.attention``), and attention with a sliding window and first tokens that stay
visible over f16 and f32 caches (``attention_window``).

``own`` chooses between the plain forms (elementary torch operations) and the framework's operators."""
import math

import torch

own = False

DEV = "cuda"
GROUP = 32                              # values that share a scale in the 4-bit cache
NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]      # element of an eight-value word held by its nibble 0, 1, ...


# ------------------------------------------------------------------------------------------- the cases
def listed():
    def rotate(name, n, heads, kv, hd, dtype, norm, start, max_seq):
        return dict(name=name, op="rotate", n=n, heads=heads, kv_heads=kv, hd=hd, dtype=dtype, norm=norm, start=start, max_seq=max_seq)

    def append(name, n, kv, hd, dtype, start, max_seq):
        return dict(name=name, op="append", n=n, kv_heads=kv, hd=hd, dtype=dtype, start=start, max_seq=max_seq)

    def attend(name, n, heads, kv, hd, dtype, start, max_seq, window, sinks):
        return dict(name=name, op="attend", n=n, heads=heads, kv_heads=kv, hd=hd, dtype=dtype, start=start, max_seq=max_seq, window=window, sinks=sinks)

    return [
        # one generated token of the 7B shape, at the end of its 384 positions
        rotate("rotate token 7b", 1, 32, 32, 128, "f16", True, 383, 384),
        # the 65B shape's 1792-token prompt
        rotate("rotate prompt 65b", 1792, 64, 64, 128, "f16", True, 0, 2048),
        # a chunk in the middle of a text, f32 cache, narrow heads, four query heads to a K/V head, rotation only
        rotate("rotate chunk f32", 333, 52, 13, 64, "f32", False, 1000, 2048),
        # one generated token of the 13B shape into the 4-bit cache
        append("append4 token 13b", 1, 40, 128, "f32", 639, 640),
        # the 65B shape's prompt into the 4-bit cache
        append("append4 prompt 65b", 1792, 64, 128, "f32", 0, 2048),
        # one generated token of the 7B shape over its whole short cache: latency
        attend("attend4 token 7b", 1, 32, 32, 128, "q4", 383, 384, 384, 0),
        # one token at the end of a long text: the bytes of the cache
        attend("attend4 token long", 1, 32, 32, 128, "q4", 65535, 65536, 65536, 0),
        # a prompt's later chunk over everything before it, 13B shape
        attend("attend4 chunk 13b", 512, 40, 40, 128, "q4", 7680, 8192, 8192, 0),
        # one token far into a stream: a wide window, four first tokens, eight query heads to a K/V head
        attend("window token shared", 1, 64, 8, 128, "f16", 131071, 131072, 16384, 4),
        # a prompt of the 65B shape with a window narrower than the prompt
        attend("window prompt 65b", 1792, 64, 64, 128, "f16", 0, 2048, 512, 4),
        # an odd chunk of the small f32 shape
        attend("window chunk f32", 77, 8, 4, 64, "f32", 300, 400, 100, 3),
        # a long prompt with shared heads: arithmetic
        attend("window prompt long", 8192, 32, 8, 128, "f16", 0, 8192, 2048, 16),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    hd = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 3, 4, 5, 8, 8, 13, 16, 32, 40, 52, 64])
    group = rng.choice([g for g in (1, 1, 1, 2, 3, 4, 5, 8, 16) if g * kv <= 64])
    op = rng.choice(["rotate", "append", "attend", "attend", "attend"])
    if op == "rotate":
        n, start = _log_uniform(rng, 1, 1792), _log_uniform(rng, 1, 30000) - 1
        return dict(op=op, n=n, heads=kv * group, kv_heads=kv, hd=hd, dtype=rng.choice(["f16", "f32"]), norm=rng.random() < 0.6, start=start,
                    max_seq=start + n + rng.randrange(0, 40))
    if op == "append":
        n, start = _log_uniform(rng, 1, 1792), _log_uniform(rng, 1, 30000) - 1
        return dict(op=op, n=n, kv_heads=kv, hd=hd, dtype=rng.choice(["f16", "f32"]), start=start, max_seq=start + n + rng.randrange(0, 40))
    dtype = rng.choice(["q4", "q4", "f16", "f16", "f32"])
    n = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 400 if dtype == "f32" else 4096)
    # no more scores in the plain form than a quarter of the largest listed case's, and no larger a cache
    most = max(n + 1, min(131072 if n == 1 else 16384, 500_000_000 // (kv * group * n), 400_000_000 // (kv * hd)))
    total = _log_uniform(rng, n, most)
    window = rng.choice([total, _log_uniform(rng, 1, total), _log_uniform(rng, 1, total)])
    return dict(op=op, n=n, heads=kv * group, kv_heads=kv, hd=hd, dtype=dtype, start=total - n, max_seq=total + rng.randrange(0, 40), window=window,
                sinks=rng.choice([0, 0, 1, 4, 16, 100]))


def _visible_pairs(c):
    """(row, position) pairs that are visible, and the positions that some row sees."""
    p = torch.arange(c["start"], c["start"] + c["n"], dtype=torch.float64)
    lo = (p + 1 - c["window"]).clamp(min=0)
    pairs = (p + 1 - lo + lo.clamp(max=c["sinks"])).sum().item()
    first = max(0, c["start"] + 1 - c["window"])
    return pairs, c["start"] + c["n"] - first + min(c["sinks"], first)


def _row_bytes(c):
    return {"f16": 2.0, "f32": 4.0, "q4": 0.5 + 2.0 / GROUP}[c["dtype"]] * c["hd"]


def work(case):
    c = case
    if c["op"] == "rotate":
        q, kv = c["n"] * c["heads"] * c["hd"], c["n"] * c["kv_heads"] * c["hd"]
        return {"bytes": q * 8.0 + kv * 8.0 + 2 * c["n"] * c["kv_heads"] * _row_bytes(c) + c["n"] * c["hd"] * 4.0, "flops": 7.0 * (q + kv)}
    if c["op"] == "append":
        kv = 2 * c["n"] * c["kv_heads"] * c["hd"]
        return {"bytes": kv * ((4 if c["dtype"] == "f32" else 2) + 2 + 2 * (0.5 + 2.0 / GROUP)), "flops": 4.0 * kv}
    pairs, positions = _visible_pairs(c)
    rows = c["n"] * c["heads"] * c["hd"]
    return {"bytes": 2.0 * positions * c["kv_heads"] * _row_bytes(c) + rows * (8 if c["dtype"] == "f32" else 6), "flops": 4.0 * pairs * c["heads"] * c["hd"]}


# ------------------------------------------------------------------------------------------- inputs
def _rope_table(max_seq, hd):
    freq = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    angle = torch.arange(max_seq, dtype=torch.float64, device=DEV)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=-1).reshape(max_seq, hd).float()


def _scales(x):
    """The 4-bit cache's scale of each group of 32 values: 8 significant bits, so that scale * code is an f16 value."""
    top = x.reshape(*x.shape[:-1], -1, GROUP).abs().amax(-1).clamp(max=65504.0)
    return (top * (1.0 / 7.0)).to(torch.bfloat16).to(torch.float16)


def _codes(x, scale):
    d = scale.float().repeat_interleave(GROUP, -1)
    return torch.where(d > 0, (x / torch.where(d > 0, d, torch.ones_like(d))).clamp(-7, 7).round(), torch.zeros_like(x))


def _pack(codes):
    """Codes -7..7 as nibbles code + 8, words of eight in the cache's order."""
    *lead, hd = codes.shape
    words = (codes + 8).to(torch.uint8).reshape(*lead, hd // GROUP, 4, 8).transpose(-3, -2)[..., NIBBLES]
    return (words[..., 0::2] | (words[..., 1::2] << 4)).reshape(*lead, hd // 2)


def _unpack(packed, scale):
    *lead, half = packed.shape
    nib = torch.stack([packed & 15, packed >> 4], dim=-1).reshape(*lead, 4, 2 * half // GROUP, 8)
    at = torch.tensor([NIBBLES.index(e) for e in range(8)], device=packed.device)
    codes = nib[..., at].transpose(-3, -2).reshape(*lead, 2 * half).float() - 8
    return codes * scale.float().repeat_interleave(GROUP, -1)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * scale

    n, kv, hd, max_seq = c["n"], c["kv_heads"], c["hd"], c["max_seq"]
    s = dict(c)
    ctype = torch.float32 if c["dtype"] == "f32" else torch.float16
    if c["op"] == "rotate":
        s["q"], s["k"], s["v"] = normal(n, c["heads"] * hd), normal(n, kv * hd), normal(n, kv * hd)
        if c["norm"]:
            s["q"] *= 3.0
            s["q_gain"], s["k_gain"] = 1 + normal(1, hd, scale=0.1), 1 + normal(1, hd, scale=0.1)
        s["table"] = _rope_table(max_seq, hd)
        s["kcache"], s["vcache"] = torch.zeros(kv * max_seq, hd, dtype=ctype, device=DEV), torch.zeros(kv * max_seq, hd, dtype=ctype, device=DEV)
        s["q_out"] = torch.empty_like(s["q"])
    elif c["op"] == "append":
        s["k"], s["v"] = normal(n, kv * hd).to(ctype), normal(n, kv * hd, scale=0.5).to(ctype)
        s["parts"] = [torch.zeros(kv * max_seq, w, dtype=t, device=DEV) for t, w in ((torch.uint8, hd // 2), (torch.float16, hd // GROUP)) * 2]
        s["k_out"], s["v_out"] = (torch.empty(n, kv * hd, dtype=torch.float16, device=DEV) for _ in range(2))
    else:
        s["q"] = normal(n, c["heads"] * hd, scale=1.5)
        s["out"] = torch.empty(n, c["heads"] * hd, dtype=ctype, device=DEV)
        if c["dtype"] == "q4":
            s["parts"] = []
            for _ in range(2):
                x = normal(kv * max_seq, hd)
                d = _scales(x)
                s["parts"] += [_pack(_codes(x, d)), d]
        else:
            s["kcache"], s["vcache"] = normal(kv * max_seq, hd).to(ctype), normal(kv * max_seq, hd).to(ctype)
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _plain_rotate(s):
    n, kv, hd, start = s["n"], s["kv_heads"], s["hd"], s["start"]
    f = s["table"][start:start + n].reshape(n, 1, hd // 2, 2)

    def turn(x, gain):
        x = x.reshape(n, -1, hd)
        if gain is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain
        x = x.reshape(n, -1, hd // 2, 2)
        a, b = x[..., 0], x[..., 1]
        return torch.stack([a * f[..., 0] - b * f[..., 1], a * f[..., 1] + b * f[..., 0]], dim=-1).reshape(n, -1, hd)

    s["q_out"].copy_(turn(s["q"], s.get("q_gain")).reshape(n, -1))
    s["kcache"].view(kv, -1, hd)[:, start:start + n] = turn(s["k"], s.get("k_gain")).transpose(0, 1).to(s["kcache"].dtype)
    s["vcache"].view(kv, -1, hd)[:, start:start + n] = s["v"].reshape(n, kv, hd).transpose(0, 1).to(s["vcache"].dtype)
    return s["q_out"], s["kcache"], s["vcache"]


def _plain_append(s):
    n, kv, hd, start = s["n"], s["kv_heads"], s["hd"], s["start"]

    def through(x, packed, scales):
        x = x.float().reshape(n, kv, hd).transpose(0, 1)
        d = _scales(x)
        packed.view(kv, -1, hd // 2)[:, start:start + n] = _pack(_codes(x, d))
        scales.view(kv, -1, hd // GROUP)[:, start:start + n] = d
        back = _unpack(packed.view(kv, -1, hd // 2)[:, start:start + n], scales.view(kv, -1, hd // GROUP)[:, start:start + n])
        return back.transpose(0, 1).reshape(n, kv * hd).half()

    kp, ks, vp, vs = s["parts"]
    return through(s["k"], kp, ks), through(s["v"], vp, vs)


def _plain_attend(s):
    n, kv, hd, start = s["n"], s["kv_heads"], s["hd"], s["start"]
    group, total = s["heads"] // kv, start + n
    first = max(0, start + 1 - s["window"])  # the positions that some row sees: the first ones and these onwards
    whole = [x.view(kv, s["max_seq"], -1) for x in (s["parts"] if s["dtype"] == "q4" else (s["kcache"], s["vcache"]))]
    parts, at = [x[:, first:total] for x in whole], torch.arange(first, total, device=DEV)
    kept = min(s["sinks"], first)
    if kept:
        parts = [torch.cat([w[:, :kept], x], 1) for w, x in zip(whole, parts)]
        at = torch.cat([torch.arange(kept, device=DEV), at])
    k, v = (_unpack(*parts[:2]), _unpack(*parts[2:])) if s["dtype"] == "q4" else (parts[0].float(), parts[1].float())
    q = s["q"].reshape(n, kv, group, hd).permute(1, 2, 0, 3).reshape(kv, group * n, hd)
    scores = (q @ k.transpose(1, 2)).mul_(1 / math.sqrt(hd)).view(kv, group, n, len(at))
    row = torch.arange(start, total, device=DEV)[:, None]
    scores.masked_fill_((at > row) | ((at <= row - s["window"]) & (at >= s["sinks"])), -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    sums = p.sum(-1, keepdim=True)
    out = (p.view(kv, group * n, len(at)) @ v).view(kv, group, n, hd) / torch.where(sums > 0, sums, torch.ones_like(sums))
    return out.permute(2, 0, 1, 3).reshape(n, -1).to(s["out"].dtype)


# ------------------------------------------------------------------------------------------- the framework's operators
_cuda = None


def _handles(s):
    """The library's views of the state's tensors, made once, as a program that keeps its tensors does."""
    global _cuda
    import rllama_b200 as R
    if _cuda is None:
        _cuda = R.Cuda(stream=torch.cuda.current_stream().cuda_stream)
    h = {k: _cuda.wrap(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if "parts" in s:
        h["cache"] = R.Cache4.wrap(_cuda, *s["parts"], s["kv_heads"], s["max_seq"], s["hd"])
    s["handles"] = h
    return h


def _own_run(s):
    h = s.get("handles") or _handles(s)
    if s["op"] == "rotate":
        h["q_out"].norm_rope_append(h["kcache"], h["vcache"], h["q"], h["k"], h["v"], h["table"], s["heads"], s["kv_heads"], s["max_seq"], s["start"],
                                    h.get("q_gain"), h.get("k_gain"), 1e-6)
        return s["q_out"], s["kcache"], s["vcache"]
    if s["op"] == "append":
        h["cache"].append(h["k"], h["v"], s["start"])
        h["cache"].read(h["k_out"], h["v_out"], s["start"])
        return s["k_out"], s["v_out"]
    if s["dtype"] == "q4":
        h["cache"].attention(h["out"], h["q"], s["heads"], s["start"], s["window"], s["sinks"])
    else:
        h["out"].attention_window(h["q"], h["kcache"], h["vcache"], s["heads"], s["kv_heads"], s["max_seq"], s["start"], s["window"], s["sinks"])
    return s["out"]


def run(state):
    if own:
        return _own_run(state)
    return {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend}[state["op"]](state)


# ------------------------------------------------------------------------------------------- 64 bits
def _exact_values(x):
    """What the 4-bit cache holds of rows x (rows, hd): each group's largest magnitude over 7, to 8 significant bits and f16's
    range, times the nearest whole number of steps."""
    g = x.double().reshape(x.shape[0], -1, GROUP)
    d = (g.abs().amax(-1, keepdim=True).clamp(max=65504.0) / 7)
    mant, exp = torch.frexp(d)
    d = torch.ldexp((mant * 256).round(), exp - 8)
    d = torch.where(d < 2.0 ** -14, (d * 2.0 ** 24).round() * 2.0 ** -24, d)
    steps = torch.where(d > 0, (g / d.clamp(min=2.0 ** -60)).clamp(-7, 7).round(), torch.zeros_like(g))
    return (steps * d).reshape(x.shape)


def _exact_cached(packed, scales, hd):
    """Values of packed rows (rows, hd / 2), one value position at a time."""
    out = torch.empty(packed.shape[0], hd, dtype=torch.float64, device=packed.device)
    groups = hd // GROUP
    for e in range(hd):
        word = (e % GROUP) // 8 * groups + e // GROUP
        nibble = NIBBLES.index(e % 8)
        byte = packed[:, word * 4 + nibble // 2].long()
        out[:, e] = ((byte // 16 if nibble % 2 else byte % 16) - 8) * scales[:, e // GROUP].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    n, kv, hd, start = s["n"], s["kv_heads"], s["hd"], s["start"]
    if s["op"] == "rotate":
        pos = torch.arange(start, start + n, dtype=torch.float64, device=DEV)[:, None, None]
        angle = pos / 10000.0 ** (torch.arange(hd // 2, dtype=torch.float64, device=DEV) * 2 / hd)
        turn = torch.polar(torch.ones_like(angle), angle)

        def through(x, gain):
            x = x.double().view(n, -1, hd)
            if gain is not None:
                x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / hd + 1e-6) * gain.double()
            return torch.view_as_real(torch.view_as_complex(x.reshape(n, -1, hd // 2, 2).contiguous()) * turn).reshape(n, -1, hd)

        kc, vc = s["kcache"].double(), s["vcache"].double()
        k, v = through(s["k"], s.get("k_gain")), s["v"].double().view(n, kv, hd)
        for h in range(kv):
            kc[h * s["max_seq"] + start:][:n] = k[:, h]
            vc[h * s["max_seq"] + start:][:n] = v[:, h]
        return through(s["q"], s.get("q_gain")).reshape(n, -1), kc, vc
    if s["op"] == "append":
        return tuple(_exact_values(s[x].reshape(n * kv, hd)).reshape(n, kv * hd) for x in ("k", "v"))
    group, total = s["heads"] // kv, start + n
    row = torch.arange(start, total, device=DEV)[:, None]
    at = torch.arange(total, device=DEV)[None]
    seen = (at <= row) & ((at > row - s["window"]) | (at < s["sinks"]))
    out = torch.zeros(n, s["heads"], hd, dtype=torch.float64, device=DEV)
    for h in range(kv):
        rows = slice(h * s["max_seq"], h * s["max_seq"] + total)
        if s["dtype"] == "q4":
            kp, ks, vp, vs = (x[rows] for x in s["parts"])
            k, v = _exact_cached(kp, ks, hd), _exact_cached(vp, vs, hd)
        else:
            k, v = s["kcache"][rows].double(), s["vcache"][rows].double()
        for j in range(h * group, (h + 1) * group):
            scores = torch.where(seen, s["q"][:, j * hd:(j + 1) * hd].double() @ k.T / math.sqrt(hd), -math.inf)
            out[:, j] = torch.nan_to_num(torch.softmax(scores, -1), nan=0.0) @ v
    return out.reshape(n, -1)
