"""Performance cases of the low-precision serving operators: the 8-bit KV cache (rope_kv8 / kv8_read), decode attention over it
(attn_decode8 / attn_decode8_rope), linears of few rows with 4-bit weights (linear_q4) and the logits processor (logits_process).

`own` selects what run() computes: False - the operators' plain form in elementary torch operations, in fp32, rounded once at the end; True -
the calls a user makes of modelcompose_amd.ops.  exact() gives the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
ST = torch.bfloat16
F32 = torch.float32
TOP = {"e4m3": 448.0, "int8": 127.0}          # the largest code of each cache format
TINY = 2.0 ** -100                            # the smallest |x| maximum a vector is scaled by: zero vectors have a scale too


# ---- the cases -------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a stage-2 batch's prompts into an empty cache, and the bf16 keys / values a chunked prefill reads back
        {"name": "kv8 4x682", "op": "kv8", "B": 4, "L": 682, "H": 32, "Hkv": 32, "D": 128, "fmt": "e4m3", "ragged": False},
        # a few requests of odd lengths, shared key heads, integer codes
        {"name": "kv8 gqa int8 3x333", "op": "kv8", "B": 3, "L": 333, "H": 32, "Hkv": 8, "D": 128, "fmt": "int8", "ragged": True},
        # the evaluation batch's spliced prompts
        {"name": "kv8 48x2793", "op": "kv8", "B": 48, "L": 2793, "H": 32, "Hkv": 32, "D": 128, "fmt": "e4m3", "ragged": True},
        # one decode step of the batch-1 evaluation: launch latency and filling the chip from 32 heads
        {"name": "attn 1x2809", "op": "attn_rope", "B": 1, "S": 2809, "H": 32, "Hkv": 32, "D": 128, "fmt": "e4m3", "ragged": False},
        # one decode step of the evaluation batch
        {"name": "attn 48x2809", "op": "attn_rope", "B": 48, "S": 2809, "H": 32, "Hkv": 32, "D": 128, "fmt": "e4m3", "ragged": True},
        # long contexts with shared key heads, integer codes
        {"name": "attn gqa 8x32768 int8", "op": "attn_rope", "B": 8, "S": 32768, "H": 32, "Hkv": 8, "D": 128, "fmt": "int8", "ragged": True},
        # short left-padded requests with masked keys and small heads, the queries already rotated
        {"name": "attn mask 5x517 d64", "op": "attn", "B": 5, "S": 517, "H": 12, "Hkv": 4, "D": 64, "fmt": "e4m3", "ragged": True},
        # one token through an attention projection
        {"name": "q4 1x4096x4096", "op": "q4", "M": 1, "N": 4096, "K": 4096, "group": 128, "zeros": False, "f32": False, "residual": True},
        # the evaluation batch through the q|k|v projection, weights with zero points
        {"name": "q4 48x12288x4096", "op": "q4", "M": 48, "N": 12288, "K": 4096, "group": 128, "zeros": True, "f32": False, "residual": False},
        # the vocabulary projection of a handful of requests, fp32 logits, small groups
        {"name": "q4 8x32000x4096 f32", "op": "q4", "M": 8, "N": 32000, "K": 4096, "group": 64, "zeros": True, "f32": True, "residual": False},
        # the logits of one request after a long prompt
        {"name": "logits 1x32000", "op": "logits", "M": 1, "V": 32000, "Lp": 2809, "Lo": 32, "nb": 8, "mask": True},
        # a large batch with a large vocabulary
        {"name": "logits 64x131072", "op": "logits", "M": 64, "V": 131072, "Lp": 4096, "Lo": 1024, "nb": 64, "mask": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["kv8", "attn_rope", "attn", "q4", "logits"])
    if op == "q4":
        group = rng.choice([32, 64, 128])
        return {"op": op, "M": _log(rng, 1, 64), "N": _log(rng, 64, 32000), "K": group * _log(rng, 2, 11008 // group), "group": group,
                "zeros": rng.random() < 0.5, "f32": rng.random() < 0.3, "residual": rng.random() < 0.5}
    if op == "logits":
        return {"op": op, "M": _log(rng, 1, 64), "V": _log(rng, 97, 131072), "Lp": _log(rng, 1, 4096), "Lo": _log(rng, 1, 1024), "nb": rng.choice([0, 1, 7, 64]),
                "mask": rng.random() < 0.6}
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8, 12, 16, 32])
    H = Hkv * rng.choice([g for g in (1, 1, 2, 3, 4, 8, 16) if g * Hkv <= 64])
    c = {"op": op, "B": 1, "L" if op == "kv8" else "S": 1, "H": H, "Hkv": Hkv, "D": D, "fmt": rng.choice(["e4m3", "int8"]), "ragged": rng.random() < 0.6}
    if op == "kv8":
        c["L"] = _log(rng, 1, 8192)
        c["B"] = _log(rng, 1, max(1, min(48, (48 * 2793 * 96 * 128 // ((H + 2 * Hkv) * D)) // c["L"])))
    else:
        c["S"] = _log(rng, 1, 65536)
        c["B"] = _log(rng, 1, max(1, min(64, (48 * 2809 * 32 * 128 // (Hkv * D)) // c["S"])))
    return c


def _lens(c):
    """Lengths of the sequences: all the same, or spread over the upper half (a function of the case alone)."""
    n = c["L"] if c["op"] == "kv8" else c["S"]
    if not c["ragged"]:
        return [n] * c["B"]
    return [max(1, n - (i * 7919) % (n // 2 + 1)) for i in range(c["B"])]


def _room(n):
    return (n + 63) // 64 * 64 + 64


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(g, rows, heads, D):
    """Pre-rotary q|k|v rows: normal, with a few channels a good deal larger, as projections have them."""
    x = torch.empty(rows, heads * D, dtype=ST, device=DEV).normal_(generator=g)
    gain = torch.where(torch.rand(heads * D, device=DEV, generator=g) < 0.02, 6.0, 1.0).to(ST)
    return x.mul_(gain)


def _tables(n, D):
    inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=F32) / D))
    ang = torch.outer(torch.arange(n, dtype=F32), inv)
    return ang.cos().to(DEV), ang.sin().to(DEV)


def _quantise(x, fmt):
    """[..., D] fp32 -> (codes, scale): one scale per vector, its largest magnitude on the largest code."""
    amax = x.abs().amax(-1).clamp_min(TINY)
    inv = torch.div(torch.full_like(amax, TOP[fmt]), amax)
    y = x * inv[..., None]
    codes = y.to(torch.float8_e4m3fn) if fmt == "e4m3" else y.round().to(torch.int8)
    return codes, amax * torch.tensor(1.0 / TOP[fmt], dtype=F32, device=x.device)


def _filled_cache(g, c, room):
    shape = (c["B"], c["Hkv"], room)
    out = []
    for _ in range(2):
        codes = torch.empty(*shape, c["D"], dtype=torch.float8_e4m3fn if c["fmt"] == "e4m3" else torch.int8, device=DEV)
        scale = torch.empty(*shape, dtype=F32, device=DEV)
        for b in range(c["B"]):
            codes[b], scale[b] = _quantise(torch.randn(c["Hkv"], room, c["D"], device=DEV, generator=g), c["fmt"])
        out += [codes, scale]
    return out


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] == "q4":
        M, N, K, G = c["M"], c["N"], c["K"], c["group"]
        s["codes"] = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=DEV, generator=g)
        s["scales"] = (0.002 + 0.002 * torch.rand(N, K // G, device=DEV, generator=g)).to(ST)
        s["zeros"] = torch.randint(5, 11, (N, K // G), dtype=torch.uint8, device=DEV, generator=g) if c["zeros"] else None
        s["x"] = torch.randn(M, K, device=DEV, generator=g).to(ST)
        s["residual"] = torch.randn(M, N, device=DEV, generator=g).to(ST) if c["residual"] else None
        return s
    if c["op"] == "logits":
        M, V = c["M"], c["V"]
        s["logits"] = torch.randn(M, V, device=DEV, generator=g) * 3
        for n, L in (("prompt", c["Lp"]), ("output", c["Lo"])):
            r = torch.rand(M, L, device=DEV, generator=g)
            s[n] = (r * r * r * V).long().clamp_max(V - 1)          # small ids are the frequent ones
            s[n + "_lens"] = torch.randint((L + 1) // 2, L + 1, (M,), dtype=torch.int32, device=DEV, generator=g)
        s["rep"] = 1.0 + 0.5 * torch.rand(M, device=DEV, generator=g)
        s["pres"] = torch.rand(M, device=DEV, generator=g)
        s["freq"] = 0.2 * torch.rand(M, device=DEV, generator=g)
        s["bias_ids"] = torch.randint(0, V, (M, c["nb"]), dtype=torch.int32, device=DEV, generator=g) if c["nb"] else None
        s["bias"] = 4 * torch.randn(M, c["nb"], device=DEV, generator=g) if c["nb"] else None
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (M, (V + 31) // 32), dtype=torch.int32, device=DEV, generator=g) if c["mask"] else None
        return s
    B, H, Hkv, D, lens = c["B"], c["H"], c["Hkv"], c["D"], _lens(c)
    n = max(lens)
    room = _room(n)
    s["cos"], s["sin"] = _tables(room, D)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if c["op"] == "kv8":
        M = B * n
        s["qkv"] = _activations(g, M, H + 2 * Hkv, D)
        order = torch.randperm(M, device=DEV, generator=g)                 # rows in routed order, padding rows marked -1
        row_b, row_t = order // n, order % n
        pad = row_t >= s["lens"].long()[row_b]
        s["row_b"] = torch.where(pad, -1, row_b).int()
        s["row_t"] = row_t.int()
        s["rows"] = (~pad).nonzero()[:, 0]                                  # the rows that are tokens
        dt = torch.float8_e4m3fn if c["fmt"] == "e4m3" else torch.int8
        s["k"], s["v"] = (torch.zeros(B, Hkv, room, D, dtype=torch.uint8, device=DEV).view(dt) for _ in range(2))
        s["ks"], s["vs"] = (torch.zeros(B, Hkv, room, dtype=F32, device=DEV) for _ in range(2))
        s["q_out"] = torch.zeros(B * n, H * D, dtype=ST, device=DEV)
        return s
    s["k"], s["ks"], s["v"], s["vs"] = _filled_cache(g, c, room)
    if c["op"] == "attn_rope":
        s["qkv"] = _activations(g, B, H + 2 * Hkv, D)
    else:
        s["q"] = torch.randn(B, H, D, device=DEV, generator=g).to(ST)
        keep = torch.rand(B, room, device=DEV, generator=g) < 0.9
        keep[:, : n // 8] = False                                           # left padding
        s["key_valid"] = keep.to(torch.uint8)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    return {"kv8": _plain_kv8, "attn": _plain_attn, "attn_rope": _plain_attn, "q4": _plain_q4, "logits": _plain_logits}[op](state)


def _own(op, s):
    from modelcompose_amd import ops
    c = s["case"]
    if op == "q4":
        w = ops.Q4Weight(s["codes"], s["scales"], s["zeros"])
        return ops.linear_q4(s["x"], w, residual=s["residual"], out_f32=c["f32"])
    if op == "logits":
        return ops.logits_process(s["logits"], prompt_ids=s["prompt"], prompt_lens=s["prompt_lens"], output_ids=s["output"], output_lens=s["output_lens"],
                                  repetition_penalty=s["rep"], presence_penalty=s["pres"], frequency_penalty=s["freq"], bias_ids=s["bias_ids"],
                                  bias=s["bias"], allowed=s["allowed"])
    cache = ops.Kv8Cache(s["k"], s["ks"], s["v"], s["vs"])
    if op == "kv8":
        n = max(_lens(c))
        ops.rope_kv8(s["qkv"], s["row_b"], s["row_t"], s["row_t"], s["cos"], s["sin"], s["q_out"], cache, c["H"], n)
        k, v = ops.kv8_read(cache, n, kv_lens=s["lens"])
        return {"q": s["q_out"], "k": k, "v": v, "k_codes": s["k"], "k_scale": s["ks"], "v_codes": s["v"], "v_scale": s["vs"]}
    if op == "attn":
        return ops.attn_decode8(s["q"], cache, kv_lens=s["lens"], key_valid=s["key_valid"])
    out = ops.attn_decode8_rope(s["qkv"], s["cos"], s["sin"], cache, s["lens"], c["H"])
    return {"out": out, "k_codes": s["k"], "k_scale": s["ks"], "v_codes": s["v"], "v_scale": s["vs"]}


def _rotate(x, cos, sin):
    """rotate-half position rotation of [rows, heads, D] fp32 by the rows' tables [rows, D / 2]."""
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_kv8(s):
    c = s["case"]
    H, Hkv, D, r = c["H"], c["Hkv"], c["D"], s["rows"]
    n = max(_lens(c))
    b, t = s["row_b"][r].long(), s["row_t"][r].long()
    x = s["qkv"][r].float().view(-1, H + 2 * Hkv, D)
    cos, sin = s["cos"][t], s["sin"][t]
    s["q_out"][b * n + t] = _rotate(x[:, :H], cos, sin).to(ST).view(-1, H * D)
    for name, y in (("k", _rotate(x[:, H:H + Hkv], cos, sin)), ("v", x[:, H + Hkv:])):
        codes, scale = _quantise(y, c["fmt"])
        s[name].view(torch.uint8).transpose(1, 2)[b, t] = codes.view(torch.uint8)
        s[name + "s"].transpose(1, 2)[b, t] = scale
    inside = (torch.arange(n, device=DEV) < s["lens"][:, None])[:, None, :, None]
    k, v = (torch.where(inside, s[m][:, :, :n].float() * s[m + "s"][:, :, :n, None], 0.0).to(ST) for m in ("k", "v"))
    return {"q": s["q_out"], "k": k, "v": v, "k_codes": s["k"], "k_scale": s["ks"], "v_codes": s["v"], "v_scale": s["vs"]}


def _plain_attn(s):
    c = s["case"]
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    if c["op"] == "attn_rope":
        x = s["qkv"].float().view(B, H + 2 * Hkv, D)
        pos = s["lens"].long() - 1
        rows = torch.arange(B, device=DEV)
        q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
        q, k = (_rotate(y, s["cos"][pos], s["sin"][pos]) for y in (q, k))
        q = q.to(ST).float()                                               # the queries of the cache's attention are 16-bit numbers
        for name, y in (("k", k), ("v", v)):
            codes, scale = _quantise(y, c["fmt"])
            s[name].view(torch.uint8).transpose(1, 2)[rows, pos] = codes.view(torch.uint8)
            s[name + "s"].transpose(1, 2)[rows, pos] = scale
    else:
        q = s["q"].float()
    n = max(_lens(c))
    seen = torch.arange(n, device=DEV) < s["lens"][:, None]
    if "key_valid" in s:
        seen = seen & (s["key_valid"][:, :n] != 0)
    k, v = (s[m][:, :, :n].float() * s[m + "s"][:, :, :n, None] for m in ("k", "v"))
    q = q.reshape(B, Hkv, H // Hkv, D).transpose(2, 3).contiguous()
    score = torch.matmul(k, q).transpose(2, 3) * (1.0 / math.sqrt(D))
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.contiguous(), v) / torch.where(total == 0, 1.0, total)
    o = o.reshape(B, H * D).to(ST)
    if c["op"] == "attn":
        return o
    return {"out": o, "k_codes": s["k"], "k_scale": s["ks"], "v_codes": s["v"], "v_scale": s["vs"]}


def _plain_q4(s):
    c = s["case"]
    N, K, G = c["N"], c["K"], c["group"]
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(N, K // G, G).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    w = ((code - zero) * s["scales"].float()[..., None]).view(N, K)
    y = torch.matmul(s["x"].float(), w.t())
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y if c["f32"] else y.to(ST)


def _counts(ids, lens, V):
    at = torch.where(torch.arange(ids.shape[1], device=DEV) < lens[:, None], ids, V)
    return torch.zeros(ids.shape[0], V + 1, dtype=torch.int32, device=DEV).scatter_add_(1, at, torch.ones_like(at, dtype=torch.int32))[:, :V]


def _plain_logits(s):
    V = s["case"]["V"]
    x = s["logits"]
    n_out = _counts(s["output"], s["output_lens"], V)
    seen = (n_out + _counts(s["prompt"], s["prompt_lens"], V)) > 0
    rep = s["rep"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (s["freq"][:, None] * n_out + s["pres"][:, None] * (n_out > 0))
    if s["bias"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].long(), s["bias"])
    if s["allowed"] is not None:
        at = torch.arange(V, device=DEV)
        x = torch.where(((s["allowed"][:, at // 32] >> (at % 32)) & 1) != 0, x, -math.inf)
    return x


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "q4":
        M, N, K, G = c["M"], c["N"], c["K"], c["group"]
        moved = N * K // 2 + N * (K // G) * (3 if c["zeros"] else 2) + 2 * M * K + M * N * (4 if c["f32"] else 2) + (2 * M * N if c["residual"] else 0)
        return {"bytes": moved, "flops": 2 * M * N * K}
    if c["op"] == "logits":
        M, V = c["M"], c["V"]
        return {"bytes": M * (8 * V + 6 * (c["Lp"] + c["Lo"]) + 8 * c["nb"] + (V // 8 if c["mask"] else 0) + 20), "flops": 6 * M * V}
    H, Hkv, D, n = c["H"], c["Hkv"], c["D"], sum(_lens(c))
    if c["op"] == "kv8":
        whole = c["B"] * max(_lens(c))
        # q|k|v read, q written, codes and scales written and read, bf16 keys and values written (the padding's zeros too)
        return {"bytes": n * (2 * (H + 2 * Hkv) * D + 2 * H * D + 2 * 2 * Hkv * (D + 4)) + whole * 2 * 2 * Hkv * D, "flops": n * (H + 2 * Hkv) * D * 4}
    moved = n * 2 * Hkv * (D + 4) + c["B"] * H * D * 2 * 2 + (n if c["op"] == "attn" else c["B"] * Hkv * (4 * D + 2 * (D + 4)))
    return {"bytes": moved, "flops": 4 * n * H * D}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------
def _code64(x, fmt):
    """Nearest code (ties to even) of x already divided by the scale."""
    if fmt == "int8":
        return torch.round(x)
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _quantise64(x, fmt):
    scale = x.abs().amax(-1).clamp_min(TINY) / TOP[fmt]
    return _code64(x / scale[..., None], fmt), scale


def _rotate64(x, cos, sin):
    h = x.shape[-1] // 2
    turned = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * torch.cat([cos, cos], -1)[:, None].double() + turned * torch.cat([sin, sin], -1)[:, None].double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "q4":
        N, K, G = c["N"], c["K"], c["group"]
        w = torch.empty(N, K, dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = (s["codes"] % 16).double(), (s["codes"] // 16).double()
        w = w.view(N, K // G, G)
        w = w - (8.0 if s["zeros"] is None else s["zeros"].double()[..., None])
        y = s["x"].double() @ (w * s["scales"].double()[..., None]).view(N, K).t().contiguous()
        return y if s["residual"] is None else y + s["residual"].double()
    if c["op"] == "logits":
        x, V = s["logits"].double(), c["V"]
        for m in range(c["M"]):
            old, new = s["prompt"][m, : int(s["prompt_lens"][m])], s["output"][m, : int(s["output_lens"][m])]
            seen = torch.cat([old, new]).unique()
            x[m, seen] = torch.where(x[m, seen] > 0, x[m, seen] / s["rep"][m].double(), x[m, seen] * s["rep"][m].double())
            x[m] -= s["freq"][m].double() * torch.bincount(new, minlength=V)
            x[m, new.unique()] -= s["pres"][m].double()
            if c["nb"]:
                x[m] += torch.bincount(s["bias_ids"][m].long(), weights=s["bias"][m].double(), minlength=V)
            if c["mask"]:
                bits = (s["allowed"][m][:, None].long() & (1 << torch.arange(32, device=DEV))) != 0
                x[m, ~bits.reshape(-1)[:V]] = -math.inf
        return x
    B, H, Hkv, D, lens = c["B"], c["H"], c["Hkv"], c["D"], _lens(c)
    if c["op"] == "kv8":
        n, room = max(lens), s["k"].shape[2]
        if s["qkv"].numel() > 1 << 29:
            return None
        q = torch.zeros(B * n, H * D, dtype=torch.float64, device=DEV)
        codes = [torch.zeros(B, Hkv, room, D, dtype=torch.float64, device=DEV) for _ in range(2)]
        scale = [torch.zeros(B, Hkv, room, dtype=torch.float64, device=DEV) for _ in range(2)]
        for b in range(B):
            at = (s["row_b"] == b).nonzero()[:, 0]
            t = s["row_t"][at].long()
            x = s["qkv"][at].double().view(-1, H + 2 * Hkv, D)
            q[b * n + t] = _rotate64(x[:, :H], s["cos"][t], s["sin"][t]).reshape(-1, H * D)
            for i, y in enumerate((_rotate64(x[:, H:H + Hkv], s["cos"][t], s["sin"][t]), x[:, H + Hkv:])):
                a, z = _quantise64(y, c["fmt"])
                codes[i][b, :, t], scale[i][b, :, t] = a.transpose(0, 1), z.transpose(0, 1)
        k, v = (codes[i][:, :, :n] * scale[i][:, :, :n, None] for i in range(2))
        return {"q": q, "k": k, "v": v, "k_codes": codes[0], "k_scale": scale[0], "v_codes": codes[1], "v_scale": scale[1]}
    k, v = s["k"].float().double(), s["v"].float().double()
    ks, vs = s["ks"].double(), s["vs"].double()
    last = torch.tensor(lens, device=DEV) - 1
    if c["op"] == "attn_rope":
        x = s["qkv"].double().view(B, H + 2 * Hkv, D)
        cos, sin = s["cos"][last], s["sin"][last]
        q = _rotate64(x[:, :H], cos, sin).to(ST).double()
        for codes, scale, y in ((k, ks, _rotate64(x[:, H:H + Hkv], cos, sin)), (v, vs, x[:, H + Hkv:])):
            for b in range(B):
                codes[b, :, lens[b] - 1], scale[b, :, lens[b] - 1] = _quantise64(y[b], c["fmt"])
    else:
        q = s["q"].double()
    o = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        at = torch.arange(lens[b], device=DEV)
        if c["op"] == "attn":
            at = at[s["key_valid"][b, : lens[b]] != 0]
        if not at.numel():
            continue
        for h in range(Hkv):
            heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
            p = torch.softmax((q[b, heads] @ (k[b, h, at] * ks[b, h, at, None]).t().contiguous()) / math.sqrt(D), -1)
            o[b, heads] = p @ (v[b, h, at] * vs[b, h, at, None])
    o = o.view(B, H * D)
    return o if c["op"] == "attn" else {"out": o, "k_codes": k, "k_scale": ks, "v_codes": v, "v_scale": vs}
