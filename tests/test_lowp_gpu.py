"""Low-precision serving operators (csrc/gemm_q4.hip, csrc/kv8.hip, csrc/logits.hip) against plain 64-bit implementations on the CPU.

Tolerances: a 16-bit output is off by at most half a step of the storage dtype (eps / 2 relative) plus the fp32 error of what is summed, bounded per
element from the terms' magnitudes (the comment at each bound); integer outputs and codes are equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FMTS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}
U = 2.0 ** -24                                             # fp32: half a step


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def _st():
    from modelcompose_amd import ops
    return ops.BF16


def _half():
    return torch.finfo(_st()).eps / 2


def _stored(ref):
    """What rounding ref to the storage dtype may add: half a step, which below the smallest normal number (fp16: 2^-14) is that of the subnormals."""
    return _half() * ref.abs().clamp_min(torch.finfo(_st()).tiny)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape):
    return torch.randn(*shape, generator=g).to(_st())


# ---- plain forms -----------------------------------------------------------------------------------------------------------------
def quantise(x, fmt):
    """fp32 [..., D] -> (codes, scale): the definition, operation by operation (CPU fp32 is IEEE: the codes must be equal bit for bit)."""
    x = x.float()
    amax = x.abs().amax(-1)
    ok = torch.isfinite(amax)
    amax = torch.where(ok, amax, torch.ones_like(amax)).clamp_min(2.0 ** -100)
    inv = torch.full_like(amax, TOP[fmt]) / amax
    y = torch.where(ok[..., None], x * inv[..., None], torch.zeros_like(x))
    codes = y.to(torch.float8_e4m3fn) if fmt == "e4m3" else y.round().to(torch.int8)
    return codes, torch.where(ok, amax * torch.tensor(1.0 / TOP[fmt], dtype=torch.float32), torch.full_like(amax, math.nan))


def rotate(x, cos, sin):
    """x [..., D] fp32, cos / sin broadcastable [..., D / 2]; products and sum rounded on their own."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def tables(n, D, theta=10000.0):
    ang = torch.outer(torch.arange(n, dtype=torch.float64), 1.0 / theta ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    return ang.cos().float(), ang.sin().float()


def value(codes, scale):
    return codes.float().double() * scale.double()[..., None]


def make_cache(g, B, Hkv, S, D, fmt, layout="bhsd"):
    """A cache of random vectors on the GPU -> (Kv8Cache, and on the CPU: k codes, k scale, v codes, v scale)."""
    from modelcompose_amd import ops
    host = []
    for _ in range(2):
        c, s = quantise(torch.randn(B, Hkv, S, D, generator=g), fmt)
        host += [c, s]

    def place(t):
        u = t.view(torch.uint8) if t.dtype in (torch.float8_e4m3fn, torch.int8) else t
        if layout == "bshd" and t.dim() == 4:                     # positions outside heads
            return u.transpose(1, 2).contiguous().cuda().transpose(1, 2).view(t.dtype) if t.dtype == torch.int8 else \
                u.transpose(1, 2).contiguous().cuda().view(t.dtype).transpose(1, 2)
        return u.cuda().view(t.dtype) if t.dim() == 4 else u.cuda()
    k, ks, v, vs = (place(t) for t in host)
    return ops.Kv8Cache(k, ks, v, vs), host


def attend(q, host, lens, scale, key_valid=None):
    """(out, bound): softmax attention in 64 bits and what 16-bit storage and fp32 arithmetic may add.  q fp64 [B, H, D]."""
    kc, ks, vc, vs = host
    B, H, D = q.shape
    Hkv = kc.shape[1]
    out, bound = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    for b in range(B):
        at = torch.arange(max(0, min(int(lens[b]), kc.shape[2])))
        if key_valid is not None:
            at = at[key_valid[b, :len(at)] != 0]
        if not len(at):
            continue
        for h in range(H):
            hk = h // (H // Hkv)
            k, v = value(kc[b, hk, at], ks[b, hk, at]), value(vc[b, hk, at], vs[b, hk, at])
            p = torch.softmax(k @ q[b, h] * scale, 0)
            out[b, h] = p @ v
            # score: D fused or D separately rounded products of fp32, two scalings; the weights carry its absolute error as a relative one, doubled
            # by the normalisation; n terms are summed, and each weight is held to 2^-17 or better
            delta = (D + 4) * U * (k.abs() @ q[b, h].abs() * abs(scale)).max()
            bound[b, h] = _stored(out[b, h]) + (2 * delta + (len(at) + 16) * 2 * U + 2.0 ** -16) * (p @ v.abs()) + 1e-30
    return out, bound


def near(got, ref, bound):
    d = (got.double().cpu() - ref).abs()
    assert torch.isfinite(got.float()).all()
    assert (d <= bound * (1 + 1e-6)).all(), f"worst {float((d / bound.clamp_min(1e-300)).max())} of the bound"


# ---- cache write and read-back -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("B,L,H,Hkv,D,layout", [(1, 1, 2, 2, 128, "bhsd"), (3, 37, 6, 2, 64, "bhsd"), (2, 65, 4, 4, 128, "bshd"), (2, 9, 17, 1, 64, "bshd")])
def test_rope_kv8_and_read(fmt, B, L, H, Hkv, D, layout):
    from modelcompose_amd import ops
    g = _gen(1)
    S = L + 3
    lens = torch.tensor([max(1, L - 5 * b) for b in range(B)], dtype=torch.int32)
    M = B * L
    qkv = _rand(g, M, (H + 2 * Hkv) * D + 8)[:, :(H + 2 * Hkv) * D]                  # row stride wider than the row
    order = torch.randperm(M, generator=g)
    row_b, row_t = (order // L).int(), (order % L).int()
    row_b[row_t >= lens[row_b.long()]] = -1
    cos, sin = tables(S, D)
    cache, host = make_cache(g, B, Hkv, S, D, fmt, layout)
    before = [t.clone() for t in host]
    qs = qkv.stride(0)
    dq = torch.empty(M, qs, dtype=_st(), device="cuda")[:, :qkv.shape[1]]
    dq.copy_(qkv)
    q_out = torch.full((B * L, H * D), 7.0, dtype=_st(), device="cuda")
    ops.rope_kv8(dq, row_b.cuda(), row_t.cuda(), row_t.cuda(), cos.cuda(), sin.cuda(), q_out, cache, H, L)
    # the 16-bit form's queries, bit for bit
    q16 = torch.full((B * L, H * D), 7.0, dtype=_st(), device="cuda")
    kc, vc = (torch.zeros(B, Hkv, S, D, dtype=_st(), device="cuda") for _ in range(2))
    ops.rope_kv(dq, row_b.cuda(), row_t.cuda(), row_t.cuda(), cos.cuda(), sin.cuda(), q16, kc, vc, H, Hkv, D, L, S)
    assert torch.equal(q_out, q16)
    want = [t.clone() for t in before]
    x = qkv.float().view(M, H + 2 * Hkv, D)
    for r in range(M):
        b, t = int(row_b[r]), int(row_t[r])
        if b < 0:
            continue
        for i, y in ((0, rotate(x[r, H:H + Hkv], cos[t], sin[t])), (2, x[r, H + Hkv:])):
            c, s = quantise(y, fmt)
            want[i].view(torch.uint8)[b, :, t] = c.view(torch.uint8)
            want[i + 1][b, :, t] = s
            # half a code step of the exact value: e4m3 2^-4 of it, or 2^-10 scales among the subnormals; int8 half a scale
            ref = y.double()
            step = torch.maximum(ref.abs() * 2.0 ** -4, s.double()[:, None] * 2.0 ** -10) if fmt == "e4m3" else s.double()[:, None] * 0.5
            assert ((value(c, s) - ref).abs() <= step * (1 + 1e-5)).all()
    for got, ref in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), want):
        got = got.cpu()
        assert torch.equal(got.view(torch.uint8) if got.dim() == 4 else got, ref.view(torch.uint8) if ref.dim() == 4 else ref)
    for n in (L, S, 1, 0):
        k, v = ops.kv8_read(cache, n, kv_lens=lens.cuda())
        inside = (torch.arange(n) < lens[:, None])[:, None, :, None]
        for got, i in ((k, 0), (v, 2)):
            assert torch.equal(got.cpu(), torch.where(inside, want[i][:, :, :n].float() * want[i + 1][:, :, :n, None], torch.tensor(0.0)).to(_st()))
    k, _ = ops.kv8_read(cache)
    assert torch.equal(k.cpu(), (want[0].float() * want[1][..., None]).to(_st()))


# rows of more heads than a workgroup of the writer takes
@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("B,L,H,Hkv,D,layout", [(2, 5, 32, 32, 128, "bhsd"), (1, 3, 40, 8, 128, "bshd"), (2, 4, 64, 4, 64, "bhsd")])
def test_rope_kv8_and_read_of_many_heads(fmt, B, L, H, Hkv, D, layout):
    test_rope_kv8_and_read(fmt, B, L, H, Hkv, D, layout)


@pytest.mark.parametrize("fmt", list(FMTS))
def test_special_vectors(fmt):
    """Zero, tiny, huge and non-finite vectors; an infinity or NaN stays in its own vector."""
    from modelcompose_amd import ops
    D, S = 64, 8
    qkv = torch.zeros(S, 3 * D, dtype=torch.float32)
    for r, x in enumerate((0.0, torch.finfo(_st()).tiny, torch.finfo(_st()).max / 4, 1.0, 2.0, 3.0, 4.0, 5.0)):
        qkv[r] = x
    qkv[4, 2 * D + 3], qkv[5, 2 * D + 7], qkv[6, 2 * D + 9] = math.inf, math.nan, -math.inf
    qkv = qkv.to(_st())
    cos, sin = torch.ones(S, D // 2), torch.zeros(S, D // 2)
    cache = ops.kv8_cache(1, 1, S, D, dtype=FMTS[fmt])
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).cuda()
    q = torch.zeros(S, D, dtype=_st(), device="cuda")
    ops.rope_kv8(qkv.cuda(), i32([0] * S), i32(range(S)), i32(range(S)), cos.cuda(), sin.cuda(), q, cache, 1, S)
    for name, part in (("k", qkv[:, D:2 * D]), ("v", qkv[:, 2 * D:])):
        c, s = quantise(part, fmt)
        assert torch.equal(getattr(cache, name)[0, 0].cpu().view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(torch.nan_to_num(getattr(cache, name + "_scale")[0, 0].cpu(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
    _, v = ops.kv8_read(cache)
    assert torch.isnan(v[0, 0, 4:7]).all() and torch.isfinite(v[0, 0, :4]).all() and torch.isfinite(v[0, 0, 7]).all()
    # masked or beyond the length they touch nothing; attended they make the row NaN
    keep = torch.ones(1, S, dtype=torch.uint8)
    keep[0, 4:7] = 0
    qq = torch.ones(1, 1, D, dtype=_st(), device="cuda") * 0.01
    assert torch.isfinite(ops.attn_decode8(qq, cache, kv_lens=i32([4]))).all()
    assert torch.isfinite(ops.attn_decode8(qq, cache, key_valid=keep.cuda())).all()
    assert torch.isnan(ops.attn_decode8(qq, cache)).all()


def test_rows_outside_write_nothing():
    from modelcompose_amd import ops
    D, S, H = 64, 6, 2
    cache = ops.kv8_cache(2, 1, S, D)
    g = _gen(3)
    qkv = _rand(g, 7, (H + 2) * D).cuda()
    i32 = lambda *t: torch.tensor(t, dtype=torch.int32).cuda()
    cos, sin = (t.cuda() for t in tables(5, D))                      # one row less than the cache
    q = torch.full((2 * 3, H * D), 3.0, dtype=_st(), device="cuda")
    #            padding  past B   pos < 0  past S   past tables  t past Lq  good
    ops.rope_kv8(qkv, i32(-1, 2, 0, 0, 0, 0, 1), i32(0, 0, -1, 6, 5, 1, 4), i32(0, 0, 0, 0, 0, 3, 2), cos, sin, q, cache, H, 3)
    ks = cache.k_scale.cpu()
    assert ks[1, 0, 4] > 0 and int((ks != 0).sum()) == 1 and int((cache.v_scale != 0).sum()) == 1
    q = q.cpu()
    assert (q[:5] == 3.0).all() and not (q[5] == 3.0).all()
    ops.rope_kv8(qkv[:0], i32(), i32(), i32(), cos, sin, q.cuda(), cache, H, 3)          # no rows: nothing happens


# ---- decode attention ----------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1, 1, 128), (1, 2, 2, 31, 128), (2, 8, 8, 33, 64), (3, 6, 2, 130, 128), (2, 16, 2, 517, 64), (2, 12, 1, 700, 128), (1, 32, 2, 1100, 128),
          (5, 4, 4, 1025, 64), (2, 3, 1, 2100, 128), (1, 24, 1, 513, 64)]


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("B,H,Hkv,S,D", SHAPES)
def test_attn_decode8(fmt, B, H, Hkv, S, D):
    from modelcompose_amd import ops
    g = _gen(B * 1000 + S)
    cache, host = make_cache(g, B, Hkv, S, D, fmt, "bshd" if B == 2 else "bhsd")
    q = _rand(g, B, H, D)
    lens = torch.tensor([S - (b * 37) % S for b in range(B)], dtype=torch.int32)
    scale = 1.0 / math.sqrt(D)
    ref, bound = attend(q.double(), host, lens, scale)
    got = ops.attn_decode8(q.cuda(), cache, kv_lens=lens.cuda()).view(B, H, D)
    near(got, ref, bound)
    got = ops.attn_decode8(q.cuda(), cache, scale=3.0 * scale).view(B, H, D)               # every position; a sharper softmax
    near(got, *attend(q.double(), host, [S] * B, 3.0 * scale))
    keep = (torch.rand(B, S + 5, generator=g) < 0.7)
    keep[:, :min(S - 1, S // 3)] = False
    keep[0] = False                                                                       # a row that is left with nothing
    keep[-1, S // 2:] = True
    ref, bound = attend(q.double(), host, lens, scale, keep)
    got = ops.attn_decode8(q.cuda(), cache, kv_lens=lens.cuda(), key_valid=keep.cuda()).view(B, H, D)
    near(got, ref, bound)
    if B > 1:
        assert (got[0] == 0).all()


@pytest.mark.parametrize("fmt", list(FMTS))
def test_lengths_of_zero_and_garbage_behind_the_end(fmt):
    """Lengths 0, negative, one, S and past S; whatever lies behind a length - codes that are no numbers, NaN and infinite scales - is never felt."""
    from modelcompose_amd import ops
    g = _gen(11)
    B, H, Hkv, S, D = 6, 4, 2, 600, 128
    cache, host = make_cache(g, B, Hkv, S, D, fmt)
    lens = torch.tensor([0, -3, 1, S, S + 9, 577], dtype=torch.int32)
    for b in range(B):
        n = max(0, int(lens[b]))
        cache.k[b, :, n:].view(torch.uint8).fill_(0xFF)
        cache.v[b, :, n:].view(torch.uint8).fill_(0x7F)
        cache.k_scale[b, :, n:] = math.nan
        cache.v_scale[b, :, n:] = math.inf
    q = _rand(g, B, H, D)
    ref, bound = attend(q.double(), host, lens, 1 / math.sqrt(D))
    out = torch.full((B, H * D + 8), 5.0, dtype=_st(), device="cuda")
    got = ops.attn_decode8(q.cuda(), cache, kv_lens=lens.cuda(), out=out[:, :H * D])
    near(got.reshape(B, H, D), ref, bound)
    assert (got[:2] == 0).all() and (out[:, H * D:] == 5.0).all()
    # the same poison at masked keys inside the length
    cache, host = make_cache(g, 1, Hkv, S, D, fmt)
    keep = torch.rand(1, S, generator=g) < 0.5
    hit = (~keep[0]).nonzero()[:, 0].cuda()
    cache.k.view(torch.uint8)[0, :, hit] = 0xFF
    cache.v.view(torch.uint8)[0, :, hit] = 0xFF
    cache.k_scale[0, :, hit], cache.v_scale[0, :, hit] = math.inf, math.nan
    near(ops.attn_decode8(q[:1].cuda(), cache, key_valid=keep.cuda()).view(1, H, D), *attend(q[:1].double(), host, [S], 1 / math.sqrt(D), keep))


def test_extreme_scores():
    """Scores of thousands with either sign: the running maximum has to carry them, also where the first keys are far below the last."""
    from modelcompose_amd import ops
    g = _gen(12)
    B, H, S, D = 2, 2, 1200, 64
    cache, host = make_cache(g, B, H, S, D, "e4m3")
    host[1].mul_(torch.linspace(0.0, 60.0, S))
    cache.k_scale.copy_(host[1])
    q = _rand(g, B, H, D) * 4
    q[1] = -q[1]
    ref, bound = attend(q.double(), host, [S] * B, 1.0)
    near(ops.attn_decode8(q.cuda(), cache, scale=1.0).view(B, H, D), ref, bound)


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("B,H,Hkv,S,D", [(1, 2, 2, 64, 128), (4, 6, 2, 530, 64), (3, 32, 32, 1027, 128), (2, 9, 1, 40, 128)])
def test_attn_decode8_rope_is_append_then_attend(fmt, B, H, Hkv, S, D):
    from modelcompose_amd import ops
    g = _gen(21)
    cache, host = make_cache(g, B, Hkv, S, D, fmt)
    lens = torch.tensor([1, S, S // 2 + 1, S - 1][:B], dtype=torch.int32)
    qkv = _rand(g, B, (H + 2 * Hkv) * D)
    cos, sin = tables(S, D)
    out = ops.attn_decode8_rope(qkv.cuda(), cos.cuda(), sin.cuda(), cache, lens.cuda(), H)
    x = qkv.float().view(B, H + 2 * Hkv, D)
    q = torch.empty(B, H, D, dtype=torch.float64)
    q16 = torch.zeros(B, H * D, dtype=_st(), device="cuda")
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).cuda()
    trash = [torch.zeros(B, Hkv, S, D, dtype=_st(), device="cuda") for _ in range(2)]
    ops.rope_kv(qkv.cuda(), i32(range(B)), i32(lens - 1), i32([0] * B), cos.cuda(), sin.cuda(), q16, *trash, H, Hkv, D, 1, S)
    q = q16.cpu().double().view(B, H, D)
    for b in range(B):
        t = int(lens[b]) - 1
        for i, y in ((0, rotate(x[b, H:H + Hkv], cos[t], sin[t])), (2, x[b, H + Hkv:])):
            c, s = quantise(y, fmt)
            host[i].view(torch.uint8)[b, :, t] = c.view(torch.uint8)
            host[i + 1][b, :, t] = s
    for got, ref in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), host):
        got = got.cpu()
        assert torch.equal(got.view(torch.uint8) if got.dim() == 4 else got, ref.view(torch.uint8) if ref.dim() == 4 else ref)
    near(out.view(B, H, D), *attend(q, host, lens, 1 / math.sqrt(D)))
    # the append and the attention over the appended cache give the same bits as the two calls
    assert torch.equal(out, ops.attn_decode8(q16.view(B, H, D), cache, kv_lens=lens.cuda()))
    keep = torch.rand(B, S, generator=g) < 0.6
    got = ops.attn_decode8_rope(qkv.cuda(), cos.cuda(), sin.cuda(), cache, lens.cuda(), H, key_valid=keep.cuda())
    near(got.view(B, H, D), *attend(q, host, lens, 1 / math.sqrt(D), keep))


def test_attn_decode8_rope_leaves_idle_sequences_alone():
    from modelcompose_amd import ops
    g = _gen(22)
    B, H, S, D = 5, 2, 48, 64
    cache, host = make_cache(g, B, H, S, D, "int8")
    cos, sin = tables(40, D)                                                           # fewer rows than the cache has positions
    lens = torch.tensor([0, S + 1, 41, 40, -7], dtype=torch.int32)
    out = torch.full((B, H * D), 9.0, dtype=_st(), device="cuda")
    ops.attn_decode8_rope(_rand(g, B, 3 * H * D).cuda(), cos.cuda(), sin.cuda(), cache, lens.cuda(), H, out=out)
    assert (out[[0, 1, 2, 4]] == 0).all() and (out[3] != 0).any()
    for b in (0, 1, 2, 4):
        assert torch.equal(cache.k[b].cpu(), host[0][b]) and torch.equal(cache.v_scale[b].cpu(), host[3][b])


def test_a_row_does_not_depend_on_its_batch_or_the_cache_size():
    from modelcompose_amd import ops
    g = _gen(23)
    H, Hkv, S, D = 8, 2, 1500, 128
    cache, host = make_cache(g, 40, Hkv, S, D, "e4m3")
    q = _rand(g, 40, H, D).cuda()
    lens = torch.randint(1, S + 1, (40,), generator=g).int()
    whole = ops.attn_decode8(q, cache, kv_lens=lens.cuda())
    for b0, b1 in ((0, 1), (7, 11), (39, 40)):
        sub = ops.Kv8Cache(cache.k[b0:b1], cache.k_scale[b0:b1], cache.v[b0:b1], cache.v_scale[b0:b1])
        assert torch.equal(ops.attn_decode8(q[b0:b1], sub, kv_lens=lens[b0:b1].cuda()), whole[b0:b1])
    n = int(lens[7])                                                                    # a cache of exactly that many positions
    sub = ops.Kv8Cache(cache.k[7:8, :, :n], cache.k_scale[7:8, :, :n], cache.v[7:8, :, :n], cache.v_scale[7:8, :, :n])
    assert torch.equal(ops.attn_decode8(q[7:8], sub), whole[7:8])


@pytest.mark.parametrize("lens", [(4096, 4097, 4100, 33), (16384, 16385, 16390, 4095), (20000, 5, 16383, 18433)])
def test_lengths_around_a_change_of_the_chunk(lens):
    from modelcompose_amd import ops
    g = _gen(lens[0])
    S, D = max(lens) + 70, 64
    cache, host = make_cache(g, len(lens), 1, S, D, "int8")
    q = _rand(g, len(lens), 3, D) * 2
    n = torch.tensor(lens, dtype=torch.int32)
    got = ops.attn_decode8(q.cuda(), cache, kv_lens=n.cuda())
    near(got.view(-1, 3, D), *attend(q.double(), host, lens, 1 / math.sqrt(D)))
    for b in range(len(lens)):                                                          # alone, in a cache of its own length
        one = ops.Kv8Cache(*(t[b:b + 1, :, :lens[b]] for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)))
        assert torch.equal(ops.attn_decode8(q[b:b + 1].cuda(), one)[0], got[b])


def test_more_partials_than_a_batch_of_the_join():
    """600 000 keys: 293 partials of 2048 keys."""
    from modelcompose_amd import ops
    g = _gen(77)
    S, D = 600_000, 64
    cache, host = make_cache(g, 1, 1, S, D, "int8")
    host[1][0, 0, 500_000:500_064] *= 6                                                    # some weight late, in the second batch of partials
    cache.k_scale.copy_(host[1])
    q = _rand(g, 1, 2, D)
    near(ops.attn_decode8(q.cuda(), cache).view(1, 2, D), *attend(q.double(), host, [S], 1 / math.sqrt(D)))


def test_workgroups_that_take_several_chunks():
    """So many sequences that a workgroup takes every other chunk: the same bits as one sequence at a time, whose workgroups take one."""
    from modelcompose_amd import ops
    g = _gen(78)
    B, H, S, D = 48, 48, 1800, 64
    cache = ops.kv8_cache(B, H, S, D)
    for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        t.view(torch.uint8).copy_(torch.randint(0, 120, t.shape, dtype=torch.uint8, device="cuda"))
        s.uniform_(0.001, 0.01)
    lens = torch.randint(1, S + 1, (B,), generator=g).int().cuda()
    q = _rand(g, B, H, D).cuda()
    whole = ops.attn_decode8(q, cache, kv_lens=lens)
    for b in (0, 13, 47):
        one = ops.Kv8Cache(*(t[b:b + 1] for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)))
        assert torch.equal(ops.attn_decode8(q[b:b + 1], one, kv_lens=lens[b:b + 1])[0], whole[b])


def test_offsets_past_32_bits():
    """A cache of more than 2^31 bytes: written, read and attended at its far end."""
    from modelcompose_amd import ops
    Hkv, S, D = 2, (1 << 23) + 77, 128                                                   # 2 x 1.07e9 bytes: head 1 ends past 2^31
    cache = ops.kv8_cache(1, Hkv, S, D, dtype=torch.int8)
    g = _gen(31)
    x = _rand(g, 1, 3 * Hkv * D)
    cos, sin = torch.ones(1, D // 2), torch.zeros(1, D // 2)
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).cuda()
    big_cos, big_sin = torch.ones(S, D // 2, device="cuda"), torch.zeros(S, D // 2, device="cuda")
    q = torch.zeros(1, Hkv * D, dtype=_st(), device="cuda")
    ops.rope_kv8(x.cuda(), i32([0]), i32([S - 1]), i32([0]), big_cos, big_sin, q, cache, Hkv, 1)
    v = x.float().view(3 * Hkv, D)[2 * Hkv:]
    c, s = quantise(v, "int8")
    assert torch.equal(cache.v[0, :, S - 1].cpu(), c) and torch.equal(cache.v_scale[0, :, S - 1].cpu(), s)
    assert int((cache.k_scale != 0).sum()) == Hkv
    keep = torch.zeros(1, S, dtype=torch.uint8, device="cuda")
    keep[0, S - 1] = 1
    out = ops.attn_decode8(x[:, :Hkv * D].view(1, Hkv, D).cuda(), cache, key_valid=keep)
    # one key: its weight is 1, and w = 1 * v_scale enters the product as hi + lo, each rounded to bfloat16.  For w in [1, 2) (any binade alike) the rest
    # w - hi is at most 2^-8, and below 2^-8 a bfloat16 step is at most 2^-16: lo is off by 2^-17 at most.  The code is exact, the two products are added
    # in fp32 (2^-23) and the division by the sum 1 is exact; the rounding to the storage type adds half a step.
    ref = c.double() * s.double()[:, None]
    assert ((out.cpu().view(Hkv, D).double() - ref).abs() <= ref.abs() * (torch.finfo(_st()).eps / 2 + 2 ** -17 + 2 ** -22)).all()
    _, vr = ops.kv8_read(cache)
    assert torch.equal(vr[0, :, S - 1].cpu(), (c.float() * s[:, None]).to(_st())) and int((vr != 0).sum()) == int((vr[0, :, S - 1] != 0).sum())


# ---- 4-bit weights ---------------------------------------------------------------------------------------------------------------------
def q4_ref(x, codes, scales, zeros, group):
    """(product, sum of the terms' magnitudes with the zero points counted on their own) in 64 bits."""
    N = codes.shape[0]
    q = torch.stack([codes & 15, codes >> 4], -1).view(N, -1).double()
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)
    s = scales.double().repeat_interleave(group, 1)
    return x.double() @ ((q - z) * s).t().contiguous(), x.double().abs() @ ((q + z) * s.abs()).t().contiguous()


def random_q4(g, N, K, group, zeros):
    codes = torch.randint(0, 256, (N, K // 2), generator=g).to(torch.uint8)
    scales = (torch.rand(N, K // group, generator=g) * 0.01 + 0.001).to(_st())
    return codes, scales, torch.randint(0, 16, (N, K // group), generator=g).to(torch.uint8) if zeros else None


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 48, 64])
@pytest.mark.parametrize("N,K,group,zeros", [(1, 32, 32, False), (16, 128, 128, True), (17, 96, 32, True), (65, 1024, 64, False), (250, 4096, 128, True),
                                             (33, 11008, 128, False), (129, 2752, 64, True), (40, 544, 32, False)])
def test_linear_q4(M, N, K, group, zeros):
    from modelcompose_amd import ops
    g = _gen(N * 31 + M)
    codes, scales, z = random_q4(g, N, K, group, zeros)
    x, res, bias = _rand(g, M, K) + 0.25, _rand(g, M, N), _rand(g, N)                      # not centred: the zero points matter
    w = ops.Q4Weight(codes.cuda(), scales.cuda(), None if z is None else z.cuda(), bias.cuda())
    ref, mag = q4_ref(x, codes, scales, z, group)
    err = (K + 16) * U * mag                                                               # K products summed in fp32 in whatever order, then scaled
    y32 = ops.linear_q4(x.cuda(), w, out_f32=True, bias=False)
    near(y32, ref, err + 1e-30)
    y = ops.linear_q4(x.cuda(), w, residual=res.cuda())
    full = ref + bias.double() + res.double()
    near(y, full, _stored(full) + err * 1.01 + 3 * U * (ref.abs() + bias.double().abs() + res.double().abs()) + 1e-30)
    # strided rows in and out, and a row's bits in another batch
    xs = torch.empty(M, K + 24, dtype=_st(), device="cuda")[:, :K]
    xs.copy_(x)
    out = torch.full((M, N + 3), 5.0, device="cuda")
    assert torch.equal(ops.linear_q4(xs, w, out=out[:, :N], out_f32=True, bias=False), y32) and (out[:, N:] == 5.0).all()
    assert torch.equal(ops.linear_q4(x[M // 2:M // 2 + 1].cuda(), w, out_f32=True, bias=False)[0], y32[M // 2])
    res2 = res.cuda()
    assert torch.equal(ops.linear_q4(x.cuda(), w, residual=res2, out=res2), y)               # the residual updated in place


@pytest.mark.parametrize("M", [3, 16, 20, 40, 61])
@pytest.mark.parametrize("N,K,group,zeros", [(4100, 96, 32, True), (5001, 1184, 32, False), (8192, 640, 64, True), (4111, 9088, 128, True),       # two blocks of columns per workgroup
                                             (8193, 32, 32, False), (8240, 1056, 32, True), (9001, 704, 64, False), (8208, 5248, 128, True), (8225, 4736, 64, True)])     # three
def test_linear_q4_of_many_columns(M, N, K, group, zeros):
    from modelcompose_amd import ops
    g = _gen(N * 37 + M)
    codes, scales, z = random_q4(g, N, K, group, zeros)
    x = _rand(g, M, K) + 0.25
    w = ops.Q4Weight(codes.cuda(), scales.cuda(), None if z is None else z.cuda())
    ref, mag = q4_ref(x, codes, scales, z, group)
    y = ops.linear_q4(x.cuda(), w, out_f32=True)
    near(y, ref, (K + 16) * U * mag + 1e-30)
    assert torch.equal(ops.linear_q4(x[M - 1:].cuda(), w, out_f32=True)[0], y[M - 1])
    assert torch.equal(ops.linear_q4(x.cuda(), w), y.to(_st()))


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("N,K,group", [(3, 32, 32), (37, 320, 64), (64, 1024, 128), (5, 4096, 128)])
def test_quantize_and_dequantize_q4(N, K, group, symmetric):
    from modelcompose_amd import ops
    g = _gen(N + K)
    w = _rand(g, N, K) * 0.02
    w[0, :group] = 0
    w[1, :group] = w[1, :group].abs()                                                       # one-sided groups
    w[2, :group] = -w[2, :group].abs()
    q = ops.quantize_q4(w.cuda(), group, symmetric)
    assert (q.N, q.K, q.group) == (N, K, group)
    v = w.float().view(N, K // group, group)
    lo, hi = v.amin(-1).clamp_max(0), v.amax(-1).clamp_min(0)
    s = (torch.maximum(hi, -lo) / 7 if symmetric else (hi - lo) / 15).to(_st())
    assert torch.equal(q.scales.cpu(), s)
    s = s.float()
    z = torch.full_like(s, 8.0) if symmetric else torch.where(s > 0, (-lo / s).round(), torch.zeros_like(s)).clamp(0, 15)
    if not symmetric:
        assert torch.equal(q.zeros.cpu(), z.to(torch.uint8))
    c = (torch.where(s[..., None] > 0, (v / s[..., None]).round(), torch.zeros_like(v)) + z[..., None]).clamp(0, 15)
    codes = torch.stack([q.codes.cpu() & 15, q.codes.cpu() >> 4], -1).view(N, K // group, group).float()
    assert torch.equal(codes, c)
    # half a step from the weight, but for what the 16-bit scale leaves outside the range (8 steps times its half step)
    assert ((codes - z[..., None]).double() * s.double()[..., None] - v.double()).abs().le(s.double()[..., None] * (0.5 + (16 * _half()) + 1e-6)).all()
    pw = ops.dequantize_q4(q)
    assert torch.equal(ops.unpack_weight(pw).cpu(), ((codes - z[..., None]) * s[..., None]).to(_st()).view(N, K))
    wt = torch.empty(N, K + 8, dtype=_st(), device="cuda")[:, :K]
    wt.copy_(w)
    q2 = ops.quantize_q4(wt, group, symmetric)
    assert torch.equal(q2.codes, q.codes) and torch.equal(q2.scales, q.scales)


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize_q4_of_non_finite_weights(symmetric):
    from modelcompose_amd import ops
    w = torch.ones(4, 128).to(_st())
    w[1, 40], w[2, 70], w[3, 127] = math.inf, math.nan, -math.inf
    q = ops.quantize_q4(w.cuda(), 32, symmetric)
    assert torch.equal(torch.isnan(q.scales.cpu()), torch.tensor([[0, 0, 0, 0], [0, 1, 0, 0], [0, 0, 1, 0], [0, 0, 0, 1]]).bool())
    y = ops.linear_q4(torch.ones(1, 128, dtype=_st(), device="cuda"), q)
    assert torch.isnan(y[0, 1:]).all() and torch.isfinite(y[0, 0])


# ---- logits ----------------------------------------------------------------------------------------------------------------------------
def logits_ref(x, prompt=None, plens=None, output=None, olens=None, rep=None, pres=None, freq=None, bids=None, bias=None, allowed=None):
    """(processed, bound) in 64 bits, token by token."""
    M, V = x.shape
    y, mag = x.double().clone(), x.double().abs()
    for m in range(M):
        cut = lambda ids, lens: [] if ids is None else [int(t) for t in ids[m, :ids.shape[1] if lens is None else max(0, min(int(lens[m]), ids.shape[1]))] if 0 <= t < V]
        old, new = cut(prompt, plens), cut(output, olens)
        r = 1.0 if rep is None else float(rep[m])
        for t in set(old + new):
            y[m, t] = y[m, t] / r if y[m, t] > 0 else y[m, t] * r
            mag[m, t] = y[m, t].abs()
        for t in set(new):
            d = (0.0 if freq is None else float(freq[m])) * new.count(t) + (0.0 if pres is None else float(pres[m]))
            y[m, t] -= d
            mag[m, t] += 2 * abs(d)
        if bids is not None:
            for i, t in enumerate(bids[m].tolist()):
                if 0 <= t < V:
                    y[m, t] += float(bias[m, i])
                    mag[m, t] += bids.shape[1] * abs(float(bias[m, i]))
        if allowed is not None:
            bits = torch.tensor([(int(allowed[m, t >> 5]) >> (t & 31)) & 1 for t in range(V)], dtype=torch.bool)
            y[m, ~bits] = -math.inf
    return y, 4 * U * mag + 1e-38                             # at most 4 roundings of what has been added up so far, and the biases' own sum


@pytest.mark.parametrize("M,V,Lp,Lo,nb", [(1, 1, 1, 1, 1), (3, 97, 40, 12, 5), (2, 2048, 300, 70, 0), (5, 2049, 1, 1, 9), (4, 5003, 700, 900, 33), (1, 32000, 50, 20, 8)])
def test_logits_process(M, V, Lp, Lo, nb):
    from modelcompose_amd import ops
    g = _gen(V + M)
    x = torch.randn(M, V, generator=g) * 4
    prompt, output = (torch.randint(-3, V + 3, (M, L), generator=g) for L in (Lp, Lo))         # ids outside the vocabulary are ignored
    prompt[0, 0] = -200
    output[:, Lo // 2:] = output[:, :1]                                                       # one token many times
    plens, olens = torch.randint(0, Lp + 1, (M,), generator=g).int(), torch.randint(0, Lo + 1, (M,), generator=g).int()
    plens[-1], olens[0] = Lp + 5, -2                                                         # clipped
    rep, pres, freq = 0.7 + torch.rand(M, generator=g), torch.randn(M, generator=g), torch.randn(M, generator=g)
    bids = torch.randint(-2, V + 2, (M, nb), generator=g).int() if nb else None
    bias = torch.randn(M, nb, generator=g) * 5 if nb else None
    if nb > 2:
        bids[:, 2] = bids[:, 0]                                                              # the same token twice
    allowed = torch.randint(-2 ** 31, 2 ** 31, (M, (V + 31) // 32), generator=g).int()
    cu = lambda t: None if t is None else t.cuda()
    full = dict(prompt_ids=cu(prompt), prompt_lens=cu(plens), output_ids=cu(output), output_lens=cu(olens), repetition_penalty=cu(rep),
                presence_penalty=cu(pres), frequency_penalty=cu(freq), bias_ids=cu(bids), bias=cu(bias), allowed=cu(allowed))

    def check(got, ref, bound):
        got = got.double().cpu()
        assert torch.equal(torch.isinf(got), torch.isinf(ref)) and not torch.isnan(got).any()
        fin = torch.isfinite(ref)
        assert ((got - ref).abs()[fin] <= bound[fin]).all()
    check(ops.logits_process(x.cuda(), **full), *logits_ref(x, prompt, plens, output, olens, rep, pres, freq, bids, bias, allowed))
    check(ops.logits_process(x.cuda(), prompt_ids=cu(prompt), repetition_penalty=cu(rep)), *logits_ref(x, prompt, rep=rep))
    check(ops.logits_process(x.cuda(), output_ids=cu(output), frequency_penalty=cu(freq)), *logits_ref(x, output=output, freq=freq))
    assert torch.equal(ops.logits_process(x.cuda()).cpu(), x)
    # rows with a stride, in place
    xs = torch.full((M, V + 1), 3.0, device="cuda")
    xs[:, :V] = x.cuda()
    want = ops.logits_process(x.cuda(), **full)
    assert torch.equal(ops.logits_process(xs[:, :V], out=xs[:, :V], **full), want) and (xs[:, V] == 3.0).all()


# so many rows that a workgroup takes 4096 tokens (rows of 16 bytes or not, slices that end early), and histories and biases of more than one round of loads
@pytest.mark.parametrize("M,V,Lp,Lo,nb", [(260, 300, 20, 9, 3), (130, 8193, 12, 30, 2), (128, 4100, 15, 8, 0), (2, 900, 9001, 5003, 1024)])
def test_logits_process_of_many_rows_and_long_histories(M, V, Lp, Lo, nb):
    test_logits_process(M, V, Lp, Lo, nb)


def test_logits_process_special_values():
    from modelcompose_amd import ops
    x = torch.tensor([[math.inf, -math.inf, 0.0, -0.0, 1e38, -1e38, 5.0, math.nan]])
    ids = torch.arange(8)[None]
    y = ops.logits_process(x.cuda(), prompt_ids=ids.cuda(), repetition_penalty=torch.tensor([2.0]).cuda()).cpu()
    assert y[0, :7].tolist() == [math.inf, -math.inf, 0.0, -0.0, float(torch.tensor(5e37)), float(torch.tensor(-2e38)), 2.5] and math.isnan(y[0, 7])
    none = torch.zeros(1, 1, dtype=torch.int32).cuda()                                       # a mask that leaves nothing
    assert torch.isneginf(ops.logits_process(x[:, :7].cuda(), allowed=none)).all()


# ---- together ----------------------------------------------------------------------------------------------------------------------------
class _Step:
    """One decoder layer's decode step as a serving loop runs it, on low-precision weights and cache, then the next token."""

    def __init__(self, seed, B=3, H=4, Hkv=2, D=64, S=80, V=1003):
        from modelcompose_amd import ops
        g = _gen(seed)
        hid = H * D
        self.dims = (B, H, Hkv, D, S, V)
        self.w = {n: ops.quantize_q4((_rand(g, N, K) * 0.05).cuda(), 32, sym) for n, N, K, sym in (
            ("qkv", (H + 2 * Hkv) * D, hid, True), ("o", hid, hid, False), ("lm", V, hid, False))}
        self.cos, self.sin = (t.cuda() for t in tables(S, D))
        self.embed = _rand(g, V, hid).cuda()
        self.cache = ops.kv8_cache(B, Hkv, S, D)
        self.lens = torch.tensor([5, 0, 17][:B], dtype=torch.int32).cuda()
        n = 17
        x = self.embed[torch.randint(0, V, (B * n,), generator=g).cuda()]
        row = torch.arange(B * n)
        b, t = (row // n).int(), (row % n).int()
        b[t >= self.lens.cpu()[b.long()]] = -1
        self.q = torch.zeros(B * n, hid, dtype=_st(), device="cuda")
        ops.rope_kv8(ops.linear_q4(x, self.w["qkv"]), b.cuda(), t.cuda(), t.cuda(), self.cos, self.sin, self.q, self.cache, H, n)
        self.ids = torch.randint(0, V, (B,), generator=g).cuda()
        self.hist = torch.full((B, S), -1, dtype=torch.int64, device="cuda")
        self.count = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.rep = torch.full((B,), 1.3, device="cuda")
        self.freq = torch.full((B,), 0.4, device="cuda")

    def __call__(self):
        from modelcompose_amd import ops
        B, H = self.dims[:2]
        self.lens.add_(1)
        x = self.embed[self.ids]
        a = ops.attn_decode8_rope(ops.linear_q4(x, self.w["qkv"]), self.cos, self.sin, self.cache, self.lens, H)
        h = ops.linear_q4(a, self.w["o"], residual=x)
        logits = ops.linear_q4(h, self.w["lm"], out_f32=True)
        logits = ops.logits_process(logits, output_ids=self.hist, output_lens=self.count, repetition_penalty=self.rep, frequency_penalty=self.freq)
        ops.argmax(logits, out=self.ids)
        self.hist.scatter_(1, self.count.long()[:, None], self.ids[:, None])
        self.count.add_(1)
        return logits, a


def test_decode_steps_against_64_bits():
    """Six steps: each step's attention from its own cache, and its logits from its own inputs, in 64 bits."""
    st = _Step(5)
    B, H, Hkv, D, S, V = st.dims
    for _ in range(6):
        ids, hist, count = st.ids.cpu().clone(), st.hist.cpu().clone(), st.count.cpu().clone()
        logits, a = st()
        host = [t.cpu().clone() for t in (st.cache.k, st.cache.k_scale, st.cache.v, st.cache.v_scale)]
        w = {n: (q.codes.cpu(), q.scales.cpu(), None if q.zeros is None else q.zeros.cpu(), q.group) for n, q in st.w.items()}
        x = st.embed.cpu()[ids]
        y, mag = q4_ref(a.cpu(), *w["o"])
        y = y + x.double()
        h = y.to(_st())
        ref, mag2 = q4_ref(h, *w["lm"])
        # the hidden state is rounded on the way: half a step (a whole one where the fp32 sum sits beside a border) through the last product
        hb = (2 * _stored(y) + (H * D + 16) * U * mag)
        wl = torch.stack([w["lm"][0] & 15, w["lm"][0] >> 4], -1).view(V, -1).double() - w["lm"][2].double().repeat_interleave(32, 1)
        prop = hb @ (wl * w["lm"][1].double().repeat_interleave(32, 1)).abs().t().contiguous()
        p, pb = logits_ref(ref, output=hist, olens=count, rep=st.rep.cpu(), freq=st.freq.cpu())
        assert ((logits.cpu().double() - p).abs() <= 1.3 * (prop + (H * D + 16) * U * mag2) + pb).all()
        q16 = None
        assert torch.isfinite(a.float()).all()
        assert torch.equal(st.ids.cpu(), logits.argmax(-1).cpu())
        _ = host, q16


def test_captured_steps_replay_like_eager_ones():
    eager, graphed = _Step(6), _Step(6)
    eager()
    graphed()                                                                               # (warm-up outside the capture)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    keep = [t.clone() for t in (graphed.lens, graphed.ids, graphed.hist, graphed.count)]
    with torch.cuda.graph(g, stream=side):
        out, att = graphed()
    for t, k in zip((graphed.lens, graphed.ids, graphed.hist, graphed.count), keep):
        assert torch.equal(t, k)                                                            # capturing runs nothing
    for _ in range(4):
        want, want_a = eager()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(att, want_a) and torch.equal(graphed.ids, eager.ids) and torch.equal(graphed.hist, eager.hist)
        for a, b in zip((graphed.cache.k, graphed.cache.v), (eager.cache.k, eager.cache.v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_streams_at_once():
    """Two loops on two streams share no scratch."""
    one, two, ref = _Step(7), _Step(8), [_Step(7), _Step(8)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, step) in enumerate(zip(streams, (one, two))):
            with torch.cuda.stream(s):
                got[i].append(step()[0])
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, ref[i]()[0])


def test_a_later_chunk_attends_to_what_is_read_back():
    """Chunked prefill: the second chunk's queries over the first chunk's keys read back from the cache and its own, through attn_prefill."""
    from modelcompose_amd import ops
    g = _gen(41)
    B, H, D, n0, n1 = 2, 4, 128, 70, 30
    S = n0 + n1
    cache = ops.kv8_cache(B, H, S, D, dtype=torch.int8)
    cos, sin = (t.cuda() for t in tables(S, D))
    for lo, n in ((0, n0), (n0, n1)):
        qkv = _rand(g, B * n, 3 * H * D).cuda()
        row = torch.arange(B * n)
        q = torch.zeros(B * n, H * D, dtype=_st(), device="cuda")
        ops.rope_kv8(qkv, (row // n).int().cuda(), (row % n + lo).int().cuda(), (row % n).int().cuda(), cos, sin, q, cache, H, n)
    k, v = ops.kv8_read(cache, S)
    out = torch.empty(B * n1, H * D, dtype=_st(), device="cuda")
    ops.attn_prefill(q, k, v, out, B, H, H, n1, S, D, (n1 * H * D, H * D, D), (H * S * D, D, S * D), (H * S * D, D, S * D), H * D, True, q_offset=n0)
    kd, vd, qd = k.cpu().double(), v.cpu().double(), q.cpu().double().view(B, n1, H, D)
    for b in range(B):
        for h in range(H):
            s = qd[b, :, h] @ kd[b, h].t() / math.sqrt(D)
            s = s.masked_fill(torch.arange(S) > torch.arange(n1)[:, None] + n0, -math.inf)
            p = torch.softmax(s, -1)
            ref = p @ vd[b, h]
            # 16-bit probabilities in the prefill kernel: half a step of each (and as much for their sum)
            bound = _stored(ref) + (3 * _half()) * (p @ vd[b, h].abs())
            assert ((out.cpu().double().view(B, n1, H, D)[b, :, h] - ref).abs() <= bound + 1e-6).all()
    last = ops.attn_decode8(q.view(B, n1, H, D)[:, -1], cache)                                # the last query as a decode step: the codes themselves
    near(last.view(B, H, D), *attend(qd[:, -1], [t.cpu() for t in (cache.k, cache.k_scale, cache.v, cache.v_scale)], [S] * B, 1 / math.sqrt(D)))


def rounded(got, ref, err):
    """Every element of got is ref rounded to the storage dtype, or - where ref lies within err of a border between two numbers - either of them."""
    lo, hi = ((ref + s * err).to(_st()) for s in (-1, 1))
    got = got.cpu()
    bad = ~((got >= lo) & (got <= hi))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements are not the rounded value"


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 7, 40])
def test_weights_times_scales_keep_fp32(fmt, D, n):
    """All scores equal (the queries are zero): the weights are 1, and what multiplies the codes is the values' scales alone.  Their 24 bits have to arrive:
    two bfloat16 parts of them (2^-17) move a few in a thousand outputs over a border of the storage dtype, three parts are the scale itself."""
    from modelcompose_amd import ops
    g = _gen(200 + n + D)
    B, H, Hkv = 24, 16, 8
    cache, host = make_cache(g, B, Hkv, n, D, fmt)
    host[3].mul_(1.0 + torch.rand(host[3].shape, generator=g))
    cache.v_scale.copy_(host[3])
    got = ops.attn_decode8(torch.zeros(B, H, D, dtype=_st(), device="cuda"), cache).view(B, Hkv, H // Hkv, D)
    v = value(host[2], host[3])
    ref, mag = v.mean(2), v.abs().mean(2)
    # three exact products a key are added in fp32, then the two halves of the columns, 4 waves' partials, one division
    rounded(got, ref[:, :, None].expand_as(got).contiguous(), ((3 * n + 12) * U * mag)[:, :, None])


def test_the_fields_of_a_weight_and_a_cache_cannot_be_replaced():
    """The kernels get the addresses, strides and sizes of construction: another tensor in a field's place would be ignored, and the old one's memory freed."""
    from modelcompose_amd import ops
    g = _gen(51)
    cache = ops.kv8_cache(2, 2, 16, 64)
    codes, scales, z = random_q4(g, 40, 64, 32, True)
    w = ops.Q4Weight(codes.cuda(), scales.cuda(), z.cuda())
    for o, names in ((cache, ("k", "k_scale", "v", "v_scale", "B", "Hkv", "S", "D", "index")), (w, ("codes", "scales", "zeros", "N", "K", "group", "index"))):
        for n in names:
            old = getattr(o, n)
            with pytest.raises(AttributeError):
                setattr(o, n, old)
            with pytest.raises(AttributeError):
                delattr(o, n)
            assert getattr(o, n) is old or getattr(o, n) == old
    with pytest.raises(AttributeError):
        cache.other = 1
    # the bias is read at each call: it may be set, if it is one
    x, bias = _rand(g, 3, 64).cuda(), _rand(g, 40).cuda()
    plain = ops.linear_q4(x, w, out_f32=True)
    w.bias = bias
    assert torch.equal(ops.linear_q4(x, w, out_f32=True), plain + bias.float())
    for bad in (bias[:39], bias.float(), bias.cpu(), torch.zeros(80, dtype=_st(), device="cuda")[::2]):
        with pytest.raises(ValueError):
            w.bias = bad
        assert w.bias is bias
    w.bias = None
    assert torch.equal(ops.linear_q4(x, w, out_f32=True), plain)


@pytest.mark.parametrize("M", [1, 5, 16, 20, 50])
@pytest.mark.parametrize("N,K,group,zeros", [(70, 224, 32, True), (33, 1024, 128, False), (4130, 320, 64, True), (8200, 256, 64, False)])
def test_linear_q4_of_infinities_and_the_largest_numbers(M, N, K, group, zeros):
    """An infinity in x gives what the definition gives: an infinity of the weight's sign, NaN where the weight is zero or two disagree; finite numbers whose products with
    the bare codes pass the range of fp32 give the finite sum.  The other rows do not notice."""
    from modelcompose_amd import ops
    g = _gen(N + M)
    codes, scales, z = random_q4(g, N, K, group, zeros)
    x = _rand(g, M, K)
    clean = x.clone()
    hit = sorted({0, M // 2, M - 1})
    top = torch.finfo(_st()).max
    for i, m in enumerate(hit):
        if i == 0:
            x[m, K - 1] = math.inf
        elif i == 1:
            x[m, 3], x[m, K // 2] = -math.inf, math.inf
        else:
            x[m, 1::2] = top
            x[m, 0::2] = -top
    w = ops.Q4Weight(codes.cuda(), scales.cuda(), None if z is None else z.cuda())
    y = ops.linear_q4(x.cuda(), w, out_f32=True).cpu()
    q = torch.stack([codes & 15, codes >> 4], -1).view(N, -1).double()
    wt = (q - (8.0 if z is None else z.double().repeat_interleave(group, 1))) * scales.double().repeat_interleave(group, 1)
    for m in hit:
        t = x[m].double() * wt                                         # (0 * inf is NaN, as in any product)
        ref = t.sum(1)
        assert torch.equal(torch.isnan(y[m]), torch.isnan(ref)) and torch.equal(torch.isposinf(y[m]), torch.isposinf(ref.float())) and torch.equal(torch.isneginf(y[m]), torch.isneginf(ref.float()))
        fin = torch.isfinite(ref.float())
        assert ((y[m].double() - ref).abs()[fin] <= ((K + 16) * U * (x[m].double().abs() @ (q + 15).mul(scales.double().repeat_interleave(group, 1)).t()))[fin]).all()
    rest = [m for m in range(M) if m not in hit]
    assert torch.equal(y[rest], ops.linear_q4(clean.cuda(), w, out_f32=True).cpu()[rest])
    assert torch.equal(ops.linear_q4(x[M - 1:].cuda(), w, out_f32=True)[0].cpu().nan_to_num(nan=7.0), y[M - 1].nan_to_num(nan=7.0))


def test_linear_q4_of_infinities_is_the_prompt_form():
    """The 16-bit form of the same weight gives the same infinities and NaN."""
    from modelcompose_amd import ops
    g = _gen(61)
    codes, scales, z = random_q4(g, 132, 256, 64, True)
    w = ops.Q4Weight(codes.cuda(), scales.cuda(), z.cuda())
    x = _rand(g, 9, 256)
    x[2, 100], x[5, 0] = math.inf, -math.inf
    a, b = ops.linear_q4(x.cuda(), w).float(), ops.linear(x.cuda(), ops.dequantize_q4(w)).float()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isposinf(a), torch.isposinf(b)) and torch.equal(torch.isneginf(a), torch.isneginf(b))
    assert torch.isinf(a[2]).any() and torch.isinf(a[5]).any()


def _same_id_row(n, V, same):
    g = _gen(n)
    x = torch.randn(1, V, generator=g)
    ids = torch.full((1, n), 5, dtype=torch.int32) if same else torch.randperm(V, generator=g)[:n].int()[None]
    return x, ids, torch.randn(1, n, generator=g)


@pytest.mark.parametrize("n", [1, 2, 3, 17, 64, 65, 100, 513, 1023, 1024])
@pytest.mark.parametrize("V", [1024, 40000])
def test_biases_of_one_token_add_up_in_the_order_of_the_list(n, V):
    """Up to 1024 times the same token, alone or between others: fp32 additions in list order, bit for bit."""
    from modelcompose_amd import ops
    x, ids, bias = _same_id_row(n, V, True)
    y = ops.logits_process(x.cuda(), bias_ids=ids.cuda(), bias=bias.cuda()).cpu()
    total = torch.zeros(())
    for v in bias[0]:
        total = total + v
    want = x.clone()
    want[0, 5] += total
    assert torch.equal(y, want)
    g = _gen(n + 1)
    M = 3
    x = torch.randn(M, V, generator=g)
    ids = torch.randint(-1, 12, (M, n), generator=g).int() * (V // 11)             # a few tokens many times, over all slices, some outside
    bias = torch.randn(M, n, generator=g)
    y = ops.logits_process(x.cuda(), bias_ids=ids.cuda(), bias=bias.cuda()).cpu()
    want = x.clone()
    for m in range(M):
        total = {}
        for t, v in zip(ids[m].tolist(), bias[m]):
            total[t] = total.get(t, torch.zeros(())) + v
        for t, v in total.items():
            if 0 <= t < V:
                want[m, t] += v
    assert torch.equal(y, want)


def test_repeated_biases_cost_about_what_different_ones_do():
    """1024 entries of one token (a ragged list padded with one id) against 1024 tokens: a sum over the list, not a walk of the list per entry."""
    from modelcompose_amd import ops
    times = []
    for same in (False, True):
        x, ids, bias = (t.cuda() for t in _same_id_row(1024, 2048, same))
        out = torch.empty_like(x)
        took = []
        for i in range(12):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            ops.logits_process(x, bias_ids=ids, bias=bias, out=out)
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        times.append(sorted(took)[4])
    assert times[1] <= 10 * times[0] + 0.1, times


def test_quantize_q4_of_the_largest_weights():
    """A range that passes fp32 (the largest numbers of either sign in a group) still has a finite scale."""
    from modelcompose_amd import ops
    g = _gen(71)
    top = torch.finfo(_st()).max
    w = _rand(g, 6, 128)
    w[1, 3], w[1, 40], w[1, 60] = top, -top, top / 2
    w[2, 3], w[2, 4] = top, -top
    w[3, 32:64] = top
    q = ops.quantize_q4(w.cuda(), 32, symmetric=False)
    s, z = q.scales.cpu().double().repeat_interleave(32, 1), q.zeros.cpu().double().repeat_interleave(32, 1)
    assert torch.isfinite(s).all()
    codes = torch.stack([q.codes.cpu() & 15, q.codes.cpu() >> 4], -1).view(6, 128).double()
    assert (((codes - z) * s - w.double()).abs() <= s * (0.5 + 16 * _half() + 1e-6)).all()


def test_quantize_q4_of_a_weight_at_an_odd_address():
    from modelcompose_amd import ops
    w = _rand(_gen(72), 6, 128).cuda()
    q = ops.quantize_q4(w, 32, symmetric=False)
    odd = torch.zeros(6 * 128 + 8, dtype=_st(), device="cuda")[1:1 + 6 * 128].view(6, 128)
    odd.copy_(w)
    for v in (odd, odd[1:, :64], odd.t().contiguous().t()):
        p, r = ops.quantize_q4(v, 32, symmetric=False), ops.quantize_q4(v.clone(memory_format=torch.contiguous_format), 32, symmetric=False)
        assert torch.equal(p.codes, r.codes) and torch.equal(p.scales, r.scales) and torch.equal(p.zeros, r.zeros)
    assert torch.equal(ops.quantize_q4(odd, 32, symmetric=False).codes, q.codes)


def test_attention_of_decode_steps_against_64_bits():
    """Six steps of the loop: each step's projection, the key and value it appends, where it appends them, and its attention over its own cache."""
    from modelcompose_amd import ops
    st = _Step(9)
    B, H, Hkv, D, S, V = st.dims
    qkv_w = st.w["qkv"]
    i32 = lambda t: torch.as_tensor(t, dtype=torch.int32).cuda()
    cache = (st.cache.k, st.cache.k_scale, st.cache.v, st.cache.v_scale)
    for _ in range(6):
        before, x = [t.cpu().clone() for t in cache], st.embed[st.ids]
        _, a = st()
        lens = st.lens.cpu()
        rows = ops.linear_q4(x, qkv_w)
        ref, mag = q4_ref(x.cpu(), qkv_w.codes.cpu(), qkv_w.scales.cpu(), None, qkv_w.group)
        near(rows, ref, _stored(ref) + (H * D + 16) * U * mag + 1e-30)
        y = rows.cpu().float().view(B, H + 2 * Hkv, D)
        want = before
        for b in range(B):
            t = int(lens[b]) - 1
            for i, part in ((0, rotate(y[b, H:H + Hkv], st.cos[t].cpu(), st.sin[t].cpu())), (2, y[b, H + Hkv:])):
                c, s = quantise(part, "e4m3")
                want[i].view(torch.uint8)[b, :, t] = c.view(torch.uint8)
                want[i + 1][b, :, t] = s
        for got, ref in zip(cache, want):
            got = got.cpu()
            assert torch.equal(got.view(torch.uint8) if got.dim() == 4 else got, ref.view(torch.uint8) if ref.dim() == 4 else ref)
        q16 = torch.zeros(B, H * D, dtype=_st(), device="cuda")
        trash = [torch.zeros(B, Hkv, S, D, dtype=_st(), device="cuda") for _ in range(2)]
        ops.rope_kv(rows, i32(range(B)), i32(lens - 1), i32([0] * B), st.cos, st.sin, q16, *trash, H, Hkv, D, 1, S)
        q = rotate(y[:, :H].double(), st.cos[lens.long() - 1].cpu().double()[:, None], st.sin[lens.long() - 1].cpu().double()[:, None])
        near(q16.view(B, H, D), q, _stored(q) + 4 * U * y[:, :H].double().abs().amax(-1, keepdim=True))
        near(a.view(B, H, D), *attend(q16.cpu().double().view(B, H, D), want, lens, 1 / math.sqrt(D)))


@pytest.mark.parametrize("M", [1, 16, 17, 48, 64])
@pytest.mark.parametrize("N,K,group,zeros", [(33, 11008, 128, False), (250, 4096, 128, True), (129, 2752, 64, True), (40, 544, 32, False), (4111, 9088, 128, True), (8208, 5248, 128, True),
                                             (8240, 1056, 32, True), (4300, 2048, 64, False)])
def test_linear_q4_sums_are_kept_in_fp32(M, N, K, group, zeros):
    """Within a bound of the group sums' and the running sum's own fp32 roundings, and exact where these are."""
    from lowp_bounds import q4_sums, whole_numbers
    from modelcompose_amd import ops
    g = _gen(N * 41 + M)
    codes, scales, z = random_q4(g, N, K, group, zeros)
    x = _rand(g, M, K) + 0.25
    cu = lambda t: None if t is None else t.cuda()
    y = ops.linear_q4(x.cuda(), ops.Q4Weight(cu(codes), cu(scales), cu(z)), out_f32=True)
    near(y, *q4_sums(x, codes, scales, z, group))
    x, codes, scales, z = whole_numbers(g, M, N, K, group, zeros, _st())
    y = ops.linear_q4(x.cuda(), ops.Q4Weight(cu(codes), cu(scales), cu(z)), out_f32=True)
    assert torch.equal(y.cpu().double(), q4_ref(x, codes, scales, z, group)[0])


@pytest.mark.parametrize("M", [1, 7, 40])
def test_linear_q4_of_a_row_of_nan(M):
    """A sequence that has become NaN stays NaN and leaves the others alone, at about the cost of any other row."""
    from modelcompose_amd import ops
    g = _gen(81)
    codes, scales, z = random_q4(g, 4100, 4096, 128, True)
    w = ops.Q4Weight(codes.cuda(), scales.cuda(), z.cuda())
    x = _rand(g, M, 4096).cuda()
    clean = ops.linear_q4(x, w)
    bad = x.clone()
    bad[M // 2] = math.nan
    y = ops.linear_q4(bad, w)
    assert torch.isnan(y[M // 2]).all()
    rest = [m for m in range(M) if m != M // 2]
    assert torch.equal(y[rest], clean[rest])
    times = []
    for v in (x, bad):
        took = []
        for _ in range(12):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            ops.linear_q4(v, w, out=y)
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        times.append(sorted(took)[4])
    assert times[1] <= 2 * times[0] + 0.05, times
