"""Refusals of the low-precision serving operators: bad arguments are turned into errors before any launch (C ABI and Python wrappers)."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import os
    import __graft_entry__ as g
    from modelcompose_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        g.build()
    return _lib


def refused(lib, rc, text):
    msg = lib.lib().mc_last_error().decode()
    assert rc == 1 and text in msg, (rc, msg)
    with pytest.raises(ValueError):
        lib.check(rc, "call")


def cache_c(lib, **kw):
    d = dict(k=4096, k_scale=4096, v=4096, v_scale=4096, sb=1 << 20, sh=1 << 16, st=128, scale_sb=1024, scale_sh=128, B=2, Hkv=2, S=128, D=128, format=1)
    d.update(kw)
    return lib.Kv8CacheC(*[d[n] for n, _ in lib.Kv8CacheC._fields_])


@pytest.mark.parametrize("bad,text", [(dict(k=0), "null cache"), (dict(v_scale=0), "null cache"), (dict(format=3), "format"), (dict(D=96), "head_dim"), (dict(S=0), "bad cache shape"),
                                      (dict(B=-1), "bad cache shape"), (dict(st=72), "16-byte"), (dict(k=4100), "16-byte"), (dict(k_scale=4097), "4-byte"),
                                      (dict(B=1 << 13, Hkv=1 << 12), "too large")])
def test_bad_caches(lib, bad, text):
    L, c = lib.lib(), cache_c(lib, **bad)
    one = 4096
    refused(lib, L.mc_kv8_read(C.byref(c), None, 1, one, one, None), text)
    refused(lib, L.mc_rope_kv8(one, 1024, one, one, one, one, one, 16, one, C.byref(c), 1, 4, 1, None), text)
    refused(lib, L.mc_attn_decode8(one, 512, 128, C.byref(c), None, None, 0, one, 512, one, 4, 1.0, None), text)
    refused(lib, L.mc_attn_decode8_rope(one, 1024, one, one, 16, C.byref(c), one, None, 0, one, 512, one, 4, 1.0, None), text)


def test_bad_cache_calls(lib):
    L, c, one = lib.lib(), C.byref(cache_c(lib)), 4096
    refused(lib, L.mc_kv8_read(c, None, 129, one, one, None), "129 positions")
    refused(lib, L.mc_kv8_read(c, None, 1, None, one, None), "null")
    refused(lib, L.mc_kv8_read(c, None, 1, one, 4104, None), "misaligned")
    refused(lib, L.mc_rope_kv8(one, 1024, one, one, one, one, one, 16, one, c, 1, 3, 1, None), "3 query heads over 2")
    refused(lib, L.mc_rope_kv8(one, 1016, one, one, one, one, one, 16, one, c, 1, 4, 1, None), "qkv rows")
    refused(lib, L.mc_rope_kv8(one, 1028, one, one, one, one, one, 16, one, c, 1, 4, 1, None), "qkv rows")
    refused(lib, L.mc_rope_kv8(one, 1024, one, None, one, one, one, 16, one, c, 1, 4, 1, None), "null")
    refused(lib, L.mc_rope_kv8(one, 1024, one, one, one, one, one, 0, one, c, 1, 4, 1, None), "tables")
    refused(lib, L.mc_rope_kv8(one, 1024, one, one, one, one, one, 16, one, c, 1, 4, 0, None), "bad shape")
    refused(lib, L.mc_rope_kv8(one, 1024, one, one, one, one, one, 16, one, c, 1 << 30, 4, 1, None), "too many rows")
    assert L.mc_rope_kv8(one, 1024, one, one, one, one, one, 16, one, c, 0, 4, 1, None) == 0          # no rows: no launch
    refused(lib, L.mc_attn_decode8(one, 512, 128, c, None, None, 0, one, 512, None, 4, 1.0, None), "null")
    refused(lib, L.mc_attn_decode8(one, 516, 128, c, None, None, 0, one, 512, one, 4, 1.0, None), "16-byte")
    refused(lib, L.mc_attn_decode8(one, 512, 128, c, None, None, 0, one, 512, one, 5, 1.0, None), "5 query heads")
    refused(lib, L.mc_attn_decode8_rope(one, 1024, one, one, 16, c, None, None, 0, one, 512, one, 4, 1.0, None), "null")
    n = C.c_int64(0)
    refused(lib, L.mc_attn_decode8_workspace_bytes(0, 1, 128, 1, C.byref(n)), "bad arguments")


def test_output_rows_that_overlap(lib):
    L, c, one = lib.lib(), C.byref(cache_c(lib)), 4096
    for stride in (0, 511):                                                                # 4 heads of 128: 512
        refused(lib, L.mc_attn_decode8(one, 512, 128, c, None, None, 0, one, stride, one, 4, 1.0, None), "output rows overlap")
        refused(lib, L.mc_attn_decode8_rope(one, 1024, one, one, 16, c, one, None, 0, one, stride, one, 4, 1.0, None), "output rows overlap")


def test_bad_q4_calls(lib):
    L, one = lib.lib(), 4096

    def w(**kw):
        d = dict(codes=4096, ldc=128, scales=4096, lds=2, zeros=0, ldz=0, N=8, K=256, group=128)
        d.update(kw)
        return lib.Q4WeightC(*[d[n] for n, _ in lib.Q4WeightC._fields_])
    call = lambda ww, M=4, ldx=256, x=one, ldo=8, out=one, ws=None: L.mc_linear_q4_bf16(x, ldx, C.byref(ww), None, None, 0, out, ldo, M, 0, ws, None)
    for bad, text in ((dict(codes=0), "null weight"), (dict(group=96), "group 96"), (dict(K=192), "multiple"), (dict(N=0), "positive"), (dict(ldc=120), "16-byte"), (dict(ldc=112), "16-byte"),
                      (dict(codes=4100), "16-byte"), (dict(lds=1), "scales or zeros"), (dict(zeros=4096, ldz=1), "scales or zeros")):
        refused(lib, call(w(**bad)), text)
        refused(lib, L.mc_dequantize_q4_bf16(C.byref(w(**bad)), one, None), text)
    refused(lib, call(w(), M=65), "at most 64")
    refused(lib, call(w(), M=17), "workspace")
    refused(lib, call(w(), M=17, ws=4104), "workspace")
    n = C.c_int64(-1)
    assert L.mc_linear_q4_workspace_bytes(16, 256, C.byref(n)) == 0 and n.value == 0
    assert L.mc_linear_q4_workspace_bytes(17, 256, C.byref(n)) == 0 and n.value == 2 * 16 * 256 * 2
    refused(lib, L.mc_linear_q4_workspace_bytes(65, 256, C.byref(n)), "bad arguments")
    refused(lib, call(w(), M=-1), "at most 64")
    refused(lib, call(w(), ldx=252), "rows of x")
    refused(lib, call(w(), ldx=248), "rows of x")
    refused(lib, call(w(), x=None), "rows of x")
    refused(lib, call(w(), ldo=7), "bad output")
    assert call(w(), M=0) == 0
    refused(lib, L.mc_dequantize_q4_bf16(C.byref(w()), None, None), "null")
    refused(lib, L.mc_quantize_q4_bf16(one, 256, one, one, None, 8, 200, 128, None), "dividing K")
    refused(lib, L.mc_quantize_q4_bf16(one, 250, one, one, None, 8, 256, 128, None), "16-byte")
    refused(lib, L.mc_quantize_q4_bf16(None, 256, one, one, None, 8, 256, 128, None), "null")


def test_bad_logits_calls(lib):
    L = lib.lib()
    call = lambda **kw: L.mc_logits_process_f32(C.byref(lib.LogitsArgsC(**{**dict(logits=4096, out=4096, ld=8, ld_out=8, M=2, V=8), **kw})), None)
    refused(lib, call(logits=0), "null")
    refused(lib, call(V=0), "bad shape")
    refused(lib, call(M=-1), "bad shape")
    refused(lib, call(ld=7), "rows overlap")
    refused(lib, call(prompt_ids=4096, prompt_cols=-1), "negative")
    refused(lib, call(bias_ids=4096, bias=0, n_bias=2), "biases")
    refused(lib, call(bias_ids=4096, bias=4096, n_bias=1025), "biases")
    assert call(M=0) == 0


def test_wrappers_refuse_host_tensors():
    from modelcompose_amd import ops
    z = torch.zeros
    st = ops.BF16
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.Q4Weight(z(8, 64, dtype=torch.uint8), z(8, 1, dtype=st))
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.Kv8Cache(z(1, 1, 4, 64, dtype=torch.int8), z(1, 1, 4), z(1, 1, 4, 64, dtype=torch.int8), z(1, 1, 4))
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.logits_process(z(2, 8))
    with pytest.raises(ValueError, match="device"):
        ops.quantize_q4(z(8, 128, dtype=st))
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.linear_q4(z(1, 64, dtype=st), None)
    with pytest.raises(ValueError, match="no CPU fallback"):
        ops.attn_decode8(z(1, 1, 64, dtype=st), None)


# ---- what the bounds of the 4-bit linears' sums reject -------------------------------------------------------------------------------
def _q4_sum(x, codes, scales, zeros, group, group_dtype=torch.float32, sum_dtype=torch.float32, drop=0):
    """linear_q4's arithmetic in torch: fp32 sums per group, scaled, added up - with the group sums or the running sum rounded to fewer bits, or the last `drop` columns left out."""
    from lowp_bounds import split
    N, G = scales.shape
    q, s = split(codes).float().view(N, G, group), scales.float()
    z = torch.full_like(s, 8.0) if zeros is None else zeros.float()
    x = x.float().clone()
    if drop:
        x[:, -drop:] = 0
    xg, y = x.view(len(x), G, group), torch.zeros(len(x), N)
    for g in range(G):
        a = (xg[:, g] @ q[:, g].t() - xg[:, g].sum(1, keepdim=True) * z[:, g]).to(group_dtype).float()
        y = (y + a * s[:, g]).to(sum_dtype).float()
    return y.double()


@pytest.mark.parametrize("M", [1, 16, 48])
@pytest.mark.parametrize("N,K,group,zeros", [(33, 11008, 128, False), (250, 4096, 128, True), (129, 2752, 64, True), (40, 544, 32, False)])
def test_bounds_of_the_4_bit_sums_reject_what_they_should(M, N, K, group, zeros):
    from lowp_bounds import q4_sums, whole_numbers
    g = torch.Generator().manual_seed(N * 41 + M)
    codes = torch.randint(0, 256, (N, K // 2), generator=g).to(torch.uint8)
    scales = (torch.rand(N, K // group, generator=g) * 0.01 + 0.001).bfloat16()
    z = torch.randint(0, 16, (N, K // group), generator=g).to(torch.uint8) if zeros else None
    x = torch.randn(M, K, generator=g).bfloat16() + 0.25
    ref, bound = q4_sums(x, codes, scales, z, group)
    inside = lambda **kw: bool(((_q4_sum(x, codes, scales, z, group, **kw) - ref).abs() <= bound).all())
    wrong = (dict(group_dtype=torch.bfloat16), dict(sum_dtype=torch.bfloat16), dict(drop=1), dict(drop=8))
    assert inside()
    for kw in wrong:
        assert not inside(**kw), kw
    x, codes, scales, z = whole_numbers(g, M, N, K, group, zeros, torch.bfloat16)
    ref = q4_sums(x, codes, scales, z, group)[0]
    assert torch.equal(_q4_sum(x, codes, scales, z, group), ref)
    for kw in wrong:
        assert not torch.equal(_q4_sum(x, codes, scales, z, group, **kw), ref), kw
