"""CPU: sdmi_cross_attention and sdmi_lora_gemm refuse bad arguments with an error code and a message, before any launch (the
pointers here are never followed), and their workspace sizes."""
import pytest

from stable_diffusion_amd import _lib as L

P = 0x10000000     # an aligned address that is never followed

ATT = dict(q=P, ldq=128, sq=128, k=P, ldk=128, sk=1280, v=P, ldv=128, sv=1280, o=P, ldo=128, so=128, batch=2, contexts=2, heads=2, kv_heads=2, dim=64, nq=1, nkv=10,
           index=None, lens=None, qr=None, sqr=0, kr=None, skr=0, scale=0.125, ws=None, ws_bytes=0, stream=None)
LORA = dict(x=P, ldx=64, w=P, ldw=64, out=P, ldo=64, m=100, n=64, k=64, bias=None, residual=None, ldr=0, a=P, b=P, scale=P, adapters=2, rank=8, groups=1, ids=P, rows=1,
            flags=0, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(o=None), "null"), (dict(batch=0), "shape"), (dict(heads=3), "shape"), (dict(kv_heads=0), "shape"),
    (dict(dim=60), "shape"), (dict(dim=264, kv_heads=1, heads=1, ldq=264, ldk=264, ldv=264, ldo=264), "shape"), (dict(dim=0), "shape"), (dict(nq=0), "shape"),
    (dict(nkv=-1), "shape"), (dict(contexts=0), "contexts"), (dict(contexts=3), "index"), (dict(ldq=120), "stride"), (dict(ldq=132), "multiples"), (dict(ldk=64), "stride"),
    (dict(ldo=66), "multiples"), (dict(ldk=1 << 22), "too large"), (dict(sk=1284), "alignment"), (dict(q=P + 8), "alignment"), (dict(o=P + 4), "alignment"),
    (dict(qr=P), "together"), (dict(kr=P), "together"), (dict(index=P + 2), "alignment"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=2e15), "scale"), (dict(nkv=1 << 30), "shape"), (dict(nq=1 << 30), "shape"),
    (dict(nq=(1 << 30) - 1), "grid"),
])
def test_attention_refuses(change, word):
    with pytest.raises(L.SdmiError, match=word):
        L.call("sdmi_cross_attention", *{**ATT, **change}.values())


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(ids=None), "null"), (dict(ws=None), "workspace"), (dict(ws=P + 8), "workspace"), (dict(n=24, groups=2), "shape"), (dict(flags=1, bias=P + 4), "alignment"), (dict(b=None), "null"), (dict(m=0), "shape"), (dict(n=60), "shape"), (dict(k=60), "shape"),
    (dict(rank=12), "shape"), (dict(rank=0), "shape"), (dict(rank=264), "shape"), (dict(groups=0), "shape"), (dict(groups=3), "shape"), (dict(adapters=0), "adapters"),
    (dict(rows=0), "rows per id"), (dict(flags=8), "flags"), (dict(flags=1), "bias"), (dict(flags=4), "residual"), (dict(flags=4, residual=P, ldr=32), "residual"),
    (dict(ldx=32), "strides"), (dict(ldw=68), "strides"), (dict(ldo=60), "strides"), (dict(ldx=1 << 22), "too large"), (dict(x=P + 8), "alignment"),
    (dict(flags=4, residual=P + 8, ldr=64), "alignment"), (dict(ids=P + 2), "alignment"), (dict(ws_bytes=8), "workspace"), (dict(m=1 << 30), "shape"),
    (dict(n=1 << 27, ldo=1 << 27), "shape"),
    (dict(m=(1 << 30) - 64, rows=(1 << 30) - 64, rank=40, ws_bytes=1 << 40), "grid"),
])
def test_lora_refuses(change, word):
    with pytest.raises(L.SdmiError, match=word):
        L.call("sdmi_lora_gemm", *{**LORA, **change}.values())


def test_no_cpu_fallback():
    import torch
    from stable_diffusion_amd import engine as E
    h = E.act_dtype()
    a = E.Act(torch.zeros((2, 8, 64), dtype=h), 2, 1, 8, 64)
    with pytest.raises(L.SdmiError, match="cpu"):
        E.cross_attention(a, a, a, 1)
    pack = E.LoraPack(torch.zeros((1, 8, 64), dtype=h), torch.zeros((1, 64, 8), dtype=h), torch.ones(1))
    with pytest.raises(L.SdmiError, match="cpu"):
        E.lora_gemm(a, torch.zeros((64, 64), dtype=h), 64, pack, torch.zeros(2, dtype=torch.int32))


def test_attention_refuses_grids_whose_size_passes_64_bits():
    """2^64 blocks and more, whose number comes out as 0 or a few."""
    wide = dict(heads=1 << 18, kv_heads=1 << 18, dim=8, ldq=1 << 21, ldk=1 << 21, ldv=1 << 21, ldo=1 << 21)
    for change in (dict(wide, batch=1 << 30, nq=1 << 23), dict(wide, batch=(1 << 30) + 1, nq=1 << 23), dict(wide, batch=1 << 30, nq=1 << 24), dict(wide, batch=1 << 24, nq=1)):
        args = {**ATT, "contexts": 1, **change}
        with pytest.raises(L.SdmiError, match="grid"):
            L.call("sdmi_cross_attention", *args.values())
        assert L.load().sdmi_cross_attention_ws_bytes(args["batch"], args["heads"], args["kv_heads"], args["dim"], args["nq"], args["nkv"]) == 0


@pytest.mark.parametrize("m", [1, 40])
def test_lora_refuses_a_few_rows_by_too_many_columns(m):
    with pytest.raises(L.SdmiError, match="grid"):
        L.call("sdmi_lora_gemm", *{**LORA, "m": m, "n": (1 << 27) - 8, "ldo": 1 << 27}.values())


def test_out_apart_from_operands():
    """An `out` whose columns share memory with an operand is refused, however the two are cut from one storage; the residual may
    be out itself.  (Host tensors: what passes here is refused as such, before any launch.)"""
    import torch
    from stable_diffusion_amd import engine as E
    h = E.act_dtype()
    big = torch.zeros((4, 8, 192), dtype=h)
    act = lambda buf, off, c: E.Act(buf, buf.shape[0], 1, buf.shape[1], buf.shape[2]).cols(off, c)
    pack = E.LoraPack(torch.zeros((1, 8, 64), dtype=h), torch.zeros((1, 64, 8), dtype=h), torch.ones(1))
    w, ids, x = torch.zeros((64, 64), dtype=h), torch.zeros(2, dtype=torch.int32), act(torch.zeros((2, 8, 64), dtype=h), 0, 64)
    lora = lambda a, **kw: E.lora_gemm(a, w, 64, pack, ids, **kw)
    att = lambda q, k, o: E.cross_attention(q, k, k, 1, out=o)
    low, mid, top = big[0:2], big[1:3], big[2:4]
    flat = big.view(-1)[:2 * 8 * 64].view(2, 8, 64)
    shared = [lambda: lora(x, residual=act(low, 0, 64), out=act(low, 8, 64)),       # a residual that other columns overwrite
              lambda: lora(x, residual=act(low, 0, 64), out=act(mid, 0, 64)), lambda: lora(x, residual=act(low, 64, 64), out=act(mid, 32, 64)),
              lambda: lora(act(low, 0, 64), out=act(mid, 0, 64)), lambda: lora(act(mid, 0, 64), out=act(low, 40, 64)), lambda: lora(act(flat, 0, 64), out=act(low, 128, 64)),
              lambda: lora(x, residual=act(flat, 0, 64), out=act(low, 0, 64)),
              lambda: att(act(mid, 0, 64), x, act(low, 0, 64)), lambda: att(x, act(low, 128, 64), act(mid, 120, 64))]
    apart = [lambda: lora(x, residual=act(low, 8, 64), out=act(low, 8, 64)), lambda: lora(x, residual=act(low, 0, 64), out=act(low, 64, 64)),
             lambda: lora(x, residual=act(low, 0, 64), out=act(top, 0, 64)), lambda: lora(act(low, 0, 64), out=act(mid, 64, 64)), lambda: lora(act(mid, 128, 64), out=act(low, 64, 64)),
             lambda: att(act(low, 0, 64), act(mid, 64, 64), act(low, 128, 64)), lambda: att(act(low, 0, 64), act(low, 0, 64), act(top, 0, 64))]
    for f in shared:
        with pytest.raises(L.SdmiError, match="memory"):
            f()
    for f in apart:
        with pytest.raises(L.SdmiError, match="cpu"):
            f()


def test_lora_refuses_a_residual_or_out_of_another_type():
    import torch
    from stable_diffusion_amd import engine as E
    h = E.act_dtype()
    act = lambda t: E.Act(torch.zeros((2, 8, 64), dtype=t), 2, 1, 8, 64)
    pack = E.LoraPack(torch.zeros((1, 8, 64), dtype=h), torch.zeros((1, 64, 8), dtype=h), torch.ones(1))
    w, ids = torch.zeros((64, 64), dtype=h), torch.zeros(2, dtype=torch.int32)
    for t in (torch.float32, torch.int16, torch.bfloat16 if h is torch.float16 else torch.float16):
        for kw in (dict(residual=act(t)), dict(out=act(t))):
            with pytest.raises(L.SdmiError, match="one type"):
                E.lora_gemm(act(h), w, 64, pack, ids, **kw)


def _packed(fmt, args):
    return fmt.pack(*(0 if v is None else v for v in args.values()))


@pytest.mark.parametrize("change", [dict(q=None), dict(dim=60), dict(contexts=3), dict(ldk=64), dict(sk=1284), dict(o=P + 4), dict(kr=P), dict(index=P + 2), dict(scale=-1.0),
                                    dict(nkv=1 << 32), dict(ldq=(1 << 32) + 128), dict(batch=-(1 << 40))])
def test_attention_in_one_block_refuses_the_same(change):
    with pytest.raises(L.SdmiError, match="cross_attention: ") as packed:
        L.call("sdmi_cross_attention_packed", _packed(L.CROSS_ATTENTION_ARGS, {**ATT, **change}))
    if all(not isinstance(v, int) or abs(v) < 1 << 31 for v in change.values()):
        with pytest.raises(L.SdmiError) as plain:
            L.call("sdmi_cross_attention", *{**ATT, **change}.values())
        assert str(packed.value).split(": ", 1)[1] == str(plain.value).split(": ", 1)[1]


@pytest.mark.parametrize("change", [dict(x=None), dict(ws=None), dict(rank=12), dict(groups=3), dict(rows=0), dict(flags=8), dict(flags=4), dict(ldw=68), dict(ids=P + 2),
                                    dict(ws_bytes=8), dict(m=1 << 32), dict(rows=1 << 31), dict(flags=1 << 32), dict(flags=-1)])
def test_lora_in_one_block_refuses_the_same(change):
    with pytest.raises(L.SdmiError, match="lora_gemm: ") as packed:
        L.call("sdmi_lora_gemm_packed", _packed(L.LORA_GEMM_ARGS, {**LORA, **change}))
    if all(v is None or 0 <= v < 1 << 31 for v in change.values()):
        with pytest.raises(L.SdmiError) as plain:
            L.call("sdmi_lora_gemm", *{**LORA, **change}.values())
        assert str(packed.value).split(": ", 1)[1] == str(plain.value).split(": ", 1)[1]


def test_blocks_are_the_headers_structs():
    """Every field of the two structs is one word of the format, in order."""
    import os
    import re
    from conftest import ROOT
    src = open(os.path.join(ROOT, "include", "sdmi.h")).read()
    for name, fmt in (("sdmi_cross_attention_args", L.CROSS_ATTENTION_ARGS), ("sdmi_lora_gemm_args", L.LORA_GEMM_ARGS)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1), flags=re.S)
        want = ""
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            for i, field in enumerate(decl.split(",")):
                want += "Q" if "*" in field else ("d" if decl.startswith("double") else "q")
        have = re.sub(r"(\d+)(.)", lambda m: m.group(2) * int(m.group(1)), fmt.format)
        assert have == want and fmt.size == 8 * len(want), name


def test_workspace_sizes():
    lib = L.load()
    assert lib.sdmi_cross_attention_ws_bytes(2, 5, 5, 64, 9216, 77) == 0            # one pass
    assert lib.sdmi_cross_attention_ws_bytes(1, 2, 2, 64, 1, 5000) > 0              # keys in pieces
    assert lib.sdmi_cross_attention_ws_bytes(1, 2, 2, 60, 1, 5000) == 0             # refused shapes need nothing
    assert lib.sdmi_lora_gemm_ws_bytes(100, 96, 64, 16, 3, 1) >= 100 * 48 * 2
    assert lib.sdmi_lora_gemm_ws_bytes(100, 96, 64, 12, 3, 1) == 0
    assert lib.sdmi_lora_gemm_ws_bytes(1, 96, 64, 16, 1, 1) == 0                       # one launch: nothing to hand over
    for m in (1, 40, 100, 5000):                                                       # one id for all rows, however it is said
        for rank in (16, 64):
            assert lib.sdmi_lora_gemm_ws_bytes(m, 96, 64, rank, 1, 2 ** 31 - 1) == lib.sdmi_lora_gemm_ws_bytes(m, 96, 64, rank, 1, m)
