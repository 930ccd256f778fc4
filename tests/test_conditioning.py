"""EncoderStates and AdapterSet through the model's own layers: a transformer block, the UNet and the sampler, against the oracle
run sample by sample with shortened contexts, masked attention and merged weights (W + scale up down).

The gates are those of the same modules without either (test_gpu_blocks.py): an adapter adds two roundings to 16 bits to a
projection (t, and the factors), as many as the projection itself has."""
import copy

import numpy as np
import pytest
import torch

import sd_oracle as O
from conftest import rel_err
from stable_diffusion_amd import engine as E, _lib as L
from stable_diffusion_amd.conditioning import AdapterSet, EncoderStates, GuidancePair
from stable_diffusion_amd.synth import fill_state_dict, make_inputs

DEV = "cuda"
T = torch.from_numpy


def _rand(rs, *shape, std=1.0):
    return T((rs.standard_normal(shape) * std).astype(np.float32))


def _adapter(rs, sd, names, rank, scale):
    """{layer: (down, up, scale)} whose product is about as large as the weight it joins."""
    ad = {}
    for i, n in enumerate(names):
        w = sd[n + ".weight"]
        r = rank + 3 * i % 5
        ad[n] = (_rand(rs, r, w.shape[1], std=w.shape[1] ** -0.5), _rand(rs, w.shape[0], r, std=r ** -0.5)) + ((scale,) if scale != 1.0 else ())
    return ad


def _merged(sd, adapters, i, ic):
    """The weights that sample with adapter i and context with adapter ic sees."""
    out = dict(sd)
    for who, context in ((i, False), (ic, True)):
        for n, v in (adapters[who].items() if 0 <= who < len(adapters) else ()):
            if (".attn2." in n and n.endswith((".to_k", ".to_v"))) == context:
                out[n + ".weight"] = sd[n + ".weight"] + (v[2] if len(v) > 2 else 1.0) * (v[1] @ v[0])
    return out


class _Masked(object):
    """oracle attention in which queries see the keys whose set meets theirs (self-attention stays whole)."""

    def __init__(self, qsets, ksets):
        self.q, self.k, self.own = qsets, ksets, O.attention

    def __call__(self, q, k, v):
        if k.shape[1] != self.k.shape[0] or q.shape[1] == k.shape[1]:
            return self.own(q, k, v)
        qs = self.q
        while qs.numel() > q.shape[1]:
            qs = qs[::2, ::2]
        seen = (qs.reshape(-1)[:, None] & self.k[None, :]) != 0
        s = (q @ k.transpose(1, 2)) * 0.125
        p = torch.softmax(s.masked_fill(~seen, float("-inf")), dim=-1)
        return torch.where(seen.any(1)[None, :, None], p, torch.zeros_like(p)) @ v


def _gate(got, ref, max_tol, l2_tol, what):
    f = 8.0 if E.act_dtype() == torch.bfloat16 else 1.0
    m, l2 = rel_err(got.float().cpu().numpy(), ref.numpy())
    print("%s: max-rel %.3e  rel-L2 %.3e" % (what, m, l2), flush=True)
    assert m <= max_tol * f and l2 <= l2_tol * f, (what, m, l2)


# ------------------------------------------------------------------------------------------------------------ one transformer
@pytest.mark.gpu
@pytest.mark.parametrize("regions", [False, True])
@pytest.mark.parametrize("adapted", [False, True])
def test_transformer_with_states_and_adapters(adapted, regions, monkeypatch):
    from layers.SpatialTransformer import SpatialTransformer
    m = SpatialTransformer(128, 2)
    sd = {k: v.clone() for k, v in fill_state_dict(m.state_dict(), seed=12).items()}
    m = m.to(DEV).eval()
    rs = np.random.RandomState(3)
    b, h, w, t = 3, 12, 10, 90
    x, tokens = _rand(rs, b, 128, h, w), _rand(rs, 2, t, 1024)
    lens, index, ids, cids = [t, 31], [1, 0, 1], [1, -1, 0], [0, 1]
    kr, qr = T(rs.randint(0, 4, (2, t))), T(rs.randint(0, 4, (b, h, w)))
    sets = dict(key_regions=kr, query_regions=qr) if regions else {}
    pre = "transformer_blocks.0."
    ads = [_adapter(rs, sd, [pre + n for n in ("attn1.to_q", "attn1.to_k", "attn1.to_v", "attn1.to_out.0", "attn2.to_q", "attn2.to_k", "attn2.to_v")], 4, 0.5),
           _adapter(rs, sd, [pre + n for n in ("attn1.to_v", "attn2.to_v", "attn2.to_out.0")], 20, 1.0)]
    if adapted:
        AdapterSet(m, ads).select(ids, cids).attach()
    y = m(x.to(DEV), context=EncoderStates(tokens.to(DEV), lens, index, **sets))
    for i in range(b):
        c = index[i]
        one = _merged(sd, ads, ids[i], cids[c]) if adapted else sd
        if regions:
            monkeypatch.setattr(O, "attention", _Masked(qr[i], kr[c][:lens[c]]))
        ref = O.spatial_transformer({"m." + k: v for k, v in one.items()}, "m", x[i:i + 1], tokens[c:c + 1, :lens[c]])
        monkeypatch.undo()
        _gate(y[i:i + 1], ref, 3e-3, 2e-3, "sample %d" % i)


# ------------------------------------------------------------------------------------------------------------ the UNet
@pytest.fixture(scope="module")
def net():
    from Unet import Unet
    unet = Unet()
    sd = {k: v.clone() for k, v in fill_state_dict(unet.state_dict(), seed=0).items()}
    return unet.to(DEV).eval(), sd


def _attention_layers(sd, every):
    return [n[:-7] for i, n in enumerate(sorted(k for k in sd if k.endswith((".to_q.weight", ".to_k.weight", ".to_v.weight", ".to_out.0.weight")))) if i % every == 0]


def _unet_adapters(rs, sd, strength):
    return [_adapter(rs, sd, _attention_layers(sd, 1), 4, strength), _adapter(rs, sd, _attention_layers(sd, 3), 16, strength)]


@pytest.mark.gpu
def test_unet_with_states_regions_and_adapters(net, monkeypatch):
    unet, sd = net
    rs = np.random.RandomState(8)
    x, tokens, t = _rand(rs, 2, 9, 16, 16), _rand(rs, 3, 120, 1024), torch.tensor([481, 481])
    lens, index, ids, cids = [120, 50, 77], [2, 0], [0, 1], [1, -1, 0]
    kr, qr = T(rs.randint(1, 8, (3, 120))), T(rs.randint(0, 8, (2, 16, 16)))
    ads = _unet_adapters(rs, sd, 0.3)
    plain = unet(x.to(DEV), timesteps=t.to(DEV), context=tokens[:2, :77].to(DEV))
    try:
        unet.set_adapters(AdapterSet(unet, ads).select(ids, cids))
        states = EncoderStates(tokens.to(DEV), lens, index, kr, qr)
        y = unet(x.to(DEV), timesteps=t.to(DEV), context=states)
        assert torch.equal(unet(x.to(DEV), timesteps=t.to(DEV), context=unet.precompute_context(states)), y)
    finally:
        unet.set_adapters(None)
    for i in range(2):
        c = index[i]
        monkeypatch.setattr(O, "attention", _Masked(qr[i], kr[c][:lens[c]]))
        ref = O.unet_forward(_merged(sd, ads, ids[i], cids[c]), x[i:i + 1], t[i:i + 1], tokens[c:c + 1, :lens[c]])
        monkeypatch.undo()
        _gate(y[i:i + 1], ref, 7e-3, 6e-3, "Unet.forward, sample %d" % i)
    # what has neither runs as before
    assert torch.equal(unet(x.to(DEV), timesteps=t.to(DEV), context=tokens[:2, :77].to(DEV)), plain)


@pytest.mark.gpu
def test_states_of_whole_contexts_are_plain_contexts(net):
    unet, sd = net
    rs = np.random.RandomState(9)
    x, ctx, t = _rand(rs, 2, 9, 16, 16).to(DEV), _rand(rs, 2, 77, 1024), torch.tensor([481, 481]).to(DEV)
    want = unet(x, timesteps=t, context=ctx.to(DEV)).cpu()
    for states in (EncoderStates(ctx.to(DEV)), EncoderStates(ctx.to(DEV), [77, 77], [0, 1]), EncoderStates(ctx.flip(0).to(DEV), None, [1, 0])):
        _gate(unet(x, timesteps=t, context=states), want, 7e-3, 6e-3, "whole contexts")
    shared = unet(x, timesteps=t, context=EncoderStates(ctx[:1].to(DEV)))       # one context for any batch
    _gate(shared, unet(x, timesteps=t, context=ctx[:1].expand(2, -1, -1).contiguous().to(DEV)).cpu(), 7e-3, 6e-3, "one shared context")


@pytest.mark.gpu
def test_a_callers_own_graph_sees_new_states_and_adapters(net):
    """Unet.forward captured by the caller: what EncoderStates.copy_ and AdapterSet.select write reaches the replays."""
    unet, sd = net
    rs = np.random.RandomState(12)
    dev = lambda v: v.to(DEV)
    x, t = dev(_rand(rs, 2, 9, 16, 16)), torch.tensor([481, 481]).to(DEV)
    make = lambda lens, index: EncoderStates(dev(_rand(rs, 2, 60, 1024)), lens, index, T(rs.randint(1, 4, (2, 60))), T(rs.randint(0, 4, (2, 16, 16))))
    states, adapters = make([60, 20], [0, 1]), AdapterSet(unet, _unet_adapters(rs, sd, 0.2)).select([0, 1], [1, 0])
    try:
        unet.set_adapters(adapters)
        unet(x, timesteps=t, context=states)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = unet(x, timesteps=t, context=states)
        for step, (lens, index, ids, cids) in enumerate((([60, 20], [0, 1], [0, 1], [1, 0]), ([7, 59], [1, 1], [1, -1], [-1, 0]), ([0, 60], [0, 1], [-1, -1], [1, 1]))):
            states.copy_(make(lens, index))
            adapters.select(ids, cids)
            want = unet(x, timesteps=t, context=states).clone()
            torch.cuda.synchronize()
            for _ in range(2):
                g.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want), step
    finally:
        unet.set_adapters(None)


# ------------------------------------------------------------------------------------------------------------ the sampler
@pytest.mark.gpu
@pytest.mark.parametrize("dual", [True, False])
def test_sampler_replays_one_step_for_other_states_and_adapters(net, dual):
    """One captured step serves batches with other lengths, contexts and adapters: the bits of the eager loop."""
    from stable_diffusion_amd.sampler import Sampler
    unet, sd = net
    rs = np.random.RandomState(4)
    dev = lambda v: v.to(DEV)
    sets = [AdapterSet(unet, _unet_adapters(rs, sd, 0.2)), AdapterSet(unet, _unet_adapters(rs, sd, 0.2)[1:])]
    graph, eager = Sampler(unet, None, dual_stream=dual), Sampler(unet, None, dual_stream=dual)
    seen = []
    try:
        for step, (use, ids) in enumerate(((0, [0, 1]), (0, [-1, 0]), (1, [0, -1]), (0, [1, 1]))):
            inp = make_inputs(2, 16, 4, seed=30 + step)
            cond = EncoderStates(dev(_rand(rs, 2, 100, 1024)), [100 - 9 * step, 40 + step])
            uncond = EncoderStates(dev(_rand(rs, 2, 77, 1024)), [77, 7 + step])
            unet.set_adapters(sets[use].select(ids))
            args = (4, cond, uncond, dev(inp["c_concat"]), dev(inp["x_T"]), [dev(n) for n in inp["noises"]], 7.5)
            xg, _ = graph.sample(*args, decode=False, use_graph=True)
            if step == 0:
                first = graph._graph
            if step == 1:
                assert graph._graph is first
            xe, _ = eager.sample(*args, decode=False, use_graph=False)
            assert torch.isfinite(xe).all() and torch.equal(xg, xe), step
            seen.append(xe)
        sets[0].detach()                # taken out layer by layer, behind the model's back
        xg, _ = graph.sample(*args, decode=False, use_graph=True)
        xe, _ = eager.sample(*args, decode=False, use_graph=False)
        assert torch.equal(xg, xe) and not torch.equal(xe, seen[-1])
        sets[0].attach()
        xg, _ = graph.sample(*args, decode=False, use_graph=True)
        assert torch.equal(xg, seen[-1])
        unet.set_adapters(None)
        xg, _ = graph.sample(*args, decode=False, use_graph=True)
        xe, _ = eager.sample(*args, decode=False, use_graph=False)
        assert torch.equal(xg, xe) and not torch.equal(xe, seen[-1])
    finally:
        unet.set_adapters(None)


@pytest.mark.gpu
def test_sampler_takes_one_context_for_the_batch_and_plain_negatives(net):
    from stable_diffusion_amd.sampler import Sampler
    unet, _ = net
    inp = make_inputs(2, 16, 2, seed=41)
    dev = lambda v: v.to(DEV)
    rest = (dev(inp["c_concat"]), dev(inp["x_T"]), [dev(n) for n in inp["noises"]], 7.5)
    one = dev(_rand(np.random.RandomState(2), 1, 90, 1024))
    got = [Sampler(unet, None, dual_stream=d).sample(2, EncoderStates(one), dev(inp["uncond"]), *rest, decode=False)[0] for d in (True, False)]
    want = Sampler(unet, None).sample(2, EncoderStates(one.expand(2, -1, -1).contiguous()), EncoderStates(dev(inp["uncond"])), *rest, decode=False)[0]
    for g in got:
        _gate(g, want.cpu(), 1.5e-2, 1.5e-2, "one context")


@pytest.mark.gpu
def test_sampler_takes_regions_beside_plain_negatives(net):
    """Both halves in one batch (the plain one in every region) and one by one (the plain one without regions)."""
    from stable_diffusion_amd.sampler import Sampler
    unet, _ = net
    rs = np.random.RandomState(6)
    inp = make_inputs(2, 16, 2, seed=43)
    dev = lambda v: v.to(DEV)
    rest = (dev(inp["c_concat"]), dev(inp["x_T"]), [dev(n) for n in inp["noises"]], 7.5)
    cond = EncoderStates(dev(_rand(rs, 2, 100, 1024)), [100, 60], None, T(rs.randint(1, 4, (2, 100))), T(rs.randint(0, 4, (2, 16, 16))))
    one = Sampler(unet, None, dual_stream=False).sample(2, cond, dev(inp["uncond"]), *rest, decode=False)[0]
    two = Sampler(unet, None, dual_stream=True).sample(2, cond, dev(inp["uncond"]), *rest, decode=False)[0]
    _gate(two, one.cpu(), 1.5e-2, 1.5e-2, "regions beside plain negatives")
    graph = Sampler(unet, None, dual_stream=False)
    for _ in range(2):
        assert torch.equal(graph.sample(2, cond, dev(inp["uncond"]), *rest, decode=False, use_graph=True)[0], one)


# ------------------------------------------------------------------------------------------------------------ refusals and layout
def test_cat_keeps_each_side_to_its_own_contexts(monkeypatch):
    monkeypatch.setattr(E, "_need_cuda", lambda t, what: None)
    a = EncoderStates(torch.zeros(1, 5, 8), lens=[3])
    b = EncoderStates(torch.ones(2, 7, 8), index=[1, 0, 5])
    c = EncoderStates.cat(a, b, batch=3)
    assert tuple(c.tokens.shape) == (3, 7, 8) and c.batch == 6
    assert c.lens.tolist() == [3, 7, 7] and c.index.tolist() == [0, 0, 0, 2, 1, -1]
    plain = EncoderStates.cat(EncoderStates(torch.zeros(2, 5, 8)), EncoderStates(torch.zeros(2, 5, 8)))
    assert plain.index is None and plain.lens is None and plain.batch == 4
    with pytest.raises(L.SdmiError, match="say of which"):
        EncoderStates.cat(a, b)
    r = EncoderStates(torch.zeros(1, 5, 8), key_regions=torch.ones(1, 5, dtype=torch.int64), query_regions=torch.arange(5 * 3).view(1, 5, 3))
    assert r.regions(3, 2).tolist() == [[0, 2, 6, 8, 12, 14]] and r.regions(1, 1).tolist() == [[0]]
    with pytest.raises(L.SdmiError, match="no level"):
        r.regions(4, 2)
    whole = EncoderStates.cat(EncoderStates(torch.zeros(1, 4, 8)), r, batch=2)          # in every region beside one that has some
    assert whole.batch == 3 and whole.lens.tolist() == [4, 5] and whole.index.tolist() == [0, 0, 1]
    assert whole.key_regions.tolist() == [[-1, -1, -1, -1, 0], [1] * 5] and whole.query_regions[:2].eq(-1).all() and torch.equal(whole.query_regions[2:], r.query_regions)
    with pytest.raises(L.SdmiError, match="query_regions of"):
        EncoderStates.cat(r, EncoderStates(torch.zeros(1, 5, 8), key_regions=torch.ones(1, 5, dtype=torch.int64), query_regions=torch.zeros(1, 3, 5, dtype=torch.int64)))
    assert EncoderStates(torch.zeros(1, 2, 8), key_regions=torch.tensor([[0xffffffff, 1]]), query_regions=torch.zeros(2, 1, 1, dtype=torch.int32)).key_regions.tolist() == [[-1, 1]]


def test_states_refuse(monkeypatch):
    with pytest.raises(L.SdmiError):
        EncoderStates(torch.zeros(2, 5, 8))                     # not on the GPU
    monkeypatch.setattr(E, "_need_cuda", lambda t, what: None)
    tok = torch.zeros(2, 5, 8)
    for kw in (dict(lens=[1]), dict(lens=[1.0, 2.0]), dict(key_regions=torch.zeros(2, 5, dtype=torch.int32)),
               dict(query_regions=torch.zeros(2, 4, 4, dtype=torch.int32)), dict(key_regions=torch.zeros(2, 4, dtype=torch.int32), query_regions=torch.zeros(2, 4, 4, dtype=torch.int32)),
               dict(key_regions=torch.zeros(2, 5, dtype=torch.int32), query_regions=torch.zeros(3, 4, 4, dtype=torch.int32)),
               dict(key_regions=torch.zeros(2, 5, dtype=torch.int32), query_regions=torch.zeros(2, 16, dtype=torch.int32))):
        with pytest.raises(L.SdmiError):
            EncoderStates(tok, **kw)
    with pytest.raises(L.SdmiError):
        EncoderStates(tok[0])
    with pytest.raises(L.SdmiError):
        EncoderStates(tok).copy_(EncoderStates(tok, [1, 2]))


def _layer():
    from layers.SpatialTransformer import SpatialTransformer
    return SpatialTransformer(64, 1)


def test_adapters_refuse(monkeypatch):
    m = _layer()
    q = "transformer_blocks.0.attn1.to_q"
    ok = (torch.zeros(4, 64), torch.zeros(64, 4))
    with pytest.raises(L.SdmiError):
        AdapterSet(m, [{q: ok}])                                # not on the GPU
    monkeypatch.setattr(E, "_need_cuda", lambda t, what: None)
    for ads in ([], [{}], [{"transformer_blocks.0.ff.net.2": ok}], [{"nothing.to_q": ok}], [{q: (ok[0], torch.zeros(64, 5))}], [{q: (torch.zeros(4, 32), ok[1])}],
                [{q: (torch.zeros(257, 64), torch.zeros(64, 257))}], [{q: (torch.zeros(0, 64), torch.zeros(64, 0))}], [{q: (ok[0], ok[1] + float("nan"))}],
                [{q: (ok[0], ok[1], float("inf"))}]):
        with pytest.raises(L.SdmiError):
            AdapterSet(m, ads)
    s = AdapterSet(m, [{q: ok}, {"transformer_blocks.0.attn2.to_k": (torch.zeros(3, 1024), torch.zeros(64, 3))}])
    with pytest.raises(L.SdmiError, match="select"):
        s.ids_for(2)
    s.select([0, 1])
    assert s.ids_for(2).tolist() == [0, 1] and s.ids_for(4).tolist() == [0, 1, 0, 1] and s.ids_for_contexts(2, False).tolist() == [0, 1]
    with pytest.raises(L.SdmiError):
        s.ids_for(3)
    with pytest.raises(L.SdmiError, match="context_ids"):
        s.ids_for_contexts(2, True)
    with pytest.raises(L.SdmiError):
        s.select([])
    kept = s.ids.data_ptr()
    s.select([1, 1, 0], [5])
    s.select([1, 0], [7])
    assert s.ids.data_ptr() == kept and s.ids_for_contexts(1, True).tolist() == [7]
    s.attach()
    block = m.transformer_blocks[0]
    assert block.attn1.adapters.pack("qkv").groups == 3 and block.attn2.adapters.pack("kv").rank == 8 and block.attn2.adapters.pack("q") is None
    with pytest.raises(L.SdmiError, match="other kind"):
        block.attn2.adapters.pack("qkv")
    twin = copy.deepcopy(m)
    assert twin.transformer_blocks[0].attn1.adapters.pack("qkv") is not None
    s.detach()
    assert block.attn1.adapters is None and block.attn2.adapters is None
    from stable_diffusion_amd.sampler import Sampler
    assert Sampler.adapters_of(m) == ([], ())
    s.attach()
    held, key = Sampler.adapters_of(m)
    s.select([0, 0, 0, 1])
    assert [la for _, la in s.layers] == held and Sampler.adapters_of(m)[1] != key


def test_a_set_belongs_to_its_model(monkeypatch):
    from Unet import Unet
    monkeypatch.setattr(E, "_need_cuda", lambda t, what: None)
    with torch.device("meta"):
        unet = Unet()
    with pytest.raises(L.SdmiError, match="another model"):
        unet.set_adapters(AdapterSet(_layer(), [{"transformer_blocks.0.attn1.to_q": (torch.zeros(4, 64), torch.zeros(64, 4))}]))

# ------------------------------------------------------------------------------------------------------------ adapters of contexts, side by side
def _set_on_host(monkeypatch, n=3):
    """An AdapterSet with n adapters on a layer's to_k (attn2), on the host."""
    monkeypatch.setattr(E, "_need_cuda", lambda t, what: None)
    return AdapterSet(_layer(), [{"transformer_blocks.0.attn2.to_k": (torch.zeros(3, 1024), torch.zeros(64, 3))}] * n)


def _side(n, index=None):
    return EncoderStates(torch.zeros(n, 5, 8), index=index)


def test_each_side_of_a_guidance_batch_has_its_own_adapters(monkeypatch):
    """Four samples on two prompts beside ordinary negatives, and the other layouts: for each side as for both in one object."""
    s, plain = _set_on_host(monkeypatch), torch.zeros(4, 7, 8)
    cases = [  # uncond, cond, ids, context_ids, what the sides read (None: refused)
        (plain, _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], [0, 1], ([0, 0, 1, 1], [0, 1])),
        (plain, _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], [2, -1, 2, -1, 0, 1], ([2, -1, 2, -1], [0, 1])),
        (plain, _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], None, None),
        (plain, _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], [0, 1, 0], None),
        (_side(1), _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], [0, 1], None),                     # the shared negative's is not said
        (_side(1), _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], [-1, 0, 1], ([-1], [0, 1])),
        (_side(2, [0, 0, 1, 1]), _side(4), [0, 0, 1, 1], [2, 1], None),                     # not twice the list
        (_side(2, [0, 0, 1, 1]), _side(4), [0, 0, 1, 1], [2, 1, 0, 0, 1, 1], ([2, 1], [0, 0, 1, 1])),
        (_side(2, [0, 0, 1, 1]), _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], [0, 1], ([0, 1], [0, 1])),
        (_side(2, [0, 1, 0, 1]), _side(2, [0, 0, 1, 1]), [0, 0, 1, 1], [0, 1], None),       # as many, read by others
        (_side(3, [2, 0, 1]), torch.zeros(3, 5, 8), [0, 1, -1], [1, 2, 0], None),
        (torch.zeros(3, 5, 8), _side(3, [2, 0, 1]), [0, 1, -1], [1, -1, 0], ([0, 1, -1], [1, -1, 0])),
        (plain, plain, [0, 1, 2, -1], None, ([0, 1, 2, -1], [0, 1, 2, -1])),
        (plain, plain, [0, 1, 2, -1], [1, 1, 0, 2], ([1, 1, 0, 2], [1, 1, 0, 2])),
        (plain, plain, [0, 1], None, None),
        (_side(1), _side(1), [1], None, ([1], [1])),                                        # one sample: its contexts are its own
        (plain[:1], _side(3, [2]), [1], None, ([1], [1, 1, 1])),
        (_side(1), _side(1), [1, 0], None, None),
        (_side(1), _side(1), [1, 0], [2], ([2], [2])),
    ]
    for uncond, cond, ids, cids, want in cases:
        s.select(ids, cids)
        pair = GuidancePair(uncond, cond)
        both = EncoderStates.cat(EncoderStates.of(uncond), EncoderStates.of(cond), batch=len(ids))
        counts = pair.counts
        ask = [lambda: s.ids_for_contexts(counts[0], pair.shared[0], pair, 0), lambda: s.ids_for_contexts(counts[1], pair.shared[1], pair, 1),
               lambda: s.ids_for_contexts(sum(counts), both.shared, both.pair), lambda: s.ids_for_contexts(sum(counts), both.shared, both.clone().pair)]
        if want is None:
            refused = 0
            for f in ask:
                try:
                    f()
                except L.SdmiError:
                    refused += 1
            assert refused >= 3, (ids, cids)                                                # a side that the list names may have its ids
        else:
            assert [f().tolist() for f in ask] == [want[0], want[1], want[0] + want[1], want[0] + want[1]], (ids, cids)
    with pytest.raises(L.SdmiError, match="sides of this batch"):
        s.ids_for_contexts(3, False, pair, 0)


def test_ids_of_contexts_by_themselves(monkeypatch):
    s = _set_on_host(monkeypatch)
    s.select([0, 1], [1, 2])
    assert s.ids_for_contexts(2, True).tolist() == [1, 2] and s.ids_for_contexts(2, False).tolist() == [1, 2]
    assert s.ids_for_contexts(4, False).tolist() == [1, 2, 1, 2]                            # [uncond | cond], a context for each sample
    for n, shared in ((4, True), (3, True), (1, False)):
        with pytest.raises(L.SdmiError, match="contexts"):
            s.ids_for_contexts(n, shared)
    s.select([0, 1, 2, 0], [1, 2])
    with pytest.raises(L.SdmiError, match="contexts"):
        s.ids_for_contexts(4, False)                                                        # not a batch of twice the samples
    assert s.select([2]).ids_for_contexts(1, True).tolist() == [2] and s.ids_for_contexts(3, True).tolist() == [2, 2, 2]


def test_states_that_cat_made_keep_their_sides(monkeypatch):
    monkeypatch.setattr(E, "_need_cuda", lambda t, what: None)
    make = lambda a, b: EncoderStates.cat(a, b, batch=4)
    one, two = make(_side(2, [0, 0, 1, 1]), _side(4)), make(_side(2, [0, 1, 0, 1]), _side(4))
    one.copy_(two)
    assert one.pair is two.pair and one.index.tolist() == [0, 1, 0, 1, 2, 3, 4, 5]
    with pytest.raises(L.SdmiError, match="sides"):
        one.copy_(make(_side(4), _side(2, [0, 1, 0, 1])))
    loose = EncoderStates(torch.zeros(6, 5, 8), index=[0] * 8)
    assert loose.copy_(one).pair is one.pair                                                # as before, states of any origin


@pytest.fixture(scope="module")
def side_refs(net):
    """eps of every sample with its own merged weights: cond, uncond with the sample's adapter, uncond of one shared negative."""
    unet, sd = net
    rs = np.random.RandomState(21)
    x, tokens, t = _rand(rs, 4, 9, 16, 16), _rand(rs, 2, 60, 1024), torch.tensor([481] * 4)
    plain, one = _rand(rs, 4, 77, 1024), _rand(rs, 1, 40, 1024)
    ads, ids, index, lens = _unet_adapters(rs, sd, 0.3), [0, 0, 1, 1], [0, 0, 1, 1], [60, 33]
    eps = lambda i, ic, ctx: O.unet_forward(_merged(sd, ads, ids[i], ic), x[i:i + 1], t[i:i + 1], ctx)
    with torch.no_grad():
        cond = [eps(i, index[i], tokens[index[i]:index[i] + 1, :lens[index[i]]]) for i in range(4)]
        own = [eps(i, ids[i], plain[i:i + 1]) for i in range(4)]
        shared = [eps(i, 1, one) for i in range(4)]
    return dict(x=x, tokens=tokens, t=t, plain=plain, one=one, ads=ads, ids=ids, index=index, lens=lens, cond=cond, own=own, shared=shared)


@pytest.mark.gpu
@pytest.mark.parametrize("negatives", ["plain", "one"])
@pytest.mark.parametrize("dual", [True, False])
def test_sampler_gives_each_side_its_own_adapters(net, side_refs, dual, negatives):
    """Two prompts for four samples beside four plain negatives, or beside one for all of them (its adapter said first)."""
    from stable_diffusion_amd.sampler import Sampler
    unet, _ = net
    r = side_refs
    dev = lambda v: v.to(DEV)
    cond = EncoderStates(dev(r["tokens"]), r["lens"], r["index"])
    uncond, cids, refs = (dev(r["plain"]), [0, 1], r["own"]) if negatives == "plain" else (EncoderStates(dev(r["one"])), [1, 0, 1], r["shared"])
    try:
        unet.set_adapters(AdapterSet(unet, r["ads"]).select(r["ids"], cids))
        xc, t = dev(r["x"]).repeat(2, 1, 1, 1), dev(r["t"]).repeat(2)
        got = []
        for use_graph in (False, True):
            s = Sampler(unet, None, dual_stream=dual)
            eps = s._unet_step(xc, t, s.make_context(uncond, cond, 4), use_graph, same_halves=True).clone()
            for i in range(4):
                _gate(eps[i:i + 1], refs[i], 7e-3, 6e-3, "uncond, sample %d" % i)
                _gate(eps[4 + i:5 + i], r["cond"][i], 7e-3, 6e-3, "cond, sample %d" % i)
            got.append(eps)
        assert torch.equal(got[0], got[1])
        inp = make_inputs(4, 16, 2, seed=51)
        args = (2, cond, uncond, dev(inp["c_concat"]), dev(inp["x_T"]), [dev(n) for n in inp["noises"]], 7.5)
        s = Sampler(unet, None, dual_stream=dual)
        eager = s.sample(*args, decode=False)[0]
        for _ in range(2):
            assert torch.equal(s.sample(*args, decode=False, use_graph=True)[0], eager)
    finally:
        unet.set_adapters(None)


@pytest.mark.parametrize("dual", [True, False])
def test_sampler_refuses_states_of_another_number_of_samples(monkeypatch, dual):
    """One and three samples in the sides of a batch of two: as many in all, but not each sample's own."""
    from stable_diffusion_amd.sampler import Sampler
    monkeypatch.setattr(E, "_need_cuda", lambda t, what: None)

    class Net(object):
        def precompute_context(self, context, pair=None, side=None):
            return context
    s = Sampler(Net(), None, dual_stream=dual)
    for uncond, cond, what in ((_side(1, [0]), _side(2, [0, 1, 1]), "unconditional"), (_side(2), _side(3), "conditional")):
        with pytest.raises(L.SdmiError, match="the %s states are for" % what):
            s.make_context(uncond, cond, 2)
    s.make_context(_side(1), _side(2), 2)


def test_numbers_past_32_bits_are_not_taken_for_others(monkeypatch):
    """A length, a context or an adapter of 2^32 is past the end, not 0; a region past the 32nd is refused."""
    s, big = _set_on_host(monkeypatch), 1 << 32
    e = EncoderStates(torch.zeros(2, 5, 8), lens=[big, -big - 1], index=[big, 1])
    assert e.lens.tolist() == [2 ** 31 - 1, -2 ** 31] and e.index.tolist() == [2 ** 31 - 1, 1]
    assert EncoderStates.cat(e, e).index.tolist() == [-1, 1, -1, 3]
    assert s.select([big, big + 2, -big, 1]).ids_for(4).tolist() == [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 1]
    for v in ([0.0, 1.0], [0.7], torch.zeros(2, dtype=torch.bfloat16)):
        with pytest.raises(L.SdmiError, match="integer"):
            s.select(v)
        with pytest.raises(L.SdmiError, match="integer"):
            s.select([0, 1], v)
    sets = lambda k, q: EncoderStates(torch.zeros(1, 2, 8), key_regions=torch.tensor([k]), query_regions=torch.tensor([[[q]]]))
    assert sets([big - 1, -2 ** 31], -1).key_regions.tolist() == [[-1, -2 ** 31]]
    for k, q in (([big, 1], 1), ([1, 1], big), ([1, -2 ** 31 - 1], 1)):
        with pytest.raises(L.SdmiError, match="32 bits"):
            sets(k, q)


@pytest.mark.gpu
def test_a_step_behind_an_image_sees_the_adapters_of_now(net):
    """A captured step asked for by itself, after an image with other adapters."""
    from stable_diffusion_amd.sampler import Sampler
    unet, sd = net
    rs = np.random.RandomState(61)
    dev = lambda v: v.to(DEV)
    inp, first, second = make_inputs(2, 16, 2, seed=61), *(AdapterSet(unet, [a]).select([0, 0]) for a in _unet_adapters(rs, sd, 0.3))
    s = Sampler(unet, None)
    try:
        unet.set_adapters(first)
        s.sample(2, dev(inp["cond"]), dev(inp["uncond"]), dev(inp["c_concat"]), dev(inp["x_T"]), [dev(n) for n in inp["noises"]], 7.5, decode=False, use_graph=True)
        unet.set_adapters(second)
        cc = s.make_context(dev(inp["uncond"]), dev(inp["cond"]))
        want = s._unet_step(s._xc, s._emb_cur, cc, False, same_halves=True).clone()
        assert torch.equal(s._unet_step(s._xc, s._emb_cur, cc, True, same_halves=True), want)
    finally:
        unet.set_adapters(None)


def test_modules_saved_whole_before_there_were_adapters_load():
    """A module's attributes as torch.save(module) wrote them when layers had no adapters."""
    import io
    from Unet import Unet
    m = _layer()
    for mod in m.modules():
        mod.__dict__.pop("adapters", None)
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    back = torch.load(buf, weights_only=False)
    assert all(a._pack(kind) is None for a in (back.transformer_blocks[0].attn1, back.transformer_blocks[0].attn2) for kind in ("qkv", "q", "kv", "out"))
    with torch.device("meta"):
        unet = Unet()
    unet.__dict__.pop("adapters", None)
    assert unet.adapters is None


def test_ids_for_the_samples_of_both_sides(monkeypatch):
    """One id for each sample of [uncond | cond] (no adapter without the prompt, say): each side's contexts go by their own."""
    s = _set_on_host(monkeypatch).select([-1, -1, 0, 1])
    plain = torch.zeros(2, 7, 8)
    assert s.ids_for(4).tolist() == [-1, -1, 0, 1]
    for uncond, cond in ((plain, plain), (EncoderStates(plain), EncoderStates(plain))):
        pair = GuidancePair(uncond, cond)
        assert s.ids_for_contexts(4, False, pair).tolist() == [-1, -1, 0, 1]
        assert [s.ids_for_contexts(2, False, pair, side).tolist() for side in (0, 1)] == [[-1, -1], [0, 1]]
    # one sample: its one context of states that fit any batch is its own
    both = EncoderStates.cat(_side(1), _side(1), batch=1)
    for pair in (both.pair, GuidancePair(_side(1), _side(1), 1)):
        assert s.select([-1, 2]).ids_for_contexts(2, both.shared, pair).tolist() == [-1, 2] and s.select([2]).ids_for_contexts(2, both.shared, pair).tolist() == [2, 2]
    with pytest.raises(L.SdmiError, match="3 ids for 2 samples"):
        s.select([0, 1, 2]).ids_for_contexts(2, False, GuidancePair(plain, plain), 0)


@pytest.mark.parametrize("dual", [True, False])
def test_sampler_asks_a_model_without_adapters_as_before(dual):
    """A model of a caller's own whose precompute_context takes the context alone, and whose contexts are updated by it alone."""
    from stable_diffusion_amd.sampler import Sampler

    class Context(object):
        def __init__(self, v):
            self.seen = [v]

        def update(self, v):
            self.seen.append(v)

    class Net(object):
        def precompute_context(self, context):
            return Context(context)
    s, a, b = Sampler(Net(), None, dual_stream=dual), torch.zeros(2, 7, 8), torch.ones(2, 7, 8)
    for _ in range(2):
        cc = s.make_context(a, b)
    sides = [c.seen for c in cc] if dual else [cc.seen]
    assert [len(v) for v in sides] == [2] * len(sides) and torch.equal(torch.cat([v[1] for v in sides]), torch.cat([a, b]))


def test_unsigned_numbers_past_63_bits_are_past_the_end_too(monkeypatch):
    s = _set_on_host(monkeypatch)
    v = np.array([2 ** 64 - 1, 1], dtype=np.uint64)
    assert EncoderStates(torch.zeros(2, 5, 8), lens=v, index=v).lens.tolist() == [2 ** 31 - 1, 1] and s.select(v).ids_for(2).tolist() == [2 ** 31 - 1, 1]
    with pytest.raises(L.SdmiError, match="32 bits"):
        EncoderStates(torch.zeros(1, 2, 8), key_regions=v[None], query_regions=torch.ones(1, 1, 1, dtype=torch.int32))
