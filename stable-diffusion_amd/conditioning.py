"""What the requests of one batch bring along: encoder states of their own lengths (EncoderStates) and low-rank adapters
(AdapterSet), for Unet.forward / precompute_context / Sampler.sample.  The reference has one fixed form of the first (every
sample its own 77 tokens, layers/SpatialTransformer.py:70-95) and none of the second.

Everything that a captured UNet step reads of them (states, lengths, contexts, regions, adapter ids) lives in buffers that are
refilled in place, so a graph captured once serves the next batch of the same shape."""
import torch

from . import _lib as L
from . import engine as E


def _int32(v, dev, sets=False):
    """Integers as int32 on `dev`, a copy.  Numbers past 32 bits stay past every count that they are compared with; of sets the bits
    count, and a bit past the 32nd is refused."""
    if v.dtype in (torch.int64, torch.uint32, torch.uint64):
        past = v.dtype is torch.uint64              # its upper half comes out negative
        v = v.to(device=dev, dtype=torch.int64)
        v = v.where(v >= 0, 2 ** 63 - 1) if past else v
        if not sets:
            v = v.clamp(-2 ** 31, 2 ** 31 - 1)
        elif v.numel() and not (v.is_cuda and torch.cuda.is_current_stream_capturing()) and bool(((v < -2 ** 31) | (v >= 2 ** 32)).any()):
            raise L.SdmiError("EncoderStates: sets of regions are 32 bits")
    return v.to(device=dev, dtype=torch.int32, copy=True).contiguous()


def _words(v, shape, dev, what):
    """An integer tensor of this shape as its own contiguous int32 on `dev` (sets of 32 regions keep their bits)."""
    if v is None:
        return None
    v = torch.as_tensor(v)
    if v.is_floating_point() or v.is_complex() or tuple(v.shape) != tuple(shape):
        raise L.SdmiError("EncoderStates: %s has to be integers of shape %s, got %s %s" % (what, tuple(shape), v.dtype, tuple(v.shape)))
    return _int32(v, dev, what.endswith("regions"))


class EncoderStates(object):
    """tokens (contexts, T, C): the encoder's states, padded to T; lens (contexts,): how many of them exist; index (b,): the
    context each sample of the batch reads (default: its own, or the only one).  Regional prompts: key_regions (contexts, T) and
    query_regions (b, h, w) at the latent's resolution are sets of up to 32 regions as bits; a position sees the tokens whose
    set meets its own, and gets zeros from the attention where there is none.  Deeper levels take every second position.
    The values are copied: changing the arguments afterwards changes nothing here."""

    def __init__(self, tokens, lens=None, index=None, key_regions=None, query_regions=None):
        if tokens.dim() != 3:
            raise L.SdmiError("EncoderStates: tokens are (contexts, T, C), got %s" % (tuple(tokens.shape),))
        E._need_cuda(tokens, "EncoderStates")
        if (key_regions is None) != (query_regions is None):
            raise L.SdmiError("EncoderStates: key_regions and query_regions go together")
        n, t, _ = tokens.shape
        dev = tokens.device
        self.tokens = tokens.detach().to(dtype=torch.float32, copy=True).contiguous()
        self.lens = _words(lens, (n,), dev, "lens")
        b = None
        if index is not None:
            b = torch.as_tensor(index).numel()
        elif query_regions is not None:
            b = torch.as_tensor(query_regions).shape[0]
        elif n > 1:
            b = n
        if index is None and n != 1 and n != b:
            raise L.SdmiError("EncoderStates: %d contexts for %d samples need an index" % (n, b))
        self.batch = b                      # None: one context for a batch of any size
        self.pair = None                    # GuidancePair of the two sides that cat() put together
        self.index = _words(index, (b,), dev, "index")
        self.key_regions = _words(key_regions, (n, t), dev, "key_regions")
        self._levels = {}                   # (h, w) -> (b, h * w) sets of the positions of that level
        self.query_regions = None
        if query_regions is not None:
            query_regions = torch.as_tensor(query_regions)
            if query_regions.dim() != 3:
                raise L.SdmiError("EncoderStates: query_regions are (b, h, w), got %s" % (tuple(query_regions.shape),))
            self.query_regions = _words(query_regions, (b,) + tuple(query_regions.shape[1:]), dev, "query_regions")
            self._fill_levels()

    @staticmethod
    def of(x):
        return x if isinstance(x, EncoderStates) else EncoderStates(x)

    def _fill_levels(self):
        q = self.query_regions
        while q is not None:
            key = tuple(q.shape[1:])
            if key in self._levels:
                self._levels[key].copy_(q.reshape(q.shape[0], -1))
            else:
                self._levels[key] = q.reshape(q.shape[0], -1).contiguous()
            # Downsample keeps positions 0, 2, 4, ... (stride 2, layers/ResBlock.py:36-37)
            q = q[:, ::2, ::2] if max(key) > 1 else None

    def regions(self, h, w):
        """(b, h * w) sets of the positions of an h x w level."""
        if self.query_regions is None:
            return None
        if (h, w) not in self._levels:
            raise L.SdmiError("EncoderStates: query_regions of %s have no level of %d x %d" % (tuple(self.query_regions.shape[1:]), h, w))
        return self._levels[(h, w)]

    def signature(self):
        """States of one signature can take each other's place in the same buffers."""
        s = lambda v: None if v is None else tuple(v.shape)
        return (s(self.tokens), str(self.tokens.device), self.batch, s(self.lens), s(self.index), s(self.key_regions), s(self.query_regions))

    @property
    def shared(self):
        """Whether samples pick their contexts by an index, or all read one: the samples' adapters then do not say the contexts'."""
        return self.index is not None or self.batch != self.tokens.shape[0]

    def copy_(self, other):
        """Takes over another batch's values in place."""
        if other.signature() != self.signature():
            raise L.SdmiError("EncoderStates.copy_: %s cannot take %s" % (self.signature(), other.signature()))
        if self.pair is not None and other.pair is not None and (self.pair.counts, self.pair.shared) != (other.pair.counts, other.pair.shared):
            raise L.SdmiError("EncoderStates.copy_: sides of %s contexts cannot take sides of %s" % (self.pair.counts, other.pair.counts))
        for name in ("tokens", "lens", "index", "key_regions", "query_regions"):
            if getattr(self, name) is not None:
                getattr(self, name).copy_(getattr(other, name))
        self.pair = other.pair
        self._fill_levels()
        return self

    def clone(self):
        twin = EncoderStates(self.tokens, self.lens, self.index, self.key_regions, self.query_regions)
        twin.pair = self.pair
        return twin

    @staticmethod
    def cat(a, b, batch=None):
        """The batch [a | b] (as the CFG batch [uncond | cond]); batch: samples of a side that has one context for any number.
        The contexts of b follow those of a; beside a side with regions, one without is in all of them."""
        ba, bb = (s.batch if s.batch is not None else batch for s in (a, b))
        if ba is None or bb is None:
            raise L.SdmiError("EncoderStates.cat: one context for a batch of any size: say of which (batch)")
        dev, t = a.tokens.device, max(a.tokens.shape[1], b.tokens.shape[1])
        pad = lambda v: torch.nn.functional.pad(v, (0, 0, 0, t - v.shape[1]) if v.dim() == 3 else (0, t - v.shape[1]))
        full = lambda n, v: torch.full((n,), v, dtype=torch.int32, device=dev)
        lens = lambda s: s.lens if s.lens is not None else full(s.tokens.shape[0], s.tokens.shape[1])
        na, nb = a.tokens.shape[0], b.tokens.shape[0]
        lens_ab = index = kr = qr = None
        if a.lens is not None or b.lens is not None or a.tokens.shape[1] != b.tokens.shape[1]:
            lens_ab = torch.cat([lens(a), lens(b)])
        if a.index is not None or b.index is not None or (na, nb) != (ba, bb):
            own = lambda s, n, m: torch.arange(m, dtype=torch.int32, device=dev) if n == m else full(m, 0)
            ia = a.index if a.index is not None else own(a, na, ba)
            ib = b.index if b.index is not None else own(b, nb, bb)
            # an index outside its own side sees nothing, and not the other side's contexts
            index = torch.cat([torch.where(ia < na, ia, full(ba, -1)), torch.where((ib >= 0) & (ib < nb), ib + na, full(bb, -1))])
        with_regions = a if a.key_regions is not None else b
        if with_regions.key_regions is not None:
            hw = with_regions.query_regions.shape[1:]
            keys = lambda s: s.key_regions if s.key_regions is not None else full(s.tokens.shape[0], -1)[:, None].expand(-1, s.tokens.shape[1])
            queries = lambda s, m: s.query_regions if s.query_regions is not None else full(m, -1)[:, None, None].expand(-1, *hw)
            if a.query_regions is not None and b.query_regions is not None and a.query_regions.shape[1:] != b.query_regions.shape[1:]:
                raise L.SdmiError("EncoderStates.cat: query_regions of %s and %s" % (tuple(a.query_regions.shape), tuple(b.query_regions.shape)))
            kr, qr = torch.cat([pad(keys(a)), pad(keys(b))]), torch.cat([queries(a, ba), queries(b, bb)])
        both = EncoderStates(torch.cat([pad(a.tokens), pad(b.tokens)]), lens_ab, index, kr, qr)
        both.pair = GuidancePair(a, b, batch)
        return both


class GuidancePair(object):
    """The contexts of the two sides of a guidance batch [uncond | cond], EncoderStates or plain (b, T, C) tokens: how many, whether
    samples share them, and which sample reads which.  The same for one object that holds both sides and for an object of each.
    batch: samples of a side, for states that say nothing of it."""

    def __init__(self, uncond, cond, batch=None):
        sides = (uncond, cond)
        self.counts = tuple((s.tokens if isinstance(s, EncoderStates) else s).shape[0] for s in sides)
        self.shared = tuple(isinstance(s, EncoderStates) and s.shared and not (s.batch is None and batch == 1) for s in sides)
        self._index = tuple(s.index.clone() if shared and s.index is not None else None for s, shared in zip(sides, self.shared))

    def alike(self):
        """Whether every sample reads the same place among the contexts on both sides.  Waits for the GPU where both have an index."""
        (na, nb), (sa, sb), (ia, ib) = self.counts, self.shared, self._index
        if na != nb or sa != sb or (ia is None) != (ib is None):
            return False
        if ia is None:
            return True
        if ia.is_cuda and torch.cuda.is_current_stream_capturing():
            return False                    # not to be asked there
        return torch.equal(ia, ib)


class LayerAdapters(object):
    """One attention layer's share of an AdapterSet: an engine.LoraPack for each projection GEMM that has adapters."""

    def __init__(self, owner, packs):
        self.owner, self.packs = owner, packs

    def pack(self, kind):
        """kind: "qkv" (one GEMM of self-attention), "q", "kv" (of the context), "out"; None: nothing adapted there."""
        if kind == "qkv" and ("q" in self.packs or "kv" in self.packs) or kind in ("q", "kv") and "qkv" in self.packs:
            raise L.SdmiError("AdapterSet: the adapters were laid out for %s-attention, this call is the other kind" % ("self" if "qkv" in self.packs else "cross"))
        return self.packs.get(kind)


class AdapterSet(object):
    """Low-rank adapters for the attention projections of a model, and the one that each sample of the batch uses.

    adapters: a list; each a dict {layer name: (down (r, k), up (n, r)[, scale])}, the layer adding scale * up @ down to its
    weight (scale: default 1; alpha / r in the usual files).  Layer names are `model.named_modules()`'s, of the projections
    to_q / to_k / to_v / to_out.0 of attn1 and attn2; ranks may differ (smaller ones are padded with zeros).

    attach() puts the set into the model's layers, detach() takes it out; select(ids[, context_ids]) chooses for the next
    batch: an adapter for each sample, anything outside [0, len(adapters)) for none, and one for each context where the set
    reaches attn2's to_k / to_v (default: the samples' ids, where every sample has a context of its own)."""

    PARTS = ("to_q", "to_k", "to_v", "to_out.0")

    def __init__(self, model, adapters):
        if not adapters:
            raise L.SdmiError("AdapterSet: no adapters")
        mods = {n: m for n, m in model.named_modules() if hasattr(m, "to_q") and hasattr(m, "to_out")}
        self.size = len(adapters)
        found = {}                          # layer -> {(adapter, part): (down, up, scale)}
        for i, ad in enumerate(adapters):
            for name, v in ad.items():
                owner, part = next(((name[:-len(p) - 1], p) for p in self.PARTS if name.endswith("." + p)), (None, None))
                if owner not in mods:
                    raise L.SdmiError("AdapterSet: %r is not an attention projection of this model (%s)" % (name, " / ".join(self.PARTS)))
                w, (down, up) = self._linear(mods[owner], part).weight, v[:2]
                if down.dim() != 2 or up.dim() != 2 or up.shape[1] != down.shape[0] or (up.shape[0], down.shape[1]) != tuple(w.shape) or not 1 <= down.shape[0] <= 256:
                    raise L.SdmiError("AdapterSet: %r of adapter %d: down %s, up %s do not fit a weight of %s (rank 1 .. 256)" %
                                      (name, i, tuple(down.shape), tuple(up.shape), tuple(w.shape)))
                found.setdefault(owner, {})[(i, part)] = (down, up, float(v[2]) if len(v) > 2 else 1.0)
        if not found:
            raise L.SdmiError("AdapterSet: the adapters change nothing")
        self.layers = []                    # (module, LayerAdapters)
        for owner, parts in found.items():
            # attn1 projects its tokens by one q|k|v GEMM; attn2's q comes from the tokens, its k|v from the context
            sets = {"qkv": ("to_q", "to_k", "to_v")} if owner.rsplit(".", 1)[-1] == "attn1" else {"q": ("to_q",), "kv": ("to_k", "to_v")}
            sets["out"] = ("to_out.0",)
            packs = {kind: self._pack(mods[owner], ps, parts) for kind, ps in sets.items() if any(p in ps for _, p in parts)}
            self.layers.append((mods[owner], LayerAdapters(self, packs)))
        self.device = next(iter(self.layers[0][1].packs.values())).a.device
        self.ids = self.context_ids = None
        self._buffers = {}                  # (what, length) -> (ids, twice the ids): a captured step's stay where they are

    @staticmethod
    def _linear(m, part):
        return m.to_out[0] if part == "to_out.0" else getattr(m, part)

    def _pack(self, m, parts, found):
        w = self._linear(m, parts[0]).weight
        E._need_cuda(w, "AdapterSet")
        (n, k), h = w.shape, E.act_dtype()
        rank = (max(v[0].shape[0] for (_, p), v in found.items() if p in parts) + 7) // 8 * 8
        a = torch.zeros((self.size, len(parts) * rank, k), dtype=h, device=w.device)
        b = torch.zeros((self.size, len(parts) * n, rank), dtype=h, device=w.device)
        for (i, p), (down, up, scale) in found.items():
            if p in parts:
                g, r = parts.index(p), down.shape[0]
                # the scale goes into `up`, to_q's with the factor that its packed weight carries (softmax in base 2), before the
                # rounding to 16 bits; beyond the range it saturates as the packed weights do
                up = up.to(w.device).float() * (scale * (E.Q_LOG2_SCALE if p == "to_q" else 1.0))
                for dst, src in ((a[i, g * rank:g * rank + r], down.to(w.device).float()), (b[i, g * n:(g + 1) * n, :r], up)):
                    if not bool(torch.isfinite(src).all()):
                        raise L.SdmiError("AdapterSet: adapter %d has infinities or NaN in %s" % (i, p))
                    dst.copy_(src.clamp(-torch.finfo(h).max, torch.finfo(h).max))
        return E.LoraPack(a, b, torch.ones((self.size,), dtype=torch.float32, device=w.device))

    def attach(self):
        for m, la in self.layers:
            m.adapters = la
        return self

    def detach(self):
        for m, la in self.layers:
            if m.adapters is la:
                m.adapters = None
        return self

    def _keep(self, what, v):
        v = torch.as_tensor(v).reshape(-1)
        if v.numel() == 0 or v.is_floating_point() or v.is_complex():
            raise L.SdmiError("AdapterSet.select: %d ids of %s: at least one integer" % (v.numel(), v.dtype))
        v = _int32(v, self.device)
        buf = self._buffers.get((what, v.numel()))
        if buf is None:
            buf = self._buffers[(what, v.numel())] = torch.empty((2 * v.numel(),), dtype=torch.int32, device=self.device)
        buf[:v.numel()].copy_(v)
        buf[v.numel():].copy_(v)
        return buf

    def select(self, ids, context_ids=None):
        """The adapters of the next batch, written where a step captured for a batch of this size reads them: ids, one for each
        sample; context_ids, one for each context of the states that come with it.  Of the two sides that a sampler takes
        [uncond | cond], context_ids are the conditional one's, or the unconditional one's followed by the conditional one's.  A
        side (or states) that they leave out goes by the samples' ids where every sample has a context of its own, and by the same
        context_ids where both sides are laid out alike; anything else is refused.  A ContextKV made before has to be made or
        updated again, as Sampler.sample does."""
        self.ids = self._keep("ids", ids)
        self.context_ids = None if context_ids is None else self._keep("contexts", context_ids)
        return self

    @staticmethod
    def _take(buf, n, what):
        if 2 * n != buf.numel() and n != buf.numel():
            raise L.SdmiError("AdapterSet: %d ids for %d %s" % (buf.numel() // 2, n, what))
        return buf[:n]

    def ids_for(self, n):
        """The ids of a batch of n samples: the selected ones, or twice them for a CFG batch [uncond | cond]."""
        if self.ids is None:
            raise L.SdmiError("AdapterSet: select(ids) first")
        return self._take(self.ids, n, "samples")

    def _one_id(self, n):
        """One id was selected for all samples: it is any context's as well."""
        return self.ids[:1].expand(n).contiguous() if self.ids is not None and self.ids.numel() == 2 else None

    def ids_for_contexts(self, n, shared, pair=None, side=None):
        """The ids of n contexts; shared: samples pick theirs by an index (or all read one), so the samples' ids do not say.
        pair: the GuidancePair that the contexts belong to; side: 0 uncond, 1 cond, None both in a row."""
        if pair is not None:
            return self._ids_for_pair(n, pair, side)
        if self.context_ids is None:
            if not shared:
                return self.ids_for(n)
            one = self._one_id(n)
            if one is None:
                raise L.SdmiError("AdapterSet: samples share contexts, whose to_k / to_v have adapters: say which (select(ids, context_ids))")
            return one
        have = self.context_ids.numel() // 2
        # contexts of the samples' own, twice as many as ids of either kind: a batch [uncond | cond]
        if n == have or (not shared and n == 2 * have and self.ids is not None and self.ids.numel() == n):
            return self.context_ids[:n]
        raise L.SdmiError("AdapterSet: %d ids for %d contexts" % (have, n))

    def _ids_for_pair(self, n, pair, side):
        given, have = self.context_ids, 0 if self.context_ids is None else self.context_ids.numel() // 2
        na, nb = pair.counts
        if n != (na + nb if side is None else pair.counts[side]):
            raise L.SdmiError("AdapterSet: %d contexts, where the sides of this batch have %d and %d" % (n, na, nb))
        if given is not None and have not in (nb, na + nb):
            raise L.SdmiError("AdapterSet: %d context_ids for %d unconditional and %d conditional contexts: give the conditional ones', or all of them" % (have, na, nb))

        def of(s):
            m = pair.counts[s]
            if have == na + nb:
                return given[:na] if s == 0 else given[na:have]
            if given is not None and (s == 1 or pair.alike()):
                return given[:m]
            if not pair.shared[s]:
                if self.ids is None:
                    raise L.SdmiError("AdapterSet: select(ids) first")
                # an id for each sample of a side, or of the whole batch [uncond | cond]
                if self.ids.numel() not in (2 * m, 4 * m):
                    raise L.SdmiError("AdapterSet: %d ids for %d samples" % (self.ids.numel() // 2, m))
                return self.ids[s * m:(s + 1) * m]
            one = self._one_id(m)
            if one is None:
                raise L.SdmiError("AdapterSet: samples share the %s contexts, whose to_k / to_v have adapters: say which (select(ids, context_ids), the "
                                  "unconditional ones' first)" % ("unconditional", "conditional")[s])
            return one
        return torch.cat([of(0), of(1)]) if side is None else of(side)
