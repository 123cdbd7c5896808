"""LlamaMXDecoder on paged caches: against the quantised model's own forward, with a shared prefix, drawing tokens."""
import pytest
import torch

from test_llama_decode_gpu import tiny_llama
from test_serving_gpu import F32, attend64, half_step, rotate64, within

pytestmark = pytest.mark.gpu


def decoder(kv_heads, seed=0, **kw):
    from mxfp4 import quantize_model_mxfp4
    from mxfp4.llama import LlamaMXDecoder
    model = tiny_llama(seed=seed, kv_heads=kv_heads)
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 1:
                p.mul_(torch.rand_like(p.float()).to(p.dtype) + 0.5)
    quantize_model_mxfp4(model, verbose=False)
    return model, LlamaMXDecoder(model, **kw)


def ids_of(batch, tokens, seed=1):
    return torch.randint(0, 160, (batch, tokens), generator=torch.Generator().manual_seed(seed)).cuda()


def done(dec):
    from mxfp4 import gemm, serving
    gemm.check_status()
    dec.chain.check_status()
    serving.check_status()


class Checked:
    """Every attention call of a decoder against 64 bits, from the projection's output that went in and where its tokens belong.

    (Logits are not compared: between the layers activations are quantised to four bits, and there a last-place difference of an
    attention output moves a code by a whole step, an eighth of the value and more.  A call's own inputs and outputs have the bounds of
    test_serving_gpu.py.)"""

    def __init__(self, dec, model):
        self.dec, self.inner, self.calls = dec, dec._attend_paged, 0
        self.freq = model.model.rotary_emb.inv_freq.double()
        dec._attend_paged = self

    def expect(self, batch0, batch, tokens, have, prefix, is_prefix=False):
        self.at = dict(batch0=batch0, batch=batch, tokens=tokens, have=have, prefix=prefix, is_prefix=is_prefix)

    def __call__(self, li, qkv, plan):
        d, e = self.dec, self.at
        before = qkv.clone()
        out = self.inner(li, qkv, plan)
        M, D, nq = len(qkv), d.head_dim, d.h_l * d.head_dim
        B, T = e["batch"], e["tokens"]
        assert M == B * T
        split = lambda x: (x[:, :nq].view(M, d.h_l, D), x[:, nq:nq + d.kv_l * D].view(M, d.kv_l, D), x[:, nq + d.kv_l * D:].view(M, d.kv_l, D))  # noqa: E731
        place = torch.arange(T, device="cuda").repeat(B) + e["have"]
        position = place + (0 if e["is_prefix"] else e["prefix"])
        u = half_step(torch.bfloat16)
        q0, k0, v0 = split(before)
        q1 = split(qkv)[0]
        want, size = rotate64(q0, position, self.freq, False, 1.0)
        ok, by = within(q1, want, u * want.abs() * (1 + 1e-3) + 8 * F32 * size)
        assert ok, by
        cache, ps = d.pages[li], d.page_size
        table = d.prefix_pages[None] if e["is_prefix"] else d.table[e["batch0"]:e["batch0"] + B]
        row = torch.arange(B, device="cuda").repeat_interleave(T)
        page = table[row, place // ps].long()
        want, size = rotate64(k0, position, self.freq, False, 1.0)
        ok, by = within(cache.k[page, :, place % ps], want, u * want.abs() * (1 + 1e-3) + 8 * F32 * size)
        assert ok, by
        assert torch.equal(cache.v[page, :, place % ps], v0)
        lens, starts = [e["have"] + T] * B, [i * T for i in range(B + 1)]
        want, _, tol, _ = attend64(q1, cache.k, cache.v, table, lens, starts, d.prefix_pages, 0 if e["is_prefix"] else e["prefix"], D ** -0.5)
        ok, by = within(out.view(M, d.h_l, D), want, tol)
        assert ok, by
        self.calls += 1
        return out


def run_checked(check, dec, ids, new, prefix):
    """prefill in two chunks and steps, without a graph; the tokens"""
    B, T = ids.shape
    toks = []
    for b0 in range(0, B, B // 2 + 1):
        n = min(B // 2 + 1, B - b0)
        check.expect(b0, n, T, 0, prefix)
        toks.append(dec._forward(ids[b0:b0 + n], T, batch0=b0).float().argmax(-1))
    nxt, out = torch.cat(toks), []
    dec.lens.zero_()
    dec.lens[:B].fill_(T)
    for j in range(new):
        out.append(nxt)
        check.expect(0, B, 1, T + j, prefix)
        nxt = dec._forward(nxt[:, None], 1).float().argmax(-1)
        dec.lens[:B].add_(1)
    return torch.stack(out, 1)


@pytest.mark.parametrize("kv_heads", [4, 2])
@pytest.mark.parametrize("P", [0, 1, 16, 21])
def test_paged_decoder(kv_heads, P):
    B, T, new = 6, 19, 5
    model, dec = decoder(kv_heads, max_batch=B + 2, max_len=T + new, page_size=16, max_prefix=32 if P else 0)
    ids, prefix = ids_of(B, T), ids_of(1, max(P, 1), seed=3)[0][:P]
    with torch.no_grad():
        check = Checked(dec, model)
        if P:
            check.expect(0, 1, P, 0, P, is_prefix=True)
            dec.set_prefix(prefix)
        tokens = run_checked(check, dec, ids, new, P)
        assert check.calls == 2 * ((1 if P else 0) + 2 + new)
        dec._attend_paged = check.inner
        first = dec.prefill(ids, chunk=B // 2 + 1)
        assert torch.equal(first, tokens[:, 0])
        assert torch.equal(dec.decode(new, use_graph=False), tokens)
        dec.prefill(ids, chunk=B // 2 + 1)
        assert torch.equal(dec.decode(new), tokens)              # the captured step, twice
        dec.prefill(ids, chunk=B // 2 + 1)
        assert torch.equal(dec.decode(new), tokens)
        with pytest.raises(ValueError, match="room"):
            dec.prefill(ids)
            dec.decode(new + 2)
        if P:
            with pytest.raises(ValueError, match="prefix"):
                dec.set_prefix(ids_of(1, 33)[0])
            dec.set_prefix(prefix[:0])                           # and none again
            run_checked(check_again(check), dec, ids, 1, 0)
    done(dec)


def check_again(check):
    check.dec._attend_paged = check
    return check


@pytest.mark.parametrize("page_size", [None, 16])
def test_drawn_tokens(page_size):
    B, T, new = 4, 6, 6
    _, dec = decoder(2, max_batch=B + 1, max_len=T + new, page_size=page_size)
    ids = ids_of(B, T)
    u0, u = torch.rand(B, generator=torch.Generator().manual_seed(5)), torch.rand(B, new - 1, generator=torch.Generator().manual_seed(6))
    greedy = [dec.prefill(ids), dec.decode(new)][1]
    for kw in (dict(temperature=0.0), dict(temperature=1.3, top_k=1), dict(top_p=0.0)):
        dec.set_sampling(**kw)
        dec.prefill(ids, uniforms=u0)
        assert torch.equal(dec.decode(new, uniforms=u), greedy)
    dec.set_sampling(temperature=torch.tensor([0.0, 0.8, 1.0, 1.5]), top_k=torch.tensor([0, 50, 0, 20]), top_p=0.95)
    dec.prefill(ids, uniforms=u0)
    graphed = dec.decode(new, uniforms=u)
    dec.prefill(ids, uniforms=u0)
    assert torch.equal(graphed, dec.decode(new, use_graph=False, uniforms=u))
    assert torch.equal(graphed[0], greedy[0]) and not torch.equal(graphed, greedy)
    with pytest.raises(ValueError, match="uniforms"):
        dec.prefill(ids)
    dec.set_sampling(temperature=None)
    dec.prefill(ids)
    assert torch.equal(dec.decode(new), greedy)
    done(dec)


def test_refusals():
    with pytest.raises(ValueError):
        decoder(2, max_batch=1, max_len=8, page_size=24)
    with pytest.raises(ValueError):
        decoder(2, max_batch=1, max_len=8, max_prefix=4)
    _, dec = decoder(2, max_batch=1, max_len=8)
    with pytest.raises(ValueError):
        dec.set_prefix(ids_of(1, 2)[0])
