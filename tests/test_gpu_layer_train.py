"""GPU: the transformer-layer operators together, as a training step runs them: a decoder layer and the track-query update, forward and every gradient, against
the oracle's formulas in 64 bits through autograd."""
import pytest
import torch

from mo_yolo_amd import modules as M
from mo_yolo_amd import ops
from oracle import track_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def double_of(module, prefix):
    """The module's parameters as 64-bit leaves on the CPU under `prefix`.name, and by name."""
    by = {n: p.detach().cpu().double().requires_grad_(True) for n, p in module.named_parameters()}
    return {f"{prefix}.{n}": t for n, t in by.items()}, by


def fill(module, seed):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in module.named_parameters():
            p.copy_(torch.randn(p.shape, generator=g) * (p.shape[-1] ** -0.5 if p.dim() == 2 else 0.1) + (1.0 if n.endswith("norm1.weight") or "norm" in n and n.endswith("weight") else 0.0))
    return module


def off(got, want):
    return float((got.detach().cpu().double() - want.detach()).norm() / want.detach().norm().clamp_min(1e-30))


def decoder_case(seed, bs=2, Lq=70):
    g = torch.Generator().manual_seed(seed)
    shapes = [(9, 13), (5, 7), (3, 4)]
    S = sum(h * w for h, w in shapes)
    embed, pos, feats = torch.randn(bs, Lq, 256, generator=g), torch.randn(bs, Lq, 256, generator=g), torch.randn(bs, S, 256, generator=g)
    box = torch.rand(bs, Lq, 4, generator=g) * 0.6 + 0.2
    return shapes, embed, pos, feats, box, torch.randn(bs, Lq, 256, generator=g)


def oracle_layer(shapes, embed, box, feats, pos, sd, mask=None, pad=None, table=None, lut=None):
    """decoder_layer of the oracle with training's masks and the position bias (track_oracle.decoder_layer without them)."""
    nh, C = 8, 256
    qk = embed + pos
    W, b = sd["l.self_attn.in_proj_weight"], sd["l.self_attn.in_proj_bias"]
    heads = lambda t: t.view(*t.shape[:2], nh, C // nh).transpose(1, 2)  # noqa: E731
    q, k, v = heads(qk @ W[:C].t() + b[:C]), heads(qk @ W[C:2 * C].t() + b[C:2 * C]), heads(embed @ W[2 * C:].t() + b[2 * C:])
    s = q @ k.transpose(-1, -2) / (C // nh) ** 0.5
    if table is not None:
        i = torch.arange(embed.shape[1])
        far = lut.shape[0] // 2
        s = s + table[lut.long()[(i[None] - i[:, None]).clamp(-far, far) + far]].permute(2, 0, 1)
    if mask is not None:
        s = s.masked_fill(mask, float("-inf"))
    o = (torch.softmax(s, -1) @ v).transpose(1, 2).flatten(2)
    e1 = O.layer_norm(embed + O.linear(o, sd, "l.self_attn.out_proj"), sd, "l.norm1")
    value = O.linear(feats, sd, "l.cross_attn.value_proj")
    if pad is not None:
        value = value.masked_fill(pad[..., None], 0.0)
    ca, _ = O.msda(e1 + pos, box, feats, shapes, sd, "l.cross_attn", nh, 4, value=value)
    e2 = O.layer_norm(e1 + ca, sd, "l.norm2")
    return O.layer_norm(e2 + O.linear(torch.relu(O.linear(e2, sd, "l.linear1")), sd, "l.linear2"), sd, "l.norm3")


@pytest.mark.parametrize("dtype,masked,tol,gtol", [(torch.float32, False, 3e-5, 3e-5), (torch.float32, True, 3e-5, 3e-5), (torch.bfloat16, True, 4e-2, 8.5e-2),
                                                   (torch.float16, False, 6e-3, 3e-2)])
def test_decoder_layer_trains(dtype, masked, tol, gtol):
    """Relative 2-norm errors: fp32, some 30 operations deep, 2^-24 each with the norms' amplification; 16 bits, about ten roundings of 2^-9 (2^-12) rms on the way
    to an output and ten more back to an input, and the sampling grid's sensitivity (levels up to 13 cells: an offset's rounding moves a sample by 13 times it).
    A gradient passes two steps besides.  The ReLU's: its arguments z, of unit size and normal, carry the rounding of ten operations in bf16 (about
    sqrt(10) 2^-9 0.8 = 5e-3 of them), so the sign of p = 5e-3 / pi = 1.6e-3 of them is the other one; half of the units are alive, so the gradient behind it is off by
    sqrt(2 p) = 5.6e-2 of its norm, and by 1.5 times that, 8.5e-2, at most (fp16: 5e-3 / 8, p = 2e-4, 2e-2 and 3e-2).  The sampling's: the gradient of a place jumps at a cell's edge, and 5e-3 of some 1.2 cells
    moves 0.5 % of the places over one in either axis, off by sqrt(2 * 0.005) = 0.1 (sampling_offsets, within its factor below)."""
    layer = fill(M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4), 1).to(DEV)
    rel = M.RelativePositionBias(16, 40, 8).to(DEV) if masked else None
    if masked:
        fill(rel, 2)
    shapes, embed, pos, feats, box, dy = decoder_case(3)
    rnd = lambda t: t.to(dtype).double()  # noqa: E731  (the same inputs on both sides)
    mask = pad = None
    if masked:
        group = torch.arange(70) // 20
        mask = (group[:, None] != group[None]) & (group[None] != 3)            # three denoising groups, who see themselves and the rest
        pad = torch.zeros(2, feats.shape[1], dtype=torch.bool)
        pad[0, 100:110] = True
    dev = [t.to(DEV, dtype).requires_grad_(True) for t in (embed, pos, feats)]
    out = layer.forward_train(dev[0], box.to(DEV), dev[2], shapes, padding_mask=None if pad is None else pad.to(DEV), attn_mask=None if mask is None else mask.to(DEV),
                              track_query_pos=dev[1], rel_bias=rel)
    out.backward(dy.to(DEV, dtype))
    sd, by = double_of(layer, "l")
    ref = [rnd(t).requires_grad_(True) for t in (embed, pos, feats)]
    table = None if rel is None else rel.weight.detach().cpu().double().requires_grad_(True)
    want = oracle_layer(shapes, ref[0], box.double(), ref[2], ref[1], sd, mask, pad, table, None if rel is None else rel.lut.cpu())
    want.backward(rnd(dy))
    assert off(out, want) < tol
    for name, a, b in zip(("embed", "pos", "feats"), dev, ref):
        assert a.grad.dtype == dtype and off(a.grad, b.grad) < gtol, name
    for n, p in layer.named_parameters():
        # the sampling offsets' gradient is a difference of neighbouring samples: its terms are some ten times its sums
        assert p.grad is not None and off(p.grad, by[n].grad) < gtol * (10 if "sampling_offsets" in n or "attention_weights" in n else 2), n
    if rel is not None:
        assert off(rel.weight.grad, table.grad) < gtol * 2


@pytest.mark.parametrize("held,dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.float16)])
def test_decoder_layer_with_16_bit_parameters(held, dtype):
    """Parameters in 16 bits, activations in the same type or another: output as above, gradients in the parameters' type."""
    layer = fill(M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4), 13).to(DEV, held)
    shapes, embed, pos, feats, box, dy = decoder_case(14)
    rnd = lambda t: t.to(dtype).double()  # noqa: E731
    out = layer.forward_train(embed.to(DEV, dtype), box.to(DEV), feats.to(DEV, dtype), shapes, track_query_pos=pos.to(DEV, dtype))
    out.backward(dy.to(DEV, dtype))
    sd, _ = double_of(layer, "l")
    want = oracle_layer(shapes, rnd(embed), box.double(), rnd(feats), rnd(pos), sd)
    assert out.dtype == dtype and off(out, want) < 4e-2
    for n, p in layer.named_parameters():
        assert p.grad is not None and p.grad.dtype == held and torch.isfinite(p.grad).all(), n


def test_forward_train_agrees_with_forward_and_forward_sees_updates():
    layer = fill(M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4), 5).to(DEV)
    shapes, embed, pos, feats, box, dy = (t if isinstance(t, list) else t.to(DEV) for t in decoder_case(6))
    opt = torch.optim.SGD(layer.parameters(), lr=1e-2)
    for _ in range(2):
        with torch.no_grad():
            a = layer(embed, box, feats, shapes, track_query_pos=pos)
        b = layer.forward_train(embed, box, feats, shapes, track_query_pos=pos)
        assert float((a - b.detach()).abs().max()) < 1e-4                             # two orders of the same fp32 sums, outputs of unit size
        opt.zero_grad()
        b.backward(dy)
        opt.step()                                                             # the inference form's prepared weights are of the old values now


def test_track_query_update_trains():
    qim = fill(M.QueryInteractionModule(None, 256, 256), 7).to(DEV)
    g = torch.Generator().manual_seed(8)
    n = 37
    emb, qp, ref, dy = torch.randn(n, 256, generator=g), torch.randn(n, 256, generator=g), torch.randn(n, 4, generator=g), torch.randn(n, 256, generator=g)
    e, q = emb.to(DEV).requires_grad_(True), qp.to(DEV).requires_grad_(True)
    out = qim.update_train(e, ref.to(DEV), q)
    out.backward(dy.to(DEV))
    sd, by = double_of(qim, "t")
    e2, q2 = emb.double().requires_grad_(True), qp.double().requires_grad_(True)
    pos = O.pos2posemb(ref).double()
    qk = (e2 + pos)[None]
    tgt = O.layer_norm(e2 + O.mha(qk, qk, e2[None], sd, "t.self_attn", 8)[0], sd, "t.norm1")
    tgt = O.layer_norm(tgt + O.linear(torch.relu(O.linear(tgt, sd, "t.linear1")), sd, "t.linear2"), sd, "t.norm2")
    want = O.layer_norm(q2 + O.linear(torch.relu(O.linear(tgt, sd, "t.linear_feat1")), sd, "t.linear_feat2"), sd, "t.norm_feat")
    want.backward(dy.double())
    assert off(out, want) < 3e-5 and off(e.grad, e2.grad) < 3e-5 and off(q.grad, q2.grad) < 3e-5
    for name, p in qim.named_parameters():
        assert off(p.grad, by[name].grad) < 6e-5, name
    empty = qim.update_train(e[:0], ref[:0].to(DEV), q[:0])
    assert empty.shape == (0, 256)


def test_cached_generation_agrees_with_the_whole_sequence():
    """One token at a time over a growing cache (keys and values written in place, lengths on the device) against the causal pass over the whole sequence."""
    g = torch.Generator(device=DEV).manual_seed(9)
    B, N, H, Hk, D = 2, 48, 8, 2, 64
    rel = M.RelativePositionBias(16, 20, H, bidirectional=False).to(DEV)
    with torch.no_grad():
        rel.weight.copy_(torch.randn(16, H, device=DEV, generator=g))
        q, k, v = (torch.randn(B, N, h, D, device=DEV, generator=g) for h in (H, Hk, Hk))
        whole = rel(q, k, v, causal=True, q_start=0)
        cache_k, cache_v = torch.full((B, 64, Hk, D), float("nan"), device=DEV), torch.full((B, 64, Hk, D), float("nan"), device=DEV)
        length = torch.zeros(B, dtype=torch.int32, device=DEV)
        for i in range(N):
            cache_k[:, i], cache_v[:, i] = k[:, i], v[:, i]
            length += 1
            one = rel(q[:, i:i + 1], cache_k, cache_v, k_len=length)
            assert float((one[:, 0] - whole[:, i]).abs().max()) < 1e-5, i      # sums of at most 48 terms of unit size in another order


def test_captured_training_step():
    """Forward, backward and an SGD step of the layer in one graph, replayed with new inputs and eager work between, against the same steps run eagerly."""
    def steps(captured):
        layer = fill(M.MOTRDecoderLayer(256, 8, 512, 0.0, None, 3, 4), 11).to(DEV)
        rel = fill(M.RelativePositionBias(16, 40, 8), 12).to(DEV)
        params = [*layer.parameters(), *rel.parameters()]
        sizes, *first = decoder_case(20)
        shapes = torch.tensor(sizes, dtype=torch.int64, device=DEV)
        held = [t.to(DEV) for t in first]
        outs = []

        def step():
            embed, pos, feats, box, dy = held
            out = layer.forward_train(embed, box, feats, shapes, track_query_pos=pos, rel_bias=rel)
            grads = torch.autograd.grad(out, params, dy)
            with torch.no_grad():
                for p, g in zip(params, grads):
                    p.sub_(g, alpha=1e-3)
            return out.detach()

        if captured:
            kept = [p.detach().clone() for p in params]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    out = step()
            torch.cuda.synchronize()
            with torch.no_grad():
                for p, k in zip(params, kept):
                    p.copy_(k)
        for i in range(4):
            for h, t in zip(held, decoder_case(20 + i)[1:]):
                h.copy_(t)
            if captured:
                graph.replay()
                outs.append(out.clone())
            else:
                outs.append(step())
            torch.cuda.synchronize()
        return outs, params

    a, pa = steps(False)
    b, pb = steps(True)
    for x, y in zip(a, b):
        assert off(x, y.cpu().double()) < 1e-5                                 # the sampling's gradient of the values is summed in any order
    for x, y in zip(pa, pb):
        assert float((x.detach() - y.detach()).abs().max()) < 1e-5
