"""A TinyViT block with rotary positions, the gated feed-forward block and residual dropout -- the operators together, in the network's own layers -- against the
same block in 64 bits (plain torch, CPU), and the whole network with these options."""
import copy

import pytest
import torch

import token_ops_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tv():
    from semiuhpe_amd.src import tiny_vit
    return tiny_vit


def block64(blk, x, held, keep, dim, heads, ws):
    """the block in 64 bits: parameters of the HIP block as leaves, `held` = the two dropout masks (values 0 / 1)"""
    P = {k: v.detach().cpu().double().requires_grad_(True) for k, v in blk.named_parameters()}
    B, H, W, C = x.shape
    dh = dim // heads
    ln = lambda v, n: torch.nn.functional.layer_norm(v, (C,), P[n + ".weight"], P[n + ".bias"], 1e-5)  # noqa: E731
    q = ln(x, "attn.norm").reshape(-1, C) @ P["attn.qkv.weight"].t() + P["attn.qkv.bias"]
    pos = torch.cartesian_prod(torch.arange(H), torch.arange(W)).repeat(B, 1).double()
    half = dh // 2
    freq = torch.cat([10000.0 ** (-2.0 * torch.arange(half // 2).double() / half)] * 2)
    ang = torch.cat([pos[:, :1].expand(-1, half // 2), pos[:, 1:].expand(-1, half // 2)], 1) * freq
    c, s = torch.cos(ang)[:, None, None], torch.sin(ang)[:, None, None]
    q = q.view(-1, heads, 3, dh)
    a, b = q[:, :, :2, :half], q[:, :, :2, half:]
    q = torch.cat([torch.cat([a * c - b * s, a * s + b * c], 3), q[:, :, 2:]], 2)
    win = q.view(B, H // ws, ws, W // ws, ws, heads, 3, dh).permute(0, 1, 3, 5, 6, 2, 4, 7).reshape(-1, heads, 3, ws * ws, dh)
    bias = P["attn.attention_biases"][:, blk.attn.attention_bias_idxs.cpu()]
    att = torch.softmax(win[:, :, 0] @ win[:, :, 1].transpose(-1, -2) * dh ** -0.5 + bias, -1) @ win[:, :, 2]
    att = att.reshape(B, H // ws, W // ws, heads, ws, ws, dh).permute(0, 1, 4, 2, 5, 3, 6).reshape(-1, C)
    o = att @ P["attn.proj.weight"].t() + P["attn.proj.bias"]
    x1 = x + (o * held[0] / keep).view_as(x)
    z = torch.nn.functional.conv2d(x1.permute(0, 3, 1, 2), P["local_conv.c.weight"], padding=1, groups=C)
    z = torch.nn.functional.batch_norm(z, None, None, P["local_conv.bn.weight"], P["local_conv.bn.bias"], True, 0.1, 1e-5).permute(0, 2, 3, 1)
    n = ln(z, "mlp.norm").reshape(-1, C)
    lin = lambda v, m: v @ P[f"mlp.ffn.{m}.weight"].t() + P[f"mlp.ffn.{m}.bias"]  # noqa: E731
    f = lin(torch.nn.functional.silu(lin(n, "gate")) * lin(n, "up"), "down")
    return z + (f * held[1] / keep).view_as(z), P


@pytest.mark.parametrize("drop", [0.0, 0.25])
def test_block_with_all_operators(tv, drop):
    from semiuhpe_amd import kernels as K
    torch.manual_seed(3)
    B, H, W, dim, heads, ws = 2, 14, 14, 96, 3, 7
    blk = tv.TinyViTBlock(dim, (H, W), heads, ws, 4.0, 0.0, mlp="gated", rope=True, drop=drop).cuda().train()
    assert blk.mlp.ffn.gate.weight.shape == (256, 96)
    with torch.no_grad():
        for p in blk.parameters():
            p.add_(0.05 * torch.randn_like(p))
    x = torch.randn(B, H, W, dim)
    dy = torch.randn(B, H, W, dim)
    K.rng_counter(torch.device("cuda", torch.cuda.current_device()), seed=11)
    tape = []
    y = blk.fwd(x.cuda(), tape)
    dx = blk.bwd(dy.cuda(), tape)
    assert not tape
    per, keep = (B * H * W * dim + 3) // 4, float(torch.tensor(1.0 - drop, dtype=torch.float32))
    held = [R.kept(11, i * per, B * H * W * dim, keep).view(-1, dim).double() if drop else 1.0 for i in range(2)]
    xd = x.double().requires_grad_(True)
    ref, P = block64(blk, xd, held, keep, dim, heads, ws)
    ref.backward(dy.double())

    def close(got, want, what):
        # fp32 through some 20 layers of sums of up to 392 terms: each adds a relative 2^-24 sqrt(terms) to the 2-norm; 1e-5 is 8 times their sum
        off = float((got.detach().cpu().double() - want).norm() / want.norm())
        assert off < 1e-5, (what, off)
    close(y, ref.detach(), "y")
    close(dx, xd.grad, "dx")
    for k, p in blk.named_parameters():
        if P[k].grad.norm() > 1e-6 * P[k].norm():           # (qkv's k bias and the depthwise filter's mean have gradients of rounding alone)
            if k not in ("attn.qkv.bias",):
                close(p.grad, P[k].grad, k)


def test_default_block_is_unchanged(tv):
    """the options' defaults give the reference's block: the same parameters, and ResidualDropout is not on its way"""
    torch.manual_seed(0)
    a = tv.TinyViT21M()
    keys = list(a.state_dict())
    assert not any("ffn" in k for k in keys) and "layers.1.blocks.0.mlp.fc1.weight" in keys
    b = tv.TinyViT21M(mlp="gated", rope=True, drop=0.1)
    assert any(k.endswith("mlp.ffn.gate.weight") for k in b.state_dict())
    with pytest.raises(ValueError):
        tv.TinyViTBlock(96, (7, 7), 3, mlp="swiglu")
    with pytest.raises(ValueError):
        tv.TinyViTBlock(96, (7, 7), 3, drop=1.0)


def test_network_with_options_trains_and_evaluates(tv):
    """one step through the autograd bridge, drop_path and dropout on: finite, gradients for every parameter, the same bits from the same seed; eval needs no draw"""
    from types import SimpleNamespace

    from semiuhpe_amd import kernels as K
    torch.manual_seed(1)
    net = tv.get_TinyViT(SimpleNamespace(num_classes=9, vit_mlp="gated", vit_rope=True, vit_drop=0.1)).cuda()
    state = copy.deepcopy(net.state_dict())
    img = torch.randn(2, 3, 224, 224, device="cuda")
    dev = torch.device("cuda", torch.cuda.current_device())
    runs = []
    for _ in range(2):
        net.load_state_dict(state)
        net.train()
        for p in net.parameters():
            p.grad = None
        K.rng_counter(dev, seed=5)
        out = net(img)
        out.square().sum().backward()
        runs.append([out.detach().clone()] + [p.grad.clone() for p in net.parameters()])
    assert all(torch.isfinite(t).all() for t in runs[0])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    ffn = [p.grad for k, p in net.named_parameters() if "ffn" in k]
    assert len(ffn) == 60 and all(float(g.abs().sum()) > 0 for g in ffn)
    net.eval()
    with torch.no_grad():
        e = net(img)
        assert torch.equal(e, net(img))


def test_mask_hook_reaches_the_residual_dropout(tv):
    from semiuhpe_amd import layers as L
    drop = L.ResidualDropout(0.5).train()
    x, skip = torch.randn(4, 8, device="cuda"), torch.randn(4, 8, device="cuda")
    mask = (torch.arange(32).view(4, 8) % 2).float() * 2
    L.set_mask_hook(lambda kind, shape, keep: mask if kind == "dropout" else None)
    try:
        tape = []
        y = drop.fwd2(x, skip, tape)
        d, s = drop.bwd2(torch.ones_like(x), tape)
    finally:
        L.set_mask_hook(None)
    assert torch.equal(y.cpu(), skip.cpu() + x.cpu() * mask) and torch.equal(d.cpu(), mask) and (s == 1).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_sixteen_bit_half_block(dtype):
    """LayerNorm -> gated feed-forward -> residual dropout as layers on 16-bit rows: the sum of the parts' own 64-bit forms, gradients in the weights' type"""
    from semiuhpe_amd import kernels as K, layers as L
    t = R.TYPES[dtype]
    torch.manual_seed(2)
    norm, ffn, drop = L.LayerNorm(64).cuda(), L.GatedFeedForward(64, 96).cuda().to(t), L.ResidualDropout(0.2).train()
    x, dy = torch.randn(50, 64).to(t), torch.randn(50, 64).to(t)
    K.rng_counter(torch.device("cuda", torch.cuda.current_device()), seed=9)
    tape = []
    n = norm.fwd(x.cuda(), tape)
    f = ffn.fwd(n, tape)
    y = drop.fwd2(f, x.cuda(), tape)
    d_branch, d_skip = drop.bwd2(dy.cuda(), tape)
    dn = ffn.bwd(d_branch, tape)
    dx = norm.bwd(dn, tape, skip=d_skip)
    assert not tape and dx.dtype == t and ffn.gate.weight.grad.dtype == t and norm.weight.grad.dtype == torch.float32
    keep = float(torch.tensor(0.8, dtype=torch.float32))
    held = R.kept(9, 0, 50 * 64, keep)
    w, b = [m.weight for m in (ffn.gate, ffn.up, ffn.down)], [m.bias for m in (ffn.gate, ffn.up, ffn.down)]
    R.within(n, *R.layernorm(x, dy, 1e-5, norm.weight, norm.bias)["y"], "norm")
    ref = R.gated_ffn(n, *w, *b, d_branch, "silu")
    R.within(f, *ref["y"], "ffn")
    R.within(y, *R.dropout(f, held, keep, x), "dropout + skip")
    R.within(d_branch, *R.dropout(dy, held, keep), "gradient of dropout")
    R.within(dn, *ref["dx"], "gradient of ffn")
    R.within(ffn.gate.weight.grad, *ref["dwg"], "dwg")
    R.within(ffn.down.bias.grad, *ref["dbd"], "dbd")
    R.within(dx, *R.layernorm(x, dn, 1e-5, norm.weight, norm.bias, skip=d_skip)["dx"], "gradient of norm + skip")
