"""The MoE layer for the few tokens of a decode step against its definition in 64 bits."""
import math

import pytest
import torch


def weights(T, d, f, E, shared, dtype, seed):
    g = torch.Generator().manual_seed(seed)

    def w(*shape, fan_in):
        return (torch.randn(*shape, generator=g) / math.sqrt(fan_in)).to(dtype)
    x = w(T, d, fan_in=1.0)
    Wg = torch.randn(d, E, generator=g) / math.sqrt(d)
    ws = [w(E, d, f, fan_in=d), w(E, d, f, fan_in=d), w(E, f, d, fan_in=f)]
    sh = (w(d, f, fan_in=d), w(d, f, fan_in=d), w(f, d, fan_in=f)) if shared else None
    return x, Wg, ws, sh


def definition(x, Wg, ws, sh, k):
    """out, and a bound on the error of: 32-bit sums (a unit of the running sum per step: the tensor cores may truncate),
    an exponential good to 2^-20, the intermediate rounded to bf16 (bf16 inputs only), one rounding of the result."""
    bf16 = x.dtype == torch.bfloat16
    u = 2.0 ** -23
    X = x.double()
    T, d = X.shape
    E = Wg.shape[1]
    z = torch.stack([(X * Wg[:, e].double()).sum(1) for e in range(E)], dim=1)      # equal columns give equal logits
    out, err = torch.zeros_like(X), torch.zeros_like(X)
    pick = [sorted(range(E), key=lambda e: (-r[e], e))[:k] for r in z.tolist()]

    def mlp(rows, gate, W1, W3, W2):
        W1, W3, W2 = W1.double(), W3.double(), W2.double()
        f = W1.shape[1]
        a, b = rows @ W1, rows @ W3
        da, db = (d + 1) * u * (rows.abs() @ W1.abs()), (d + 1) * u * (rows.abs() @ W3.abs())
        sa = a * torch.sigmoid(a)
        h = gate[:, None] * sa * b
        # |silu'| <= 1.1, silu itself is off by the exponential's error and two roundings
        dh = gate.abs()[:, None] * ((1.1 * da + sa.abs() * 2.0 ** -18) * (b.abs() + db) + (sa.abs() + 1.1 * da) * db)
        dh = dh + h.abs() * 2.0 ** -20
        if bf16:
            dh = dh + (h.abs() + dh) * 2.0 ** -8
        return h @ W2, dh @ W2.abs() + (f + 1) * u * ((h.abs() + dh) @ W2.abs())
    for t in range(T):
        zt = z[t, pick[t]]
        w = torch.softmax(zt, dim=0)
        for j, e in enumerate(pick[t]):
            o, q = mlp(X[t:t + 1], w[j:j + 1], *(m[e] for m in ws))
            out[t] += o[0]
            err[t] += q[0] + (k + 2) * u * o[0].abs()
    if sh is not None:
        o, q = mlp(X, torch.ones(T, dtype=torch.float64), *sh)
        out += o
        err += q
    err = err + (k + 1) * u * out.abs()
    err = err + (out.abs() + err) * (2.0 ** -8 if bf16 else 2.0 ** -24)
    return out, err


def check(got, want, err):
    diff = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    assert (diff <= err).all(), f"worst {float((diff / err).max()):.3f} of the bound, error {float(diff.max()):.3e}"


def test_c_entry_point_refuses_bad_arguments():
    from flashdmla import _lib
    L = _lib.lib()
    ws = L.fdmla_moe_few_workspace_bytes(4, 128, 64, 8, 2, 0, 1)
    assert ws > 0
    assert L.fdmla_moe_few_workspace_bytes(129, 128, 64, 8, 2, 0, 1) == 0
    call = lambda ptrs, wsb, T, d, f, E, k, dt=1: L.fdmla_moe_few(*ptrs, 256, wsb, T, d, f, E, k, dt, None)
    null, one = (None,) * 9, (256,) * 9
    assert call(null, 0, 0, 128, 64, 8, 2) == 0                               # no tokens
    assert call(null, ws, 4, 128, 64, 8, 2) == -1
    assert call(one, ws, 4, 128, 64, 8, 2, 5) == -1                           # dtype
    assert call(one, ws, 4, 0, 64, 8, 2) == -1
    assert call((256,) * 6 + (None, 256, 256), ws, 4, 128, 64, 8, 2) == -1    # half a shared expert
    assert call(one, ws, 129, 128, 64, 8, 2) == -2                            # too many tokens
    assert call(one, ws, 4, 128, 64, 8, 9) == -2                              # more choices than experts
    assert call(one, ws, 4, 128, 64, 40, 33) == -2
    assert call(one, ws, 4, 128, 64, 4096, 2) == -2
    assert call(one, 100, 4, 128, 64, 8, 2) == -4                             # workspace


def test_refuses_cpu_tensors():
    import flashdmla as F
    x, Wg, ws, sh = weights(2, 64, 64, 4, False, torch.float32, 0)
    with pytest.raises(F.FlashDMLAError):
        F.moe_few(x, Wg, *ws, 2)


CASES = [
    # T, d, f, E, k, shared, dtype
    (1, 64, 64, 1, 1, False, torch.bfloat16),
    (1, 1024, 512, 8, 2, False, torch.bfloat16),
    (1, 128, 64, 64, 8, True, torch.bfloat16),
    (2, 192, 320, 5, 5, True, torch.bfloat16),                # every expert, odd numbers of 64-wide blocks
    (16, 256, 128, 16, 4, False, torch.bfloat16),
    (17, 576, 192, 40, 3, True, torch.bfloat16),
    (32, 128, 1024, 8, 2, False, torch.bfloat16),
    (37, 2112, 704, 12, 5, False, torch.bfloat16),
    (64, 512, 256, 100, 8, True, torch.bfloat16),
    (65, 320, 64, 33, 32, False, torch.bfloat16),
    (128, 256, 192, 300, 8, True, torch.bfloat16),
    (128, 64, 64, 3, 1, True, torch.bfloat16),
    (4, 4096, 256, 8, 2, True, torch.bfloat16),               # few tiles, long sums: many pieces per tile
    (128, 1024, 512, 4, 2, True, torch.bfloat16),             # more than 64 tokens per expert
    (3, 100, 36, 7, 2, True, torch.bfloat16),                 # widths the tensor cores do not take
    (1, 33, 5, 2, 1, False, torch.bfloat16),
    (1, 64, 128, 8, 2, True, torch.float32),
    (29, 200, 72, 11, 4, False, torch.float32),
    (128, 96, 64, 6, 3, True, torch.float32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,d,f,E,k,shared,dtype", CASES)
def test_layer_matches_the_definition(cuda, T, d, f, E, k, shared, dtype):
    import flashdmla as F
    x, Wg, ws, sh = weights(T, d, f, E, shared, dtype, seed=T * 7 + E)
    want, err = definition(x, Wg, ws, sh, k)
    dev = [t.to(cuda) for t in (x, Wg, *ws)]
    dsh = tuple(t.to(cuda) for t in sh) if sh else None
    out = F.moe_few(*dev, k, dsh)
    assert F.device_error_flag() == 0
    check(out, want, err)
    again = F.moe_few(*dev, k, dsh, out=torch.full_like(out, float("nan")))
    assert torch.equal(out, again)                            # no atomic decides an order


@pytest.mark.gpu
def test_cuda_core_kernels_take_the_same_shapes(cuda):
    import flashdmla as F
    x, Wg, ws, sh = weights(9, 256, 128, 16, True, torch.bfloat16, 5)
    want, err = definition(x, Wg, ws, sh, 4)
    F.set_backend(F.BACKEND_PORTABLE)
    try:
        out = F.moe_few(*[t.to(cuda) for t in (x, Wg, *ws)], 4, tuple(t.to(cuda) for t in sh))
        assert F.last_kernel() == "portable"
    finally:
        F.set_backend(F.BACKEND_AUTO)
    check(out, want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_skewed_choices_and_strange_tokens(cuda, dtype):
    """Equal logits go to the lower expert; all tokens may choose one expert; a token with a NaN or an infinity spoils its own
    row only; a token of zeros gives zeros."""
    import flashdmla as F
    T, d, f, E, k = 21, 128, 64, 12, 3
    x, Wg, ws, sh = weights(T, d, f, E, False, dtype, 11)
    Wg = Wg.clone()
    Wg[:, 5] = Wg[:, 2]                                        # 2 and 5 tie on every token
    Wg[:, 9] = Wg[:, 2]
    x = x.abs()
    Wg[:, 2] += 0.05
    Wg[:, 5] += 0.05
    Wg[:, 9] += 0.05
    x[4] = 0.0                                                 # all logits tie: experts 0, 1, 2
    want, err = definition(x, Wg, ws, None, k)
    out = F.moe_few(*[t.to(cuda) for t in (x, Wg, *ws)], k)
    check(out, want, err)
    assert (out[4] == 0).all()
    bad = x.clone()
    bad[7, 3] = float("nan")
    bad[11, 0] = float("inf")
    out2 = F.moe_few(*[t.to(cuda) for t in (bad, Wg, *ws)], k)
    rest = [t for t in range(T) if t not in (7, 11)]
    assert torch.equal(out2[rest], out[rest])
    assert out2[7].isnan().any() and not out2[11].isfinite().all()
    # infinities in an expert's weights reach the tokens that chose it, nobody else
    Wg2 = torch.randn(d, E, generator=torch.Generator().manual_seed(3)) / math.sqrt(d)
    out3 = F.moe_few(*[t.to(cuda) for t in (x, Wg2, *ws)], k)
    chose = torch.topk(x.double() @ Wg2.double(), k, dim=1).indices
    users = (chose == 1).any(1)
    users[4] = True                                            # the token of zeros chooses experts 0, 1, 2
    assert 0 < int(users.sum()) < T
    ws2 = [w.clone() for w in ws]
    for w in ws2:
        w[1, 3, 5] = float("inf")
    out4 = F.moe_few(*[t.to(cuda) for t in (x, Wg2, *ws2)], k)
    assert torch.equal(out4[~users], out3[~users])
    users[4] = False
    assert not out4[users].isfinite().all(dim=1).any()
    assert F.device_error_flag() == 0


@pytest.mark.gpu
def test_layer_object_strides_streams_and_graph(cuda):
    from flashdmla import FlashDMLAError, MoEFFN
    layer = MoEFFN(d_model=256, d_ff=128, n_experts=16, top_k=4, device=cuda, seed=3)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(256, 24, generator=g).to(torch.bfloat16).to(cuda)
    xt = x.t()                                                 # strided input
    y = layer.forward_few(xt)
    want, err = definition(xt.cpu(), layer.Wg.cpu(), [t.cpu() for t in (layer.W1, layer.W3, layer.W2)],
                           tuple(t.cpu() for t in layer.shared), 4)
    check(y, want, err)
    # with room for everybody the layer with a capacity computes the same up to its own roundings (bf16 after every product)
    z = layer.forward(xt.contiguous(), capacity=24)
    assert (z.float() - y.float()).abs().max() <= 0.05 * y.float().abs().max()
    s1, s2 = torch.cuda.Stream(device=cuda), torch.cuda.Stream(device=cuda)
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2, s1, s2):                                 # two calls in flight at once, each with its own scratch
        with torch.cuda.stream(s):
            outs.append(layer.forward_few(xt))
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for o in outs)
    xin, out = torch.zeros_like(xt.contiguous()), torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward_few(xin, out)
    for src in (xt, xt.flip(0), xt):
        xin.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer.forward_few(src))
    # two calls side by side inside one graph
    fork, outs = torch.cuda.CUDAGraph(), [torch.empty_like(y) for _ in range(2)]
    with torch.cuda.graph(fork):
        cur = torch.cuda.current_stream()
        s1.wait_stream(cur)
        with torch.cuda.stream(s1):
            layer.forward_few(xin, outs[0])
        layer.forward_few(xin, outs[1])
        cur.wait_stream(s1)
    for _ in range(5):
        fork.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], y) and torch.equal(outs[1], y)
    assert layer.forward_few(xt[:0]).shape == (0, 256)
    with pytest.raises(FlashDMLAError):
        layer.forward_few(torch.zeros(129, 256, dtype=torch.bfloat16, device=cuda))


@pytest.mark.gpu
def test_refusals(cuda):
    import flashdmla as F
    x, Wg, ws, sh = weights(4, 64, 64, 4, True, torch.bfloat16, 0)
    ok = [t.to(cuda) for t in (x, Wg, *ws)]
    dsh = tuple(t.to(cuda) for t in sh)

    def call(i=None, t=None, k=2, shared=dsh, **kw):
        a = list(ok)
        if i is not None:
            a[i] = t
        with pytest.raises(F.FlashDMLAError):
            F.moe_few(*a, k, shared, **kw)
    call(0, ok[0].float())
    call(0, ok[0].half())
    call(0, ok[0][:, :32])
    call(1, ok[1].bfloat16())
    call(1, ok[1][:, :3])
    call(2, ok[2][:2])
    call(4, ok[4].transpose(1, 2)[:, :, :32])
    call(3, ok[3].cpu())
    call(k=0)
    call(k=5)
    call(shared=(dsh[0], dsh[1], dsh[2][:32]))
    call(out=torch.empty(4, 64, device=cuda))
    call(out=torch.empty(64, 4, dtype=torch.bfloat16, device=cuda).t())


@pytest.mark.gpu
def test_tensors_that_start_at_odd_addresses(cuda):
    """Views a few elements into larger buffers: the kernels that copy in bulk step aside."""
    import flashdmla as F
    x, Wg, ws, sh = weights(5, 128, 64, 6, True, torch.bfloat16, 9)
    want, err = definition(x, Wg, ws, sh, 2)

    def view(t, shift):
        buf = torch.zeros(t.numel() + 32, dtype=t.dtype, device=cuda)
        v = buf[shift:shift + t.numel()].view(t.shape)
        v.copy_(t)
        return v
    for shift in (1, 4):
        for which in range(9):
            ts = [view(t, shift if i == which else 0) for i, t in enumerate((x, Wg, *ws, *sh, torch.zeros_like(x)))]
            out = F.moe_few(*ts[:5], 2, tuple(ts[5:8]), out=ts[8])
            check(out, want, err)
    assert F.device_error_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_random_shapes(cuda, seed):
    import random
    import flashdmla as F
    r = random.Random(seed)
    T, E = r.choice([1, 2, 3, 5, 15, 16, 17, 33, 64, 65, 100, 128]), r.randint(1, 70)
    d, f, k = 64 * r.randint(1, 12), 64 * r.randint(1, 9), r.randint(1, min(E, 9))
    x, Wg, ws, sh = weights(T, d, f, E, r.random() < 0.5, torch.bfloat16, 100 + seed)
    want, err = definition(x, Wg, ws, sh, k)
    out = F.moe_few(*[t.to(cuda) for t in (x, Wg, *ws)], k, tuple(t.to(cuda) for t in sh) if sh else None)
    check(out, want, err)


# 2 to 16 tokens of wider layers: more than 256 * 148 elements of h, summed four columns a thread
SMALL_BATCHES = [
    # T, d, f, E, k, shared
    (3, 1024, 2048, 9, 8, True),
    (4, 256, 2048, 16, 8, True),
    (5, 64, 4096, 8, 8, False),                               # one step of d: tiles are not cut
    (16, 320, 1216, 24, 6, False),                            # half a tile of f at the end
    (16, 192, 2496, 12, 4, True),
    (9, 2112, 704, 11, 7, True),
    (13, 512, 256, 20, 12, True),                             # more than nine terms in the weighted sum
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,d,f,E,k,shared", SMALL_BATCHES)
def test_small_batches_of_wide_layers(cuda, T, d, f, E, k, shared):
    import flashdmla as F
    assert 1 < T <= 16 and T * (k + shared) * f > 256 * 148
    x, Wg, ws, sh = weights(T, d, f, E, shared, torch.bfloat16, seed=T * 11 + E)
    want, err = definition(x, Wg, ws, sh, k)
    dev = [t.to(cuda) for t in (x, Wg, *ws)]
    dsh = tuple(t.to(cuda) for t in sh) if sh else None
    out = F.moe_few(*dev, k, dsh)
    assert F.last_kernel() == "tcgen05" and F.device_error_flag() == 0
    check(out, want, err)
    for _ in range(3):
        assert torch.equal(out, F.moe_few(*dev, k, dsh))
    assert F.moe_few(*dev, k, dsh, out=dev[0]) is dev[0] and torch.equal(out, dev[0])        # in place of the tokens


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 20])
def test_outputs_stay_as_they_were_after_a_time_out(cuda, T):
    """While the flag of an earlier time-out stands a call writes nothing; once it is cleared, calls work again."""
    import flashdmla as F
    from flashdmla import _lib
    x, Wg, ws, sh = weights(T, 256, 128, 16, True, torch.bfloat16, 5)
    want, err = definition(x, Wg, ws, sh, 4)
    dev = [t.to(cuda) for t in (x, Wg, *ws)]
    dsh = tuple(t.to(cuda) for t in sh)
    out = torch.full((T, 256), 7.0, dtype=torch.bfloat16, device=cuda)
    try:
        assert _lib.lib().fdmla_set_device_error_flag(44) == 0
        F.moe_few(*dev, 4, dsh, out=out)
        assert (out == 7).all() and F.device_error_flag(reset=True) == 44
        F.moe_few(*dev, 4, dsh, out=out)
    finally:
        F.device_error_flag(reset=True)
    check(out, want, err)
