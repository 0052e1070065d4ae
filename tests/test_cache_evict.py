"""A latent cache that may not grow: the attention weight every row has received, eviction, and both inside
PagedLatentCache."""
import math

import numpy as np
import pytest
import torch


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def evict_oracle(weights, positions, lens, nxt, keep, recent):
    """Per sequence: the row each row j < min(n, keep) held before.  weights, positions: lists of arrays in row order."""
    out = []
    for w, p, n, x in zip(weights, positions, lens, nxt):
        K = min(n, keep)
        src = list(range(K))
        if n > keep:
            def rank(i):                                      # protected rows, then by weight (NaN last), then the lower row
                return (0, 0, 0.0, i) if p[i] >= x - recent else (1, 1, 0.0, i) if np.isnan(w[i]) else (1, 0, -float(w[i]), i)
            order = sorted(range(n), key=rank)
            stays = np.zeros(n, dtype=bool)
            stays[order[:K]] = True
            for hole, mover in zip(np.flatnonzero(~stays[:K]), K + np.flatnonzero(stays[K:])):
                src[hole] = int(mover)
        out.append(src)
    return out


def accumulate_oracle(Q, keys, m, l, scale, causal=True):
    """Weight each key receives (64 bits) and a bound on the error of a 32-bit evaluation.  Q [H,Sq,d], keys [n,d]."""
    H, Sq, d = Q.shape
    n = keys.shape[0]
    q, k = Q.double().reshape(H * Sq, d), keys.double()
    s = q @ k.T * scale
    vis = torch.ones(H * Sq, n, dtype=torch.bool)
    if causal:
        i = torch.arange(Sq).repeat(H)
        vis = torch.arange(n)[None, :] <= (i + n - Sq)[:, None]
    ok = (l.double().reshape(-1) > 0)[:, None] & vis
    mm = torch.where(ok, m.double().reshape(-1, 1).expand_as(s), torch.zeros_like(s))
    ll = torch.where(ok, l.double().reshape(-1, 1).expand_as(s), torch.ones_like(s))
    p = torch.where(ok, torch.exp(torch.where(ok, s - mm, torch.zeros_like(s))) / ll, torch.zeros_like(s))
    # d products summed in 32 bits, each step off by at most a unit in the last place of the running sum (2^-23: the tensor
    # cores may truncate), the exponent's argument and the exponential by a few, R values summed per key
    ds = (d + 2) * 2.0 ** -23 * (q.abs() @ k.abs().T) * scale
    arg = 4 * 2.0 ** -23 * (s.abs() + mm.abs())
    err = (p * (torch.expm1(ds + arg) + 2.0 ** -20)).sum(0) + H * Sq * 2.0 ** -23 * p.sum(0)
    return p.sum(0), err


def stats(Q, keys, scale, causal=True):
    H, Sq, d = Q.shape
    n = keys.shape[0]
    s = torch.einsum("hqd,nd->hqn", Q.double(), keys.double()) * scale
    if causal:
        s = s.masked_fill(torch.arange(n)[None, None, :] > (torch.arange(Sq) + n - Sq)[None, :, None], float("-inf"))
    m = s.amax(-1) if n else torch.full((H, Sq), float("-inf"), dtype=torch.float64)
    l = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m)[..., None]).sum(-1)
    return m.float(), l.float()


def paged(lens, page, d, dtype, g, spare=3, std=1.0):
    """Rows of every sequence on permuted pages of a pool whose other rows hold NaN; (pool, table, physical rows)."""
    per = [(n + page - 1) // page for n in lens]
    N = sum(per) + spare
    perm = torch.randperm(N, generator=g)
    pool = torch.full((N, page, d), float("nan"), dtype=dtype)
    table = torch.zeros(len(lens), max(max(per), 1) + 1, dtype=torch.int32)
    phys, o = [], 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = perm[o:o + per[b]].to(torch.int32)
        t = torch.arange(n)
        rows = table[b].long()[t // page] * page + t % page
        pool.view(-1, d)[rows] = (torch.randn(n, d, generator=g) * std).to(dtype)
        phys.append(rows)
        o += per[b]
    return pool, table, phys


# ---------------------------------------------------------------------------------------------------- host side, no GPU
def test_shrinking_gives_pages_back_without_a_gpu():
    from flashdmla import FlashDMLAError
    from flashdmla.cache import PagedLatentCache
    c = PagedLatentCache(num_pages=10, page_size=4, d_qk=8, max_seqs=3, max_pages_per_seq=8, device="cpu", track_weights=True)
    a, b = c.new_sequence(), c.new_sequence()
    c.reserve([a], 18)
    c.reserve([b], 3)
    first = c.pages_of(a)
    assert c.free_pages == 4 and c.position(a) == 18
    c._shrink([a, b], 9)
    assert c.length(a) == 9 and c.position(a) == 18 and c.pages_of(a) == first[:3]
    assert c.length(b) == 3 and c.position(b) == 3 and len(c.pages_of(b)) == 1
    assert c.free_pages == 6 and c.h_table[a, 3:].tolist() == [0] * 5
    assert c.reserve([a], 1).tolist() == [9] and c.position(a) == 19          # rows go on at the end, positions too
    c.free_sequence(a)
    assert c.position(c.new_sequence()) == 0
    with pytest.raises(FlashDMLAError):
        c.evict([b], 2)                                                       # no CPU fallback


def test_slots_outside_the_cache_are_refused_before_anything_is_launched():
    """The tables are gathered on the GPU, where an index out of range would be a device assert.  Here the device side is the
    host's own tensors."""
    from flashdmla import FlashDMLAError
    from flashdmla.cache import PagedLatentCache
    c = PagedLatentCache(num_pages=10, page_size=4, d_qk=8, max_seqs=3, max_pages_per_seq=8, device="cpu", track_weights=True)
    a = c.new_sequence()
    c.reserve([a], 9)
    c.on_gpu, c.d_table, c.d_len = True, c.h_table.clone(), c.h_len.clone()
    assert c.tables([a, 2])[1].tolist() == [9, 0]
    for slots in ([3], [-1], [a, 10 ** 6]):
        for call in (lambda: c.tables(slots), lambda: c.evict(slots, 4), lambda: c.gather(slots, 1),
                     lambda: c.decode(torch.zeros(len(slots), 2, 8), slots, 4)):
            with pytest.raises(FlashDMLAError, match="slot"):
                call()
    assert c.length(a) == 9 and len(c.pages_of(a)) == 3


def test_bounds_that_an_int_does_not_hold_are_refused(monkeypatch):
    """Behind the binding they would be cut to 32 bits: keep = 2^32 + 5 would leave five rows."""
    import flashdmla as F
    from flashdmla import ops
    monkeypatch.setattr(ops, "_need_cuda", lambda *t: None)                   # the checks of arguments alone, on CPU tensors
    z = torch.zeros
    state = (z(1, 4, 8), z(1, 4), z(1, 4).int())
    for keep, recent in ((2 ** 32 + 5, 0), (2 ** 31, 0), (2 ** 30 + 1, 3), (0, 0), (4, 5)):
        with pytest.raises(F.FlashDMLAError, match="keep"):
            F.cache_evict(*state, z(1, 1).int(), z(1).int(), z(1).int(), keep, recent)
    for n in (2 ** 32 + 1, 2 ** 31, -1):
        with pytest.raises(F.FlashDMLAError, match="n_tokens"):
            F.cache_stamp(*state[1:], z(1, 1).int(), z(1).int(), z(1).int(), n)


def test_positions_that_an_int_does_not_hold_are_refused():
    """A bounded cache may go on for ever, its positions are 32-bit."""
    from flashdmla import FlashDMLAError
    from flashdmla.cache import PagedLatentCache
    c = PagedLatentCache(num_pages=10, page_size=4, d_qk=8, max_seqs=2, max_pages_per_seq=8, device="cpu", track_weights=True)
    a, b = c.new_sequence(), c.new_sequence()
    c.reserve([a], 3)
    c.h_next[a] = 2 ** 31 - 3
    assert c.reserve([a], 2).tolist() == [3] and c.position(a) == 2 ** 31 - 1
    with pytest.raises(FlashDMLAError, match="position"):
        c.reserve([b, a], 1)
    assert c.position(a) == 2 ** 31 - 1 and c.length(a) == 5 and c.length(b) == 0 and c.free_pages == 8


def test_c_entry_points_refuse_bad_arguments():
    from flashdmla import _lib
    L = _lib.lib()
    acc = lambda *a: L.fdmla_cache_accumulate(*a)
    p8 = (1,) * 7
    assert acc(*(None,) * 7, None, 0, 0, 8, 1, 576, 64, 4, 4, 0.1, 1, 1, None) == 0            # empty batch
    assert acc(*(None,) * 7, None, 0, 2, 8, 1, 576, 64, 4, 4, 0.1, 1, 1, None) == -1           # null pointers
    assert acc(*p8, None, 0, 2, 8, 1, 576, 64, 4, 4, 0.1, 1, 7, None) == -1                    # dtype
    assert acc(*p8, None, 0, 2, 8, 1, 576, 0, 4, 4, 0.1, 1, 1, None) == -1                     # page size
    assert acc(*p8, None, 0, 2, 8, 1, 576, 1 << 20, 1 << 12, 4, 0.1, 1, 1, None) == -2         # more rows than an int counts
    assert acc(*p8, None, 0, 2, 8, 1, 4000, 64, 4, 4, 0.1, 1, 0, None) == -2                   # wider than the kernels take
    ev = lambda *a: L.fdmla_cache_evict(*a)
    assert ev(*(None,) * 9, 0, 0, 4, 0, 576, 64, 4, 4, 1, None) == 0
    assert ev(*(None,) * 9, 0, 1, 4, 0, 576, 64, 4, 4, 1, None) == -1
    assert ev(*(1,) * 9, 1 << 20, 1, 0, 0, 576, 64, 4, 4, 1, None) == -1                       # keep 0
    assert ev(*(1,) * 9, 1 << 20, 1, 4, 5, 576, 64, 4, 4, 1, None) == -1                       # recent > keep
    assert ev(*(1,) * 9, 15, 1, 4, 0, 576, 64, 4, 4, 1, None) == -4                            # workspace
    assert ev(*(1,) * 9, 1 << 30, 1, 4, 0, 576, 64, 20000, 4, 1, None) == -2                   # too many rows per sequence
    assert ev(*(1,) * 9, 1 << 30, 1, 4, 0, 576, 1, 2 ** 31 - 1, 4, 1, None) == -2
    assert ev(*(256,) * 9, 1 << 30, 1, 2 ** 30 + 1, 0, 576, 64, 4, 4, 1, None) == -2
    assert L.fdmla_cache_evict_workspace_bytes(3, 100, 64, 1) == 2 * 3 * 64 * 4
    assert L.fdmla_cache_stamp(None, None, None, None, None, 0, 1, 64, 4, 4, None) == 0
    assert L.fdmla_cache_stamp(None, None, None, None, None, 1, 1, 64, 4, 4, None) == -1


def test_operators_refuse_cpu_tensors():
    import flashdmla as F
    z = torch.zeros
    with pytest.raises(F.FlashDMLAError):
        F.accumulate_weights(z(1, 2, 8), z(1, 4, 8), z(1, 1).int(), z(1).int(), z(1, 2), z(1, 2), z(1, 4))
    with pytest.raises(F.FlashDMLAError):
        F.cache_evict(z(1, 4, 8), z(1, 4), z(1, 4).int(), z(1, 1).int(), z(1).int(), z(1).int(), 2)


# ------------------------------------------------------------------------------------------------------------ eviction
def evict_case(lens, keep, recent, page, d, dtype, kind, seed):
    g = torch.Generator().manual_seed(seed)
    pool, table, phys = paged(lens, page, d, dtype, g)
    weights = torch.randn(pool.shape[:2], generator=g).exp()
    if kind == "ties":                                        # three different weights, zeros of both signs
        weights = torch.randint(0, 3, pool.shape[:2], generator=g).float() * torch.where(torch.rand(pool.shape[:2], generator=g) < 0.5, 1.0, -0.0)
    elif kind == "equal":
        weights = torch.ones(pool.shape[:2])
    elif kind == "wild":                                      # infinities, NaN, denormals, negative values
        pick = torch.randint(0, 8, pool.shape[:2], generator=g)
        vals = torch.tensor([float("inf"), float("nan"), 1e-42, -1.0, 3.4e38, 0.0, -0.0, float("-inf")])
        weights = torch.where(torch.rand(pool.shape[:2], generator=g) < 0.5, vals[pick], weights)
    positions = torch.full(pool.shape[:2], -1, dtype=torch.int32)
    nxt = []
    for n, rows in zip(lens, phys):
        seen = n + n // 3
        positions.view(-1)[rows] = torch.randperm(max(seen, 1), generator=g)[:n].to(torch.int32)
        nxt.append(seen)
    return pool, weights, positions, table, phys, nxt


def check_evicted(got, case, lens, keep, recent):
    pool, weights, positions, table, phys, nxt = case
    gpool, gw, gp, kept, new = got
    src = evict_oracle([weights.view(-1)[r].numpy() for r in phys], [positions.view(-1)[r].numpy() for r in phys], lens, nxt, keep, recent)
    assert new.tolist() == [min(n, keep) for n in lens]
    want_pool, want_w, want_p = pool.clone(), weights.clone(), positions.clone()
    d = pool.shape[2]
    for b, s in enumerate(src):
        assert kept[b].tolist() == s + [-1] * (keep - len(s)), f"sequence {b}"
        to, frm = phys[b][:len(s)], phys[b][torch.tensor(s, dtype=torch.long)]
        want_pool.view(-1, d)[to] = pool.view(-1, d)[frm]
        want_w.view(-1)[to] = weights.view(-1)[frm]
        want_p.view(-1)[to] = positions.view(-1)[frm]
    bits = {torch.float32: torch.int32, torch.bfloat16: torch.int16}
    assert torch.equal(gpool.view(bits[pool.dtype]), want_pool.view(bits[pool.dtype]))     # rows from keep on as they were
    assert torch.equal(gw.view(torch.int32), want_w.view(torch.int32)) and torch.equal(gp, want_p)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,keep,recent,page,d,dtype,kind", [
    ([10], 4, 0, 4, 8, torch.float32, "random"),
    ([10], 4, 4, 4, 8, torch.float32, "random"),              # only the newest
    ([1, 0, 2, 700], 1, 1, 16, 3, torch.bfloat16, "random"),  # rows of 6 bytes
    ([64, 65, 63, 129], 64, 7, 64, 576, torch.bfloat16, "ties"),
    ([2000, 5, 1025, 1999], 1000, 100, 64, 576, torch.bfloat16, "equal"),
    ([3000, 2999], 2998, 50, 48, 160, torch.float32, "wild"),
    ([9000, 4097, 300], 4096, 512, 64, 64, torch.bfloat16, "ties"),       # several CTAs a sequence
    ([70001], 30000, 1, 64, 64, torch.bfloat16, "random"),
    ([70001, 12], 69999, 3000, 64, 8, torch.float32, "wild"),
    ([33] * 300, 17, 4, 16, 64, torch.bfloat16, "random"),
])
def test_evict_matches_the_definition(cuda, lens, keep, recent, page, d, dtype, kind):
    import flashdmla as F
    case = evict_case(lens, keep, recent, page, d, dtype, kind, seed=len(lens) * 1000 + keep)
    pool, weights, positions, table, phys, nxt = case
    dp, dw, dpos = pool.to(cuda), weights.to(cuda), positions.to(cuda)
    kept, new = F.cache_evict(dp, dw, dpos, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                              torch.tensor(nxt, dtype=torch.int32, device=cuda), keep, recent)
    check_evicted((dp.cpu(), dw.cpu(), dpos.cpu(), kept.cpu(), new.cpu()), case, lens, keep, recent)
    assert F.device_error_flag() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("capacity", [9000, 131072, 700000])
@pytest.mark.parametrize("kind", ["random", "ties", "wild"])
def test_evict_with_a_table_far_wider_than_the_lengths(cuda, capacity, kind):
    """The CTAs of a sequence share its rows by the table's capacity: some have none, and the others hold all of them."""
    import flashdmla as F
    lens, keep, recent, page, d = [700, 5000, 301, 64, 0, 300, 8999], 300, 40, 64, 64
    case = evict_case(lens, keep, recent, page, d, torch.bfloat16, kind, seed=capacity)
    pool, weights, positions, table, phys, nxt = case
    wide = torch.full((len(lens), -(-capacity // page)), 10 ** 9, dtype=torch.int32)         # no page of the rest is looked at
    for b, n in enumerate(lens):
        wide[b, :-(-n // page)] = table[b, :-(-n // page)]
    dp, dw, dpos = pool.to(cuda), weights.to(cuda), positions.to(cuda)
    kept, new = F.cache_evict(dp, dw, dpos, wide.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                              torch.tensor(nxt, dtype=torch.int32, device=cuda), keep, recent)
    check_evicted((dp.cpu(), dw.cpu(), dpos.cpu(), kept.cpu(), new.cpu()), case, lens, keep, recent)
    assert F.device_error_flag() == 0


@pytest.mark.gpu
def test_evict_in_a_graph_on_another_stream_with_shared_lengths(cuda):
    """Captured once, replayed on new contents; the new lengths overwrite the old ones (C entry point)."""
    import flashdmla as F
    from flashdmla import _lib
    lens, keep, recent = [500, 80, 1000], 200, 20
    cases = [evict_case(lens, keep, recent, 64, 128, torch.bfloat16, kind, seed=s) for s, kind in ((1, "random"), (1, "ties"))]
    pool, weights, positions, table, phys, nxt = cases[0]
    bufs = [t.to(cuda) for t in (pool, weights, positions)]
    dtab, dnext = table.to(cuda), torch.tensor(nxt, dtype=torch.int32, device=cuda)
    dl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    kept = torch.empty(len(lens), keep, dtype=torch.int32, device=cuda)
    L = _lib.lib()
    ws = torch.empty(L.fdmla_cache_evict_workspace_bytes(len(lens), keep, 64, table.shape[1]), dtype=torch.uint8, device=cuda)

    def call():
        rc = L.fdmla_cache_evict(*[t.data_ptr() for t in bufs], dtab.data_ptr(), dl.data_ptr(), dnext.data_ptr(), kept.data_ptr(),
                                 dl.data_ptr(), ws.data_ptr(), ws.numel(), len(lens), keep, recent, 128, 64, table.shape[1],
                                 pool.shape[0], _lib.BF16, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    check_evicted([t.cpu() for t in (*bufs, kept, dl)], cases[0], lens, keep, recent)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for case in cases[::-1]:
        for t, v in zip(bufs, case[:3]):
            t.copy_(v)
        dl.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        check_evicted([t.cpu() for t in (*bufs, kept, dl)], case, lens, keep, recent)


@pytest.mark.gpu
def test_evict_reports_bad_pages_and_lengths(cuda):
    """A page id outside the pool is neither read nor written: its rows count as the lightest (code 4)."""
    import flashdmla as F
    lens, keep = [128, 100], 70
    pool, weights, positions, table, phys, nxt = evict_case(lens, keep, 0, 64, 64, torch.bfloat16, "random", 5)
    bad = table.clone()
    bad[0, 1] = pool.shape[0] + 5
    bad[1, 0] = -3
    dp, dw, dpos = pool.to(cuda), weights.to(cuda), positions.to(cuda)
    kept, new = F.cache_evict(dp, dw, dpos, bad.to(cuda), torch.tensor([128, 100], dtype=torch.int32, device=cuda),
                              torch.tensor([0, 0], dtype=torch.int32, device=cuda) + 10 ** 6, keep)
    assert F.device_error_flag(reset=True) == 4
    # sequence 0: all 64 good rows stay, the first six of the bad page fill up; sequence 1: 36 good rows behind, 34 bad ones
    assert kept[0].tolist() == list(range(70)) and new.tolist() == [70, 70]
    assert sorted(kept[1].tolist())[-30:] == list(range(70, 100))
    lens2 = torch.tensor([-5, 10 ** 9], dtype=torch.int32, device=cuda)       # clamped to 0 and to the table's capacity
    kept, new = F.cache_evict(dp, dw, dpos, table.to(cuda)[:, :2].contiguous(), lens2, lens2.abs(), keep)
    assert new.tolist() == [0, 70] and kept[0].tolist() == [-1] * 70
    assert F.device_error_flag(reset=True) == 4


@pytest.mark.gpu
def test_evict_refusals(cuda):
    import flashdmla as F
    pool, weights, positions, table, phys, nxt = evict_case([100], 50, 0, 64, 64, torch.bfloat16, "random", 5)
    ok = [t.to(cuda) for t in (pool, weights, positions, table)] + [torch.tensor([100], dtype=torch.int32, device=cuda)] * 2

    def call(i, t, keep=50, recent=0):
        a = list(ok)
        if i is not None:
            a[i] = t
        with pytest.raises(F.FlashDMLAError):
            F.cache_evict(*a, keep, recent)
    call(0, ok[0].transpose(0, 1))
    call(0, ok[0].half())
    call(1, ok[1].double())
    call(1, ok[1][:1])
    call(2, ok[2].long())
    call(3, ok[3].long())
    call(4, ok[4].long())
    call(5, ok[5].expand(2))
    call(4, ok[4].cpu())
    call(None, None, keep=0)
    call(None, None, keep=5, recent=6)
    call(None, None, keep=5, recent=-1)


# ------------------------------------------------------------------------------------------------------ accumulated weight
ACC_CASES = [
    # lens, H, Sq, d, page, dtype
    ([1], 1, 1, 64, 64, torch.bfloat16),
    ([0, 1, 63, 64, 65], 16, 1, 576, 64, torch.bfloat16),
    ([127, 128, 129, 700], 128, 1, 576, 64, torch.bfloat16),
    ([300, 900], 37, 1, 192, 128, torch.bfloat16),
    ([200, 31], 160, 1, 576, 64, torch.bfloat16),             # more than one tile of heads
    ([500, 130, 7], 8, 33, 576, 64, torch.bfloat16),          # a window of queries, longer than the last sequence
    ([260], 128, 9, 64, 64, torch.bfloat16),
    ([90, 200], 3, 200, 128, 64, torch.bfloat16),
    ([500, 130, 3, 256], 8, 4, 576, 64, torch.bfloat16),      # a few queries of a few heads: one tile of query rows, masked
    ([300, 257, 15], 16, 16, 192, 64, torch.bfloat16),        # exactly one tile
    ([300, 2000], 1, 257, 64, 64, torch.bfloat16),            # one row more
    ([1500, 640, 0, 31], 128, 3, 576, 192, torch.bfloat16),   # pages that end inside a tile
    ([300, 20, 0], 8, 1, 160, 16, torch.float32),
    ([70, 33], 5, 4, 24, 48, torch.float32),
    ([70, 33], 5, 4, 31, 5, torch.bfloat16),                  # odd width and page
    ([100], 2, 1, 576, 1, torch.bfloat16),
]


def acc_inputs(lens, H, Sq, d, page, dtype, causal, seed=3):
    g = torch.Generator().manual_seed(seed + sum(lens) + H)
    pool, table, phys = paged(lens, page, d, dtype, g)
    Q = torch.randn(len(lens), H, Sq, d, generator=g).to(dtype)
    weights = torch.randn(pool.shape[:2], generator=g).exp()
    scale = 1.0 / math.sqrt(d)
    st = [stats(Q[b], pool.view(-1, d)[r], scale, causal) for b, r in enumerate(phys)]
    return pool, table, phys, Q, weights, scale, torch.stack([s[0] for s in st]), torch.stack([s[1] for s in st])


def check_accumulated(got, inputs, causal):
    pool, table, phys, Q, weights, scale, m, l = inputs
    d = pool.shape[2]
    want, tol = weights.double().clone().view(-1), torch.zeros(weights.numel(), dtype=torch.float64)
    for b, rows in enumerate(phys):
        w, e = accumulate_oracle(Q[b], pool.view(-1, d)[rows], m[b], l[b], scale, causal)
        want[rows] += w
        tol[rows] = e + 2.0 ** -23 * want[rows].abs()
    diff = (got.double().view(-1) - want).abs()
    assert torch.isfinite(got).all()
    assert (diff <= tol).all(), f"worst {float((diff - tol).max()):.3e} over the bound, error {float(diff.max()):.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,Sq,d,page,dtype,causal",
                         [c + (True,) for c in ACC_CASES] + [c + (False,) for c in ACC_CASES if c[2] > 1])
def test_accumulate_matches_the_definition(cuda, lens, H, Sq, d, page, dtype, causal):
    import flashdmla as F
    inp = acc_inputs(lens, H, Sq, d, page, dtype, causal)
    pool, table, phys, Q, weights, scale, m, l = inp
    w = weights.to(cuda)
    args = [t.to(cuda) for t in (pool, table)] + [torch.tensor(lens, dtype=torch.int32, device=cuda)]
    out = F.accumulate_weights(Q.to(cuda), *args, m.to(cuda), l.to(cuda), w, scale, causal)
    assert out is w and F.device_error_flag() == 0
    check_accumulated(w.cpu(), inp, causal)
    if Sq == 1:                                              # the three-dimensional form, strided inputs
        w2 = weights.to(cuda)
        q2 = Q[:, :, 0].to(cuda).transpose(0, 1).contiguous().transpose(0, 1)
        F.accumulate_weights(q2, *args, m[:, :, 0].to(cuda), l[:, :, 0].to(cuda), w2, scale)
        assert torch.equal(w, w2)


@pytest.mark.gpu
def test_accumulate_on_cuda_cores_agrees(cuda):
    import flashdmla as F
    lens, H = [300, 65], 48
    inp = acc_inputs(lens, H, 1, 576, 64, torch.bfloat16, True)
    pool, table, phys, Q, weights, scale, m, l = inp
    w = weights.to(cuda)
    F.set_backend(F.BACKEND_PORTABLE)
    try:
        F.accumulate_weights(Q.to(cuda), pool.to(cuda), table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda),
                             m.to(cuda), l.to(cuda), w, scale)
        assert F.last_kernel() == "portable"
    finally:
        F.set_backend(F.BACKEND_AUTO)
    check_accumulated(w.cpu(), inp, True)


@pytest.mark.gpu
def test_accumulate_reports_bad_pages_and_leaves_other_rows_alone(cuda):
    import flashdmla as F
    lens = [200, 64]
    pool, table, phys, Q, weights, scale, m, l = acc_inputs(lens, 16, 1, 576, 64, torch.bfloat16, True)
    bad = table.clone()
    bad[0, 1] = pool.shape[0]
    bad[0, 2] = -1
    w = weights.to(cuda)
    F.accumulate_weights(Q.to(cuda), pool.to(cuda), bad.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), m.to(cuda), l.to(cuda), w, scale)
    assert F.device_error_flag(reset=True) == 4
    touched = torch.zeros(weights.numel(), dtype=torch.bool)
    touched[phys[0][:64]] = touched[phys[0][192:]] = touched[phys[1]] = True
    w = w.cpu().view(-1)
    assert torch.equal(w[~touched], weights.view(-1)[~touched]) and (w[touched] > weights.view(-1)[touched]).all()


@pytest.mark.gpu
def test_accumulate_refusals(cuda):
    import flashdmla as F
    lens = [100]
    pool, table, phys, Q, weights, scale, m, l = acc_inputs(lens, 4, 1, 64, 64, torch.bfloat16, True)
    ok = [t.to(cuda) for t in (Q, pool, table, torch.tensor(lens, dtype=torch.int32), m, l, weights)]

    def call(i, t):
        a = list(ok)
        a[i] = t
        with pytest.raises(F.FlashDMLAError):
            F.accumulate_weights(*a)
    call(0, ok[0].float())
    call(0, ok[0][..., :32])
    call(0, ok[0][0])
    call(2, ok[2].long())
    call(3, ok[3].expand(2))
    call(4, ok[4].double())
    call(5, ok[5][:, :2])
    call(6, ok[6].half())
    call(6, ok[6].t())
    call(6, ok[6].cpu())


# -------------------------------------------------------------------------------------------------------- in the cache
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dq,dv,ps", [(torch.bfloat16, 576, 512, 64), (torch.float32, 48, 32, 8)])
def test_cache_tracks_weights_and_evicts(cuda, dtype, dq, dv, ps):
    """Decode steps with a bound on the rows: lengths, positions, weights and outputs follow a host-side restatement."""
    from flashdmla import FlashDMLAError
    from flashdmla.cache import PagedLatentCache
    g = torch.Generator().manual_seed(4)
    H, keep, recent, scale = 16, 96, 8, 1 / math.sqrt(dq)
    c = PagedLatentCache(num_pages=200, page_size=ps, d_qk=dq, max_seqs=3, max_pages_per_seq=64, dtype=dtype, device=cuda, track_weights=True)
    slots = [c.new_sequence(), c.new_sequence()]
    rows = {s: torch.zeros(0, dq, dtype=dtype) for s in slots}
    wts = {s: np.zeros(0) for s in slots}
    pos = {s: np.zeros(0, dtype=np.int64) for s in slots}

    def add(ss, n):
        x = torch.randn(len(ss), n, dq, generator=g).to(dtype)
        c.append(ss, x.to(cuda))
        for i, s in enumerate(ss):
            p0 = int(pos[s].max()) + 1 if len(pos[s]) else 0
            rows[s], wts[s] = torch.cat((rows[s], x[i])), np.concatenate((wts[s], np.zeros(n)))
            pos[s] = np.concatenate((pos[s], np.arange(p0, p0 + n)))
    add(slots[:1], 110)
    add(slots[1:], 40)
    for step in range(6):
        add(slots, 1 + 9 * (step % 2))
        Q = torch.randn(2, H, dq, generator=g).to(dtype)
        O, m, l = c.decode(Q.to(cuda), slots, dv, scale)
        for i, s in enumerate(slots):
            k = rows[s].double()
            p = torch.softmax(Q[i].double() @ k.T * scale, dim=-1)
            want = p @ k[:, :dv]
            assert (O[i].cpu().double() - want).abs().max() < (2e-2 if dtype == torch.bfloat16 else 1e-4)
            wts[s] = wts[s] + p.sum(0).numpy()
        if step in (1, 4):
            w_dev = {s: c.row_state(s)[0].cpu().numpy() for s in slots}        # what the eviction ranks by
            kept = c.evict(slots, keep, recent).cpu()
            src = evict_oracle([w_dev[s] for s in slots], [pos[s] for s in slots], [len(pos[s]) for s in slots],
                               [c.position(s) for s in slots], keep, recent)
            for i, s in enumerate(slots):
                assert kept[i, :len(src[i])].tolist() == src[i] and (kept[i, len(src[i]):] == -1).all()
                rows[s], wts[s], pos[s] = rows[s][src[i]], wts[s][src[i]], pos[s][src[i]]
        for s in slots:
            w, p = c.row_state(s)
            assert c.length(s) == len(pos[s]) and len(c.pages_of(s)) == -(-c.length(s) // ps)
            assert p.cpu().tolist() == pos[s].tolist()
            # m and l come from the attention kernel, which is held to 1e-3 (m: of max(1, |m|), and |m| < 5 here)
            assert np.allclose(w.cpu().numpy(), wts[s], rtol=6e-3, atol=1e-6)
    assert len(set(c.pages_of(slots[0]) + c.pages_of(slots[1]))) + c.free_pages == 200
    with pytest.raises(FlashDMLAError):
        c.evict([slots[0], slots[0]], keep)
    with pytest.raises(FlashDMLAError):
        c.decode(Q.to(cuda), slots, dv, scale, kv_end=10)
    plain = PagedLatentCache(num_pages=4, page_size=ps, d_qk=dq, max_seqs=1, max_pages_per_seq=2, dtype=dtype, device=cuda)
    with pytest.raises(FlashDMLAError):
        plain.evict([plain.new_sequence()], 4)


@pytest.mark.gpu
def test_block_step_with_bounded_cache_and_few_token_moe(cuda):
    """The operators together as one decode step: MLA over a cache that is cut to a bound, then the MoE layer; the rotary
    position goes on counting after an eviction."""
    from flashdmla import AbsorbedMLA, MoEFFN, PagedLatentCache
    d = 256
    mla = AbsorbedMLA(d, n_heads=8, device=cuda, seed=2)
    ffn = MoEFFN(d_model=d, d_ff=128, n_experts=8, top_k=2, device=cuda, seed=3)
    c = PagedLatentCache(num_pages=16, page_size=64, d_qk=576, max_seqs=2, max_pages_per_seq=4, device=cuda, track_weights=True)
    g = torch.Generator().manual_seed(8)
    slots = [c.new_sequence(), c.new_sequence()]
    h0 = (torch.randn(2, 100, d, generator=g)).to(torch.bfloat16).to(cuda)
    pos0 = torch.arange(100, device=cuda).expand(2, 100)
    c.append(slots, mla.cache_rows(h0, pos0))
    for step in range(4):
        h = torch.randn(2, d, generator=g).to(torch.bfloat16).to(cuda)
        o = mla.decode(c, slots, h)
        for i, s in enumerate(slots):
            held = c.gather([s], c.length(s))[0]
            want = mla.reference_decode(held, h[i], c.position(s) - 1)
            # bf16 attention against an fp32 restatement with other rounding points: as the block's own test
            assert (o[i].float() - want).norm() <= 2e-2 * want.norm()
        y = ffn.forward_few(o)
        assert y.shape == o.shape and torch.isfinite(y.float()).all()
        c.evict(slots, keep=90, recent=10)
        assert all(c.length(s) == 90 and c.position(s) == 101 + step for s in slots)
        assert all(101 + step - 1 in c.row_state(s)[1].tolist() for s in slots)     # the newest row is still there


# ------------------------------------------------------------------------------------------ pointers, streams, far pages
@pytest.mark.gpu
@pytest.mark.parametrize("d,shift", [(6, 1), (6, 2), (64, 1), (64, 2), (64, 8)])
def test_pools_that_start_at_odd_addresses(cuda, d, shift):
    """A pool (and Q) that is a view `shift` elements into a larger buffer: wide copies and bulk copies may not be used."""
    import flashdmla as F
    lens, keep = [150, 70, 10], 60
    case = evict_case(lens, keep, 9, 64, d, torch.bfloat16, "random", 21)
    pool, weights, positions, table, phys, nxt = case

    def view(t):
        buf = torch.zeros(t.numel() + 32, dtype=t.dtype, device=cuda)
        v = buf[shift:shift + t.numel()].view(t.shape)
        v.copy_(t)
        return v
    dlens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    # accumulate first, on clean rows
    g = torch.Generator().manual_seed(2)
    Q = torch.randn(len(lens), 4, 1, d, generator=g).to(torch.bfloat16)
    scale = 1.0 / math.sqrt(d)
    st = [stats(Q[b], pool.view(-1, d)[r], scale) for b, r in enumerate(phys)]
    m, l = torch.stack([s[0] for s in st]), torch.stack([s[1] for s in st])
    w = weights.to(cuda)
    F.accumulate_weights(view(Q), view(pool), table.to(cuda), dlens, m.to(cuda), l.to(cuda), w, scale)
    check_accumulated(w.cpu(), (pool, table, phys, Q, weights, scale, m, l), True)
    dp, dw, dpos = view(pool), weights.to(cuda), positions.to(cuda)
    kept, new = F.cache_evict(dp, dw, dpos, table.to(cuda), dlens, torch.tensor(nxt, dtype=torch.int32, device=cuda), keep, 9)
    check_evicted((dp.cpu(), dw.cpu(), dpos.cpu(), kept.cpu(), new.cpu()), case, lens, keep, 9)
    assert F.device_error_flag() == 0


@pytest.mark.gpu
def test_pages_behind_two_to_the_31_elements(cuda):
    """Pages whose first element lies beyond 2^31 elements (4 GB) of the pool."""
    import flashdmla as F
    g = torch.Generator().manual_seed(6)
    lens, d, H, keep = [200, 321], 576, 16, 130
    small, table, phys = paged(lens, 64, d, torch.bfloat16, g)
    N = 60000
    far = torch.randperm(1000, generator=g)[: small.shape[0]].sort().values + (N - 1000)
    pool = torch.empty(N, 64, d, dtype=torch.bfloat16, device=cuda)
    pool[far.to(cuda)] = small.to(cuda)
    ftable = far[table.long()].to(torch.int32)
    Q = torch.randn(2, H, 1, d, generator=g).to(torch.bfloat16)
    scale = 1 / math.sqrt(d)
    st = [stats(Q[b], small.view(-1, d)[r], scale) for b, r in enumerate(phys)]
    m, l = torch.stack([s[0] for s in st]), torch.stack([s[1] for s in st])
    weights = torch.randn(small.shape[:2], generator=g).exp()
    big_w = torch.zeros(N, 64, device=cuda)
    big_w[far.to(cuda)] = weights.to(cuda)
    dlens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    F.accumulate_weights(Q.to(cuda), pool, ftable.to(cuda), dlens, m.to(cuda), l.to(cuda), big_w, scale)
    check_accumulated(big_w[far.to(cuda)].cpu(), (small, table, phys, Q, weights, scale, m, l), True)
    positions = torch.zeros(small.shape[:2], dtype=torch.int32)
    case = (small, weights, positions, table, phys, [1000, 1000])
    big_w[far.to(cuda)] = weights.to(cuda)
    big_p = torch.zeros(N, 64, dtype=torch.int32, device=cuda)
    kept, new = F.cache_evict(pool, big_w, big_p, ftable.to(cuda), dlens, torch.full((2,), 1000, dtype=torch.int32, device=cuda), keep)
    check_evicted((pool[far.to(cuda)].cpu(), big_w[far.to(cuda)].cpu(), big_p[far.to(cuda)].cpu(), kept.cpu(), new.cpu()), case, lens, keep, 0)
    assert F.device_error_flag() == 0


@pytest.mark.gpu
def test_accumulate_shared_pages_streams_and_graph(cuda):
    """Two sequences on the same pages add up; calls on two streams do not disturb each other; a captured call replays."""
    import flashdmla as F
    lens, H, d = [300, 300], 32, 576
    pool, table, phys, Q, weights, scale, m, l = acc_inputs(lens, H, 1, d, 64, torch.bfloat16, True)
    table[1] = table[0]
    st = [stats(Q[b], pool.view(-1, d)[phys[0]], scale) for b in range(2)]
    m, l = torch.stack([s[0] for s in st]), torch.stack([s[1] for s in st])
    want, tol = weights.double().clone().view(-1), torch.zeros(weights.numel(), dtype=torch.float64)
    for b in range(2):
        w, e = accumulate_oracle(Q[b], pool.view(-1, d)[phys[0]], m[b], l[b], scale)
        want[phys[0]] += w
        tol[phys[0]] += e
    tol += 2 * 2.0 ** -23 * want.abs()
    args = [t.to(cuda) for t in (Q, pool, table, torch.tensor(lens, dtype=torch.int32), m, l)]
    bufs = [weights.to(cuda) for _ in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=cuda) for _ in range(2)]
    for i, b in enumerate(bufs):
        with torch.cuda.stream(streams[i % 2]):
            F.accumulate_weights(*args, b, scale)
    torch.cuda.synchronize()
    for b in bufs:
        assert ((b.cpu().double().view(-1) - want).abs() <= tol).all()
    w = weights.to(cuda)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        F.accumulate_weights(*args, w, scale)
    for _ in range(2):
        w.copy_(weights)
        g.replay()
        torch.cuda.synchronize()
        assert ((w.cpu().double().view(-1) - want).abs() <= tol).all()


@pytest.mark.gpu
def test_reserved_rows_start_without_weight(cuda):
    """Pages handed on to another sequence do not carry over weights or positions, however their rows are written."""
    from flashdmla import PagedLatentCache
    c = PagedLatentCache(num_pages=4, page_size=64, d_qk=64, max_seqs=2, max_pages_per_seq=4, device=cuda, track_weights=True)
    a = c.new_sequence()
    c.append([a], torch.randn(1, 200, 64, device=cuda).bfloat16())
    c.decode(torch.randn(1, 4, 64, device=cuda).bfloat16(), [a], 64)
    assert (c.row_state(a)[0] > 0).all() and c.row_state(a)[1].tolist() == list(range(200))
    c.free_sequence(a)
    b = c.new_sequence()
    c.reserve([b], 130)
    w, p = c.row_state(b)
    assert (w == 0).all() and p.tolist() == list(range(130))
    assert c.evict([b], 100).tolist() == [list(range(100))]               # all weights equal: the lower rows stay
    c.reserve([b], 1)
    assert c.row_state(b)[1].tolist() == list(range(100)) + [130]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,Sq,d,page,dtype,causal", [
    ([700, 64, 0], 16, 1, 576, 64, torch.bfloat16, True),     # the query rows of a step are resident
    ([700, 64, 0], 64, 1, 576, 64, torch.bfloat16, True),
    ([900, 300], 8, 5, 64, 64, torch.bfloat16, False),
    ([1100, 500], 16, 40, 192, 64, torch.bfloat16, True),     # the query rows stream past
    ([300, 40], 5, 3, 24, 16, torch.float32, True),           # CUDA cores
])
def test_query_rows_with_l_zero_add_nothing_whatever_they_hold(cuda, lens, H, Sq, d, page, dtype, causal):
    """The rows of a padded batch: l = 0, and a query that is NaN, infinite, or large enough to overflow the score."""
    import flashdmla as F
    pool, table, phys, Q, weights, scale, m, l = acc_inputs(lens, H, Sq, d, page, dtype, causal)
    dirty, m_dirty, l = Q.clone(), m.clone(), l.clone()
    R = H * Sq
    for b in range(len(lens)):
        for r, v in ((0, float("nan")), (R // 2, float("inf")), (R - 1, 3e38)):
            dirty[b].view(R, d)[r] = v
            m_dirty[b].view(R)[r] = v
            l[b].view(R)[r] = 0.0
    w = weights.to(cuda)
    F.accumulate_weights(*[t.to(cuda) for t in (dirty, pool, table, torch.tensor(lens, dtype=torch.int32), m_dirty, l)], w, scale, causal)
    check_accumulated(w.cpu(), (pool, table, phys, Q, weights, scale, m, l), causal)
    assert F.device_error_flag() == 0


# lens, table rows beyond the longest sequence, H, Sq, d, causal: what a pair of CTAs (74 of them) has to do several times over.
# Counts of tiles of 256 keys below are those of the lengths.
MANY_TILES = [
    ("resident queries, 294 tiles", [(97 * i) % 2501 for i in range(60)] + [0, 256, 257], 0, 16, 1, 64, True),
    ("resident queries, masked", [(97 * i) % 2501 for i in range(60)], 0, 16, 4, 64, True),
    ("resident queries, nine chunks, runs across sequences", [(331 * i) % 1801 for i in range(40)], 0, 32, 1, 576, True),
    ("streamed queries, 3 splits of 5 row tiles", [(137 * i) % 1301 for i in range(30)], 0, 28, 40, 64, True),
    ("streamed queries, not causal", [(137 * i) % 1301 for i in range(30)], 0, 28, 40, 64, False),
    ("streamed queries, one split", [(97 * i) % 2501 for i in range(46)], 0, 10, 33, 64, True),
    ("streamed queries, one split, not causal", [(97 * i) % 2501 for i in range(46)], 0, 10, 33, 64, False),
    ("streamed queries, nine chunks, several row tiles an item", [(137 * i) % 1301 for i in range(34)], 0, 20, 41, 576, True),
    ("streamed queries, row tiles that see nothing of an item", [(231 * i) % 1901 for i in range(30)], 0, 2, 700, 64, True),
    ("streamed queries, a table far wider than the lengths", [700, 0, 260, 1], 16384, 24, 60, 128, True),
    ("resident queries, a table far wider than the lengths", [700, 0, 260, 1], 16384, 64, 1, 128, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,wider,H,Sq,d,causal", [c[1:] for c in MANY_TILES], ids=[c[0] for c in MANY_TILES])
def test_accumulate_with_several_tiles_per_pair(cuda, lens, wider, H, Sq, d, causal):
    """Reuse of the resident operand, of both accumulators and of the row statistics, runs that cross sequences, sums over
    several tiles of query rows, with and without partial sums."""
    import flashdmla as F
    inp = acc_inputs(lens, H, Sq, d, 64, torch.bfloat16, causal)
    pool, table, phys, Q, weights, scale, m, l = inp
    wide = torch.full((len(lens), table.shape[1] + wider // 64), 10 ** 9, dtype=torch.int32)      # no page of the rest is looked at
    for b, n in enumerate(lens):
        wide[b, :(n + 63) // 64] = table[b, :(n + 63) // 64]
    w = weights.to(cuda)
    args = [t.to(cuda) for t in (Q, pool, wide, torch.tensor(lens, dtype=torch.int32), m, l)]
    F.accumulate_weights(*args, w, scale, causal)
    assert F.last_kernel() == "tcgen05" and F.device_error_flag() == 0
    check_accumulated(w.cpu(), inp, causal)
    w2 = weights.to(cuda)
    F.accumulate_weights(*args, w2, scale, causal)
    assert torch.equal(w, w2)


# ------------------------------------------------------------------------------------------------ after a time-out
def test_error_flag_takes_only_codes_of_waits():
    from flashdmla import _lib
    for code in (0, 4, 31, 40, 45, 50, 54, -1):
        assert _lib.lib().fdmla_set_device_error_flag(code) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("lens,H,Sq", [([500, 130, 7], 8, 33), ([300, 65], 16, 1)])
def test_weights_stay_as_they_were_after_a_time_out(cuda, lens, H, Sq):
    """While the flag of an earlier time-out stands a call adds nothing, not even what its scratch happened to hold; once it
    is cleared, calls work again."""
    import flashdmla as F
    from flashdmla import _lib
    L = _lib.lib()
    inp = acc_inputs(lens, H, Sq, 576, 64, torch.bfloat16, True)
    pool, table, phys, Q, weights, scale, m, l = inp
    nbytes = L.fdmla_cache_accumulate_workspace_bytes(len(lens), H, Sq, 576, 64, table.shape[1], _lib.BF16)
    assert (nbytes > 0) == (Sq > 1)                          # the window's query rows are split: partial sums in the scratch
    dev = [t.to(cuda) for t in (Q, pool, table, torch.tensor(lens, dtype=torch.int32), m, l)]
    w = weights.to(cuda)
    ws = torch.full((max(nbytes // 4, 1),), 1.0, device=cuda)

    def call():
        ws.fill_(1.0)
        rc = L.fdmla_cache_accumulate(*[t.data_ptr() for t in (*dev, w, ws)], nbytes, len(lens), H, Sq, 576, 64, table.shape[1],
                                      pool.shape[0], scale, 1, _lib.BF16, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
    try:
        assert L.fdmla_set_device_error_flag(52) == 0
        call()
        assert torch.equal(w.cpu(), weights)
        assert F.device_error_flag(reset=True) == 52
        call()
    finally:
        F.device_error_flag(reset=True)
    check_accumulated(w.cpu(), inp, True)
