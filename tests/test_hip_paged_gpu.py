"""The paged-cache operators on the GPU against plain implementations in 64 bits / plain integers (on the CPU).

Tolerances of the attention, from its arithmetic (u = 2^-24): a score is a dot product of dh terms and one scaling, its absolute error at most
(dh + 6) u S with S = scale * sum |q||k|, plus 4 u |score| for the change of base and the exponential; a probability's relative error is at most that plus
the running sums' (length + 8) u (numerator and denominator: twice), plus 2^-16 where a probability is handed to the matrix unit as two bf16 parts.  The
result's error is at most that factor times sum p |v|, plus half a step of the output type (eps / 2 relative; bf16 2^-8, fp32 2^-24)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

I32, BF, F32 = torch.int32, torch.bfloat16, torch.float32


def dev():
    return torch.device("cuda:0")


# ----------------------------------------------------------------------------- plan
class PlanOracle:
    """the same bookkeeping, request by request, on Python lists"""

    def __init__(self, N, M, s, pages):
        self.M, self.s, self.P = M, s, len(pages)
        self.free, self.head = list(pages), 0            # free pages in the order in which they are taken
        self.len = [0] * N
        self.rows = [[-1] * M for _ in range(N)]

    def plan(self, new, max_tokens):
        s, M = self.s, self.M
        length = [min(max(n, 0), M * s) for n in self.len]
        slots, positions, granted, cu = [-1] * max_tokens, [0] * max_tokens, [], [0]
        end = used = 0                                    # used: pages wanted so far, by accepted rows and by the ones the pool refused
        taken, back = 0, []
        for i, n in enumerate(new):
            start, end = end, end + max(n, 0)
            cu.append(min(end, max_tokens))
            have = -(-length[i] // s)
            if n < 0:
                back += self.rows[i][:have]
                self.rows[i] = [-1] * M
                self.len[i] = 0
                granted.append(0)
                continue
            fits = n > 0 and length[i] + n <= M * s and end <= max_tokens
            want = -(-(length[i] + n) // s) - have if fits else 0
            used += want
            if not fits or (want and used > len(self.free)):
                granted.append(0)
                self.len[i] = length[i]
                continue
            self.rows[i][have:have + want] = self.free[used - want:used]
            taken += want
            for j in range(n):
                page = self.rows[i][(length[i] + j) // s]
                positions[start + j] = length[i] + j
                slots[start + j] = page * s + (length[i] + j) % s if 0 <= page < self.P else -1
            self.len[i] = length[i] + n
            granted.append(n)
        self.head = (self.head + taken) % self.P
        self.free = self.free[taken:] + back
        return slots, positions, cu, granted


def same_state(o, lengths, table, free, ring):
    assert lengths.tolist() == o.len
    assert table.tolist() == o.rows
    head, count = ring.tolist()
    assert (head, count) == (o.head, len(o.free))
    assert [free.tolist()[(head + k) % o.P] for k in range(count)] == o.free


@pytest.mark.parametrize("N,M,s,P,steps,most", [
    (1, 1, 16, 1, 6, 20), (3, 4, 16, 9, 40, 30), (64, 9, 16, 300, 30, 40), (7, 130, 1, 500, 20, 90), (130, 33, 32, 2000, 12, 700),
    (1023, 3, 16, 1500, 6, 30), (1024, 3, 16, 1500, 6, 30), (2500, 5, 64, 4000, 6, 200)])
def test_plan_follows_the_oracle_over_many_steps(N, M, s, P, steps, most):
    from vilmedic_amd import ops
    g = torch.Generator().manual_seed(N * 31 + M)
    pages = torch.randperm(P, generator=g).to(I32)
    o = PlanOracle(N, M, s, pages.tolist())
    lengths, table = torch.zeros(N, dtype=I32, device=dev()), torch.full((N, M + 3), -1, dtype=I32, device=dev())[:, :M]
    free, ring = pages.to(dev()), torch.tensor([0, P], dtype=I32, device=dev())
    for step in range(steps):
        new = torch.randint(1, most + 1, (N,), generator=g)
        pick = torch.rand(N, generator=g)
        new = torch.where(pick < 0.25, torch.full_like(new, -1), torch.where(pick < 0.5, torch.zeros_like(new), torch.where(pick < 0.75, torch.ones_like(new), new)))
        total = int(new.clamp(min=0).sum())
        cut = [total, total + 5, max(0, total - 7), total // 2, 0][step % 5]         # exact, roomy, and too small for the last rows
        got = ops.paged_plan(lengths, new.to(I32).to(dev()), table, free, ring, s, cut)
        want = o.plan(new.tolist(), cut)
        assert [t.dtype for t in got] == [torch.int64, torch.int64, I32, I32]
        for name, a, b in zip(("slots", "positions", "cu_tokens", "granted"), got, want):
            assert a.tolist() == b, (step, name)
        same_state(o, lengths, table, free, ring)


def test_plan_admits_long_prompts_over_many_workgroups():
    from vilmedic_amd import ops
    N, M, s = 40, 256, 32
    g = torch.Generator().manual_seed(5)
    new = torch.randint(1, M * s + 1, (N,), generator=g)
    P = int(((new + s - 1) // s).sum()) - 3                                          # the last rows do not all fit
    pages = torch.randperm(P, generator=g).to(I32)
    o = PlanOracle(N, M, s, pages.tolist())
    lengths, table = torch.zeros(N, dtype=I32, device=dev()), torch.full((N, M), -1, dtype=I32, device=dev())
    free, ring = pages.to(dev()), torch.tensor([0, P], dtype=I32, device=dev())
    total = int(new.sum())
    for step_new, cut in ((new, total + 100), (torch.full_like(new, -1), 0), (new.flip(0), total)):
        got = ops.paged_plan(lengths, step_new.to(I32).to(dev()), table, free, ring, s, cut)
        for a, b in zip(got, o.plan(step_new.tolist(), cut)):
            assert a.tolist() == b
        same_state(o, lengths, table, free, ring)


def test_plan_clamps_lengths_and_marks_pages_that_do_not_exist():
    from vilmedic_amd import ops
    lengths = torch.tensor([-5, 1000, 20, 17], dtype=I32, device=dev())
    table = torch.tensor([[-1, -1], [0, 1], [7, -1], [2, 99]], dtype=I32, device=dev())
    free, ring = torch.tensor([3, 4, 5, 6], dtype=I32, device=dev()), torch.tensor([3, 1], dtype=I32, device=dev())
    slots, positions, cu, granted = ops.paged_plan(lengths, torch.tensor([1, 1, 1, 1], dtype=I32, device=dev()), table, free, ring, 16, 4)
    assert granted.tolist() == [1, 0, 1, 1] and cu.tolist() == [0, 1, 2, 3, 4]       # row 1 is full; row 3's next token lies in page 99 of 4
    assert slots.tolist() == [-1, -1, -1, -1] and positions.tolist() == [0, 0, 20, 17]      # (the ring handed out page 6: of the pool's four, none either)
    assert lengths.tolist() == [1, 32, 21, 18] and table[0].tolist() == [6, -1] and ring.tolist() == [0, 0]


def test_plan_counts_far_beyond_everything_without_overflow():
    from vilmedic_amd import ops
    big = 2 ** 31 - 1
    o = PlanOracle(5, 4, 16, list(range(20)))
    new = [3, big, big, 5, big]
    lengths, table = torch.zeros(5, dtype=I32, device=dev()), torch.full((5, 4), -1, dtype=I32, device=dev())
    free, ring = torch.arange(20, dtype=I32, device=dev()), torch.tensor([0, 20], dtype=I32, device=dev())
    got = ops.paged_plan(lengths, torch.tensor(new, dtype=I32, device=dev()), table, free, ring, 16, 64)
    want = o.plan(new, 64)
    assert got[3].tolist() == want[3] == [3, 0, 0, 0, 0]                               # row 3's tokens lie behind max_tokens in the packed order
    for a, b in zip(got, want):
        assert a.tolist() == b
    same_state(o, lengths, table, free, ring)
    many = torch.full((3000,), big, dtype=I32, device=dev())
    lengths, table = torch.zeros(3000, dtype=I32, device=dev()), torch.full((3000, 1), -1, dtype=I32, device=dev())
    slots, _, cu, granted = ops.paged_plan(lengths, many, table, free, ring, 16, 7)
    assert not granted.any() and not lengths.any() and bool((slots == -1).all()) and cu.tolist() == [0] + [7] * 3000


@pytest.mark.parametrize("N,M", [(40, 8), (1500, 3)])
def test_plan_replayed_from_a_graph(N, M):
    """one launch, and two launches with scratch memory: every replay takes the step after the last one"""
    from vilmedic_amd import ops
    P = N * M
    o = PlanOracle(N, M, 16, list(range(P)))
    lengths, table = torch.zeros(N, dtype=I32, device=dev()), torch.full((N, M), -1, dtype=I32, device=dev())
    free, ring = torch.arange(P, dtype=I32, device=dev()), torch.tensor([0, P], dtype=I32, device=dev())
    new = torch.zeros(N, dtype=I32, device=dev())
    graph = torch.cuda.CUDAGraph()
    with ops.capture(graph):
        out = ops.paged_plan(lengths, new, table, free, ring, 16, 3 * N)
    g = torch.Generator().manual_seed(N)
    for step in range(8):
        n = torch.randint(-1, 4, (N,), generator=g)
        new.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, o.plan(n.tolist(), 3 * N)):
            assert a.tolist() == b, step
        same_state(o, lengths, table, free, ring)
        ops.paged_plan(lengths, torch.zeros_like(new), table, free, ring, 16, 0)      # an eager plan in between: nothing to do
        o.plan([0] * N, 0)


# ----------------------------------------------------------------------------- write
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,dh,s,skew", [(1, 1, 8, 16, 0), (5, 2, 40, 16, 0), (64, 12, 64, 16, 8), (33, 3, 96, 32, 1), (700, 8, 128, 64, 0), (9, 1, 256, 128, 3), (257, 2, 48, 16, 4)])
def test_write_puts_every_row_into_its_slot_and_nothing_else(dtype, T, H, dh, s, skew):
    """k, v are column slices of one projection output whose rows start ``skew`` elements off a 16-byte boundary"""
    from vilmedic_amd import ops
    g = torch.Generator().manual_seed(T)
    P = -(-T // s) + 2
    kv = torch.randn(T, 2 * H * dh + skew + 3, generator=g).to(dtype).to(dev())
    k, v = kv[:, skew:skew + H * dh].view(T, H, dh), kv[:, skew + H * dh:skew + 2 * H * dh].unflatten(1, (H, dh))
    pages = torch.randn(2, P, H, s, dh, generator=g).to(dtype).to(dev())
    want = pages.clone()
    slots = torch.randperm(P * s, generator=g)[:T].to(dev())
    off = torch.randperm(T, generator=g)[:T // 4]
    slots[off[::2]] = -1
    slots[off[1::2]] = P * s + 5                                                       # behind the pool: skipped like -1
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < P * s:
            want[0, slot // s, :, slot % s], want[1, slot // s, :, slot % s] = k[t], v[t]
    ops.paged_kv_write(k, v, pages[0], pages[1], slots)
    assert torch.equal(pages.view(torch.uint8), want.view(torch.uint8))


def test_write_takes_heads_in_any_stride():
    from vilmedic_amd import ops
    k = torch.randn(4, 6, 16, device=dev()).transpose(0, 1)                            # [6 tokens, 4 heads, 16]: heads outside
    v = torch.randn(1, 4, 16, device=dev()).expand(6, 4, 16)                           # one row for all tokens
    pages = torch.zeros(2, 2, 4, 16, 16, device=dev())
    slots = torch.tensor([3, 31, 0, 17, 16, 8], device=dev())
    ops.paged_kv_write(k, v, pages[0], pages[1], slots)
    for t, slot in enumerate(slots.tolist()):
        assert torch.equal(pages[0, slot // 16, :, slot % 16], k[t]) and torch.equal(pages[1, slot // 16, :, slot % 16], v[t])


# ----------------------------------------------------------------------------- attention
def attend_ref(q, k_pages, v_pages, table, lengths, scale):
    """-> (result, error bound without the output's rounding), both float64 on the CPU"""
    N, Hq, dh = q.shape
    P, H, s, _ = k_pages.shape
    u = 2.0 ** -24
    out, tol = torch.zeros(N, Hq, dh, dtype=torch.float64), torch.zeros(N, Hq, dh, dtype=torch.float64)
    for n in range(N):
        length = min(max(int(lengths[n]), 0), table.shape[1] * s)
        pages = table[n, :-(-length // s)].long()
        for h in range(H):
            alive = ((pages >= 0) & (pages < P))[:, None].expand(-1, s).reshape(-1)[:length]
            at = pages.clamp(0, P - 1)
            k, v = (c[at, h].double().reshape(-1, dh)[:length][alive] for c in (k_pages, v_pages))
            if k.shape[0] == 0:
                continue
            rows = slice(h * Hq // H, (h + 1) * Hq // H)
            qq = q[n, rows].double()
            sc, S = qq @ k.t() * scale, qq.abs() @ k.abs().t() * scale
            p = torch.softmax(sc, 1)
            # the error that a common shift of all scores causes cancels, the largest remaining one is twice the largest score error
            rel = 2 * ((dh + 6) * u * S.amax(1) + 4 * u * sc.abs().amax(1)) + 2 * (length + 8) * u + (2.0 ** -16 if q.dtype == BF else 0)
            out[n, rows] = p @ v
            tol[n, rows] = rel[:, None] * (p @ v.abs())
    return out, tol


def make_cache(dtype, H, dh, s, lens, *, spare=3, seed=0, M=None):
    """pages in a random order, every slot behind a row's length NaN, as are pages nobody owns"""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // s) for n in lens]
    M = M or max(1, max(need))
    P = sum(need) + spare
    order = torch.randperm(P, generator=g).to(I32)
    table = torch.full((len(lens), M), -1, dtype=I32)
    pages = torch.full((2, P, H, s, dh), float("nan"), dtype=dtype)
    at = 0
    for i, n in enumerate(lens):
        table[i, :need[i]] = order[at:at + need[i]]
        for c in range(need[i]):
            live = min(s, n - c * s)
            pages[:, order[at + c], :, :live] = torch.randn(2, H, live, dh, generator=g).to(dtype)
        at += need[i]
    return pages[0], pages[1], table, torch.tensor(lens, dtype=I32)


def check_attention(q, k, v, table, lengths, scale=None, got=None):
    from vilmedic_amd import ops
    if got is None:
        got = ops.paged_attention(*(t.to(dev()) for t in (q, k, v, table, lengths)), **({} if scale is None else {"scale": scale}))
    want, tol = attend_ref(q, k, v, table, lengths, q.shape[2] ** -0.5 if scale is None else scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    err = (got.double().cpu() - want).abs()
    tol = tol * 1.01 + torch.finfo(q.dtype).eps / 2 * (want.abs() + tol) + 1e-30
    assert bool((err <= tol).all()), (err - tol).max()


SHAPES = [  # N, Hq, H, dh, page, lengths
    (1, 1, 1, 8, 16, [1]), (2, 1, 1, 64, 16, [0, 5]), (4, 12, 12, 64, 16, [1, 15, 16, 17]), (5, 8, 2, 128, 16, [31, 32, 33, 63, 65]),
    (3, 16, 1, 64, 16, [128, 129, 200]), (2, 20, 1, 32, 32, [77, 300]), (2, 32, 1, 128, 16, [100, 1]), (3, 6, 2, 48, 16, [0, 47, 511]), (2, 10, 2, 96, 64, [640, 1000]),
    (2, 4, 4, 40, 16, [90, 91]), (2, 6, 3, 80, 32, [256, 257]), (3, 4, 1, 256, 16, [5, 64, 700]), (2, 2, 1, 160, 128, [129, 1]), (1, 8, 8, 128, 256, [3000]), (2, 7, 1, 72, 16, [1025, 4]), (2, 16, 1, 256, 16, [33, 400]), (1, 33, 1, 256, 32, [90]),
    (2, 4, 2, 64, 4096, [4097, 5000])]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("N,Hq,H,dh,s,lens", SHAPES)
def test_attention(dtype, N, Hq, H, dh, s, lens):
    k, v, table, lengths = make_cache(dtype, H, dh, s, lens, seed=dh)
    q = (1.5 * torch.randn(N, Hq, dh, generator=torch.Generator().manual_seed(1))).to(dtype)
    check_attention(q, k, v, table, lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens", [[20011], [9001, 0, 3, 16385]])
def test_attention_over_long_histories(dtype, lens):
    k, v, table, lengths = make_cache(dtype, 2, 64, 16, lens, seed=7)
    q = torch.randn(len(lens), 8, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    check_attention(q, k, v, table, lengths)
    check_attention(q * 8, k, v, table, lengths, scale=0.3)                            # sharp distributions


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_with_a_wide_table_of_short_rows_and_many_rows(dtype):
    lens = [(37 * i) % 90 for i in range(300)]
    k, v, table, lengths = make_cache(dtype, 2, 64, 16, lens, seed=3, M=400)
    q = torch.randn(300, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    check_attention(q, k, v, table, lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,H,dh,M", [(2, 2, 64, 8), (6, 2, 32, 8), (4, 2, 128, 100), (34, 1, 40, 8), (2, 2, 200, 8)])
def test_attention_of_so_many_rows_that_one_wave_serves_each(dtype, Hq, H, dh, M):
    N = 1600 if H == 2 else 1100                       # (34 query heads of one key head: three blocks of up to 16)
    lens = [(i * 53) % 129 for i in range(N)]
    if M == 100:
        lens[7], lens[900] = 1600, 1111
    k, v, table, lengths = make_cache(dtype, H, dh, 16, lens, seed=dh, M=M)
    q = torch.randn(N, Hq, dh, generator=torch.Generator().manual_seed(2)).to(dtype)
    check_attention(q, k, v, table, lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_strides_of_q_and_table(dtype):
    from vilmedic_amd import ops
    lens = [40, 3, 129]
    k, v, table, lengths = make_cache(dtype, 2, 64, 16, lens)
    wide = torch.randn(3, 3 * 8 * 64 + 5, generator=torch.Generator().manual_seed(4)).to(dtype)
    q = wide[:, 3:3 + 8 * 64].view(3, 8, 64)                                           # an unaligned column slice of a projection output
    t2 = torch.full((3, table.shape[1] + 5), 12345, dtype=I32)
    t2[:, 2:2 + table.shape[1]] = table
    t2 = t2[:, 2:2 + table.shape[1]]
    kd, vd = k.to(dev()), v.to(dev())
    wd, td = wide.to(dev()), torch.full((3, table.shape[1] + 5), 12345, dtype=I32, device=dev())
    td[:, 2:2 + table.shape[1]] = table.to(dev())
    qd = wd[:, 3:3 + 8 * 64].view(3, 8, 64)
    got = ops.paged_attention(qd, kd, vd, td[:, 2:2 + table.shape[1]], lengths.to(dev()))
    check_attention(q, k, v, t2, lengths, got=got)
    hq = qd.transpose(0, 1).contiguous().transpose(0, 1)                               # heads outermost
    assert torch.equal(ops.paged_attention(hq, kd, vd, td[:, 2:2 + table.shape[1]], lengths.to(dev())), got)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_leaves_out_pages_that_do_not_exist_and_clamps_lengths(dtype):
    k, v, table, lengths = make_cache(dtype, 1, 64, 16, [100, 64, 48, 32, 64], seed=9)
    P = k.shape[0]
    table[0, 2] = -1
    table[0, 5] = P
    table[1, 0] = 2 ** 31 - 1
    table[2, :] = -2 ** 31                                                             # nothing left: zeros
    lengths[3] = -7
    lengths[4] = 10 ** 9                                                               # clamped to the table's width: 7 pages, of which 4 exist
    q = torch.randn(5, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    check_attention(q, k, v, table, lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_rows_may_share_pages(dtype):
    k, v, table, lengths = make_cache(dtype, 2, 64, 16, [100, 1, 1], seed=9)
    table[1], table[2] = table[0], table[0]
    lengths[1], lengths[2] = 64, 100
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    check_attention(q, k, v, table, lengths)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_propagates_nan_and_inf_of_live_keys_only(dtype):
    from vilmedic_amd import ops
    k, v, table, lengths = make_cache(dtype, 1, 64, 16, [30, 30, 30], seed=9)
    k[table[1, 0], 0, 3, 5] = float("nan")
    v[table[2, 1], 0, 2, 7] = float("inf")
    q = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    got = ops.paged_attention(*(t.to(dev()) for t in (q, k, v, table, lengths))).cpu()
    assert bool(torch.isfinite(got[0]).all()) and bool(torch.isnan(got[1]).all())
    assert bool((got[2, :, 7] == float("inf")).all()) and bool(torch.isfinite(got[2, :, :7]).all()) and bool(torch.isfinite(got[2, :, 8:]).all())


@pytest.mark.parametrize("dh", [8, 40, 64, 72, 80, 96, 104, 160, 256])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_gives_a_key_of_score_minus_infinity_no_weight(dtype, dh):
    """an infinity in a key's last column, against a negative query column: the row is what it is without that key (exactly zero weight)"""
    lens = [1 + 20, 1 + 47, 1 + 700]
    k, v, table, lengths = make_cache(dtype, 2, dh, 16, lens, seed=dh)
    for n, length in enumerate(lens):
        k[table[n, (length - 1) // 16], :, (length - 1) % 16, -1] = float("inf")
    q = torch.randn(3, 6, dh, generator=torch.Generator().manual_seed(dh)).to(dtype)
    q[:, :, -1] = -q[:, :, -1].abs() - 0.5
    from vilmedic_amd import ops
    got = ops.paged_attention(*(t.to(dev()) for t in (q, k, v, table, lengths)))
    check_attention(q, k, v, table, lengths - 1, got=got)


@pytest.mark.parametrize("dh", list(range(8, 257, 8)))
@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_of_every_head_size(dtype, dh):
    """rows of one wave's tile, of several, and split over workgroups; pages that end inside a tile"""
    lens = [3, 0, 64, 161, 1200]
    k, v, table, lengths = make_cache(dtype, 2, dh, 16, lens, seed=dh)
    check_attention(torch.randn(5, 10, dh, generator=torch.Generator().manual_seed(dh)).to(dtype), k, v, table, lengths)


@pytest.mark.parametrize("dh", [72, 88, 120, 136, 192, 256])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_of_wide_heads_by_one_wave_each(dtype, dh):
    g = torch.Generator().manual_seed(dh)
    lens = torch.randint(0, 97, (1030,), generator=g).tolist()
    k, v, table, lengths = make_cache(dtype, 3, dh, 16, lens, seed=dh, M=6)
    check_attention(torch.randn(1030, 3, dh, generator=g).to(dtype), k, v, table, lengths)


def test_attention_reaches_beyond_32_bit_offsets():
    """a pool of 2.2e9 elements (4.5 GB each for K and V): pages at its very end"""
    from vilmedic_amd import ops
    H, s, dh = 8, 64, 128
    P = (2 ** 31 + 2 ** 27) // (H * s * dh)
    kp, vp = (torch.empty(P, H, s, dh, dtype=BF, device=dev()) for _ in range(2))
    lens = [200, 70]
    k, v, table, lengths = make_cache(BF, H, dh, s, lens, seed=5, spare=0)
    n = k.shape[0]
    far = torch.tensor([P - 1 - 2 * i for i in range(n)], dtype=I32)
    far_table = torch.where(table >= 0, far[table.clamp(min=0).long()], table)
    g = torch.Generator().manual_seed(8)
    q = torch.randn(2, 16, dh, generator=g).to(BF)
    # written through the slot map, one token at a time in packed order
    slots, ks, vs = [], [], []
    for i, length in enumerate(lens):
        for j in range(length):
            slots.append(int(far_table[i, j // s]) * s + j % s)
            ks.append(k[table[i, j // s], :, j % s])
            vs.append(v[table[i, j // s], :, j % s])
    kd, vd = torch.stack(ks).to(dev()), torch.stack(vs).to(dev())
    for i, page in enumerate(far_table[far_table >= 0].tolist()):
        kp[page], vp[page] = float("nan"), float("nan")
    ops.paged_kv_write(kd, vd, kp, vp, torch.tensor(slots, device=dev()))
    got = ops.paged_attention(q.to(dev()), kp, vp, far_table.to(dev()), lengths.to(dev()))
    check_attention(q, k, v, table, lengths, got=got)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_repeats_bit_for_bit_and_rows_do_not_depend_on_their_neighbours(dtype):
    from vilmedic_amd import ops
    lens = [500, 1, 0, 3000, 64, 65]
    k, v, table, lengths = (t.to(dev()) for t in make_cache(dtype, 2, 64, 16, lens, seed=4))
    q = torch.randn(len(lens), 8, 64, generator=torch.Generator().manual_seed(2)).to(dtype).to(dev())
    a = ops.paged_attention(q, k, v, table, lengths)
    for _ in range(5):
        assert torch.equal(ops.paged_attention(q, k, v, table, lengths), a)
    order = torch.tensor([3, 0, 5, 2, 1, 4], device=dev())
    assert torch.equal(ops.paged_attention(q[order], k, v, table[order], lengths[order]), a[order])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_on_two_streams_at_once(dtype):
    from vilmedic_amd import ops
    lens = [4000, 12, 2500]
    k, v, table, lengths = (t.to(dev()) for t in make_cache(dtype, 2, 64, 16, lens, seed=4))
    q = torch.randn(3, 8, 64, generator=torch.Generator().manual_seed(2)).to(dtype).to(dev())
    want, want2 = ops.paged_attention(q, k, v, table, lengths), ops.paged_attention(q * 2, k, v, table, lengths)
    torch.cuda.synchronize()
    q2 = q * 2
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(20):
        for st, x in zip(streams, (q, q2)):
            with torch.cuda.stream(st):
                outs.append(ops.paged_attention(x, k, v, table, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, [want, want2] * 20))


# ----------------------------------------------------------------------------- the run of them, as a decode step uses them
def decode_step(ops, st, x_q, x_kv):
    slots, pos, cu, granted = ops.paged_plan(st["lengths"], st["new"], st["table"], st["free"], st["ring"], st["page"], x_q.shape[0])
    H, dh = st["k"].shape[1], st["k"].shape[3]
    ops.paged_kv_write(x_kv[:, :H * dh].view(-1, H, dh), x_kv[:, H * dh:].view(-1, H, dh), st["k"], st["v"], slots)
    return ops.paged_attention(x_q, st["k"], st["v"], st["table"], st["lengths"]), slots, pos


def serving_state(N, H, dh, s, M, P, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return dict(page=s, lengths=torch.zeros(N, dtype=I32, device=dev()), new=torch.ones(N, dtype=I32, device=dev()),
                table=torch.full((N, M), -1, dtype=I32, device=dev()), free=torch.randperm(P, generator=g).to(I32).to(dev()),
                ring=torch.tensor([0, P], dtype=I32, device=dev()), k=torch.full((P, H, s, dh), float("nan"), dtype=dtype, device=dev()),
                v=torch.full((P, H, s, dh), float("nan"), dtype=dtype, device=dev()))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("graph", [False, True])
def test_admission_steps_and_release_against_a_dense_cache(dtype, graph):
    """prompts of different lengths, decode steps (eager, or one captured step replayed with the program's own work in between), a row that leaves and
    one that takes its place; every step against attention over the rows' own dense histories"""
    from vilmedic_amd import ops
    N, Hq, H, dh, s, M, P = 6, 4, 2, 64, 16, 8, 40
    st = serving_state(N, H, dh, s, M, P, dtype)
    g = torch.Generator().manual_seed(11)
    hist = [torch.zeros(0, 2, H, dh) for _ in range(N)]

    def admit(counts):
        new = torch.tensor(counts, dtype=I32)
        T = int(new.clamp(min=0).sum())
        slots, pos, cu, granted = ops.paged_plan(st["lengths"], new.to(dev()), st["table"], st["free"], st["ring"], s, T)
        assert granted.tolist() == [max(c, 0) for c in counts]
        kv = torch.randn(T, 2, H, dh, generator=g).to(dtype)
        kvd = kv.to(dev())
        ops.paged_kv_write(kvd[:, 0], kvd[:, 1], st["k"], st["v"], slots)
        for i, c in enumerate(counts):
            a, b = cu.tolist()[i], cu.tolist()[i + 1]
            hist[i] = torch.zeros(0, 2, H, dh) if c < 0 else torch.cat([hist[i], kv[a:b].float()])

    x_q, x_kv = torch.zeros(N, Hq, dh, dtype=dtype, device=dev()), torch.zeros(N, 2 * H * dh, dtype=dtype, device=dev())
    captured = {}

    def step():
        q, kv = torch.randn(N, Hq, dh, generator=g).to(dtype), torch.randn(N, 2 * H * dh, generator=g).to(dtype)
        x_q.copy_(q)
        x_kv.copy_(kv)
        if graph:
            captured["graph"].replay()
            out, slots, pos = captured["out"]
        else:
            out, slots, pos = decode_step(ops, st, x_q, x_kv)
        assert pos.tolist() == [h.shape[0] for h in hist]
        for i in range(N):
            hist[i] = torch.cat([hist[i], kv[i].float().view(1, 2, H, dh)])
        lens = [h.shape[0] for h in hist]
        assert st["lengths"].tolist() == lens
        L = max(lens)
        kd, vd = torch.zeros(N, H, L, dh), torch.zeros(N, H, L, dh)
        for i, h in enumerate(hist):
            kd[i, :, :lens[i]], vd[i, :, :lens[i]] = h[:, 0].transpose(0, 1), h[:, 1].transpose(0, 1)
        # a dense history is a paged one with one page per row (padded to a power of two)
        size = 1 << (L - 1).bit_length()
        kd, vd = (torch.nn.functional.pad(t, (0, 0, 0, size - L)).to(dtype) for t in (kd, vd))
        check_attention(q, kd, vd, torch.arange(N, dtype=I32)[:, None], torch.tensor(lens, dtype=I32), got=out)

    if graph:
        saved = {n: t.clone() for n, t in st.items() if torch.is_tensor(t)}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode_step(ops, st, x_q, x_kv)
        torch.cuda.current_stream().wait_stream(side)
        captured["graph"] = torch.cuda.CUDAGraph()
        with ops.capture(captured["graph"]):
            captured["out"] = decode_step(ops, st, x_q, x_kv)
        for n, t in saved.items():
            st[n].copy_(t)
    admit([5, 16, 1, 31, 47, 20])
    for _ in range(4):
        step()
        if graph:
            ops.paged_attention(x_q, st["k"], st["v"], st["table"], st["lengths"])     # the program's own eager work between replays
            torch.cuda.synchronize()
    admit([0, -1, 0, 0, -1, 0])
    admit([0, 70, 0, 0, 3, 0])
    for _ in range(15):
        step()
    admit([-1] * N)
    assert st["ring"].tolist()[1] == P and sorted(st["free"].tolist()) == list(range(P))


def test_two_captured_steps_replayed_in_turn_share_nothing():
    from vilmedic_amd import ops
    sides = []
    for seed, lens in ((1, [4000, 7]), (2, [33, 3500])):
        k, v, table, lengths = (t.to(dev()) for t in make_cache(BF, 2, 64, 16, lens, seed=seed))
        q = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(seed)).to(BF).to(dev())
        want = ops.paged_attention(q, k, v, table, lengths)
        graph = torch.cuda.CUDAGraph()
        with ops.capture(graph):
            out = ops.paged_attention(q, k, v, table, lengths)
        sides.append((graph, out, want, (q, k, v, table, lengths)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for (graph, out, want, _), stream in zip(sides, streams):
            out.zero_()
        torch.cuda.synchronize()
        for (graph, out, want, _), stream in zip(sides, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for graph, out, want, _ in sides:
            assert torch.equal(out, want)
