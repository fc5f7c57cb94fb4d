"""The operators between the simulator and a policy network, against plain implementations in 64 bits."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import policy_util as ref  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
DEV = "cuda:0"


@pytest.fixture(scope="module")
def policy():
    from multigrid_amd import policy
    return policy


def gen(seed):
    return torch.Generator(device="cpu").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g)


# ---- embedding -----------------------------------------------------------------------------------------------------------


def some_ids(g, n, sizes, dtype, outside=True):
    ids = torch.stack([torch.randint(0, r, (n,), generator=g) for r in sizes], -1)
    if outside and n > 3:
        bad = torch.rand((n, len(sizes)), generator=g) < 0.1
        far = torch.tensor(sizes) + (200 - max(sizes) if dtype == torch.uint8 and max(sizes) < 200 else 0)
        ids = torch.where(bad, far.expand_as(ids) if dtype == torch.uint8 else torch.where(ids % 2 == 0, -1 - ids, far + ids), ids)
        ids = ids.clamp(max=255) if dtype == torch.uint8 else ids
    return ids.to(dtype)


EMBED = [  # tokens, sizes of the fields, dim
    (1, (1,), 1), (1, (24,), 5), (98, (11, 6, 7), 32), (63, (11, 6, 7), 16), (257, (11, 6, 7), 7), (1000, (11, 6, 7), 130),
    (150001, (700,), 8), (70000, (11, 6, 7), 16), (140000, (11, 6, 7), 7), (131072, (30, 3), 24), (60000, (2, 3), 8), (63, (24,), 16), (64, (24,), 17), (127, (11, 6, 7), 40), (40000, (2, 3), 8), (70000, (7,), 9), (30000, (300, 2, 5000), 20), (5, (300,), 1), (64, (2, 3), 8), (65, (1, 1, 1, 1, 1, 1, 1, 1), 3), (333, (64,), 40), (333, (65,), 33), (1025, (997,), 264),
    (2049, (33, 200, 70), 24), (6000, (5000,), 9), (40, (131072,), 64), (3, (7,), 5000), (5000, (17,), 64), (20000, (11, 6, 7), 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,sizes,dim", EMBED)
def test_embed(policy, n, sizes, dim, dtype):
    for k, ids_type in enumerate((torch.uint8, torch.int32, torch.int64)):
        if ids_type == torch.uint8 and max(sizes) > 250:
            continue
        g = gen(1000 * n + dim + k)
        ids = some_ids(g, n, sizes, ids_type)
        table, grad = randn(g, sum(sizes), dim).to(dtype), randn(g, n, dim).to(dtype)
        w = table.to(DEV).requires_grad_()
        fields = sizes if len(sizes) > 1 else None
        at = (ids if fields else ids[:, 0]).to(DEV)
        out = policy.embed(at, w, fields=fields, scale=1.7)
        assert out.dtype == dtype and out.shape == (n, dim)
        ref.close(out, *ref.embed(ids, table, sizes, 1.7), dtype)
        dw, = torch.autograd.grad(out, w, grad.to(DEV))
        assert dw.dtype == dtype
        ref.close(dw, *ref.embed_grad(ids, grad, sizes, 1.7), dtype)
        again = policy.embed_grad(grad.to(DEV), at, sum(sizes), fields=fields, scale=1.7)
        assert torch.equal(again, dw), "the same call gave other bits"


@pytest.mark.parametrize("n", [3000, 20000])
@pytest.mark.parametrize("rows", [24, 64, 100, 5000])
@pytest.mark.parametrize("how", ["one row", "two rows", "frequent", "all outside"])
def test_embed_grad_of_few_and_frequent_rows(policy, n, rows, how):
    g = gen(n + rows)
    if how == "one row":
        ids = torch.full((n,), rows - 1)
    elif how == "two rows":
        ids = torch.where(torch.arange(n) < n // 3, 0, rows - 1)
    elif how == "frequent":
        ids = (torch.exp(torch.rand(n, generator=g) * math.log(rows)).long() - 1).clamp(0, rows - 1)
    else:
        ids = torch.where(torch.arange(n) % 2 == 0, -1, rows)
    for dtype in DTYPES:
        grad = randn(g, n, 72).to(dtype)
        dw = policy.embed_grad(grad.to(DEV), ids.to(DEV), rows)
        ref.close(dw, *ref.embed_grad(ids, grad, (rows,), 1.0), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows", [(100, 24), (6000, 24), (6000, 60), (100, 3000), (6000, 3000)])
def test_embed_grad_keeps_infinities_and_nan_to_their_rows(policy, n, rows, dtype):
    """A NaN or an infinity in the gradient of one token reaches the rows that this token reads and no others; in the
    gradient of a padded token it reaches nothing."""
    g = gen(n + rows)
    ids = torch.randint(3, rows, (n,), generator=g)
    grad = randn(g, n, 40).to(dtype)
    ids[n // 2], ids[n // 3], ids[n // 4], ids[n // 5], ids[1] = 0, 1, 1, -1, rows
    grad[n // 2, 3], grad[n // 3, 4], grad[n // 4, 4], grad[n // 5], grad[1] = math.nan, math.inf, -math.inf, math.nan, math.inf
    grad[n // 3, 7] = -math.inf
    dw = policy.embed_grad(grad.to(DEV), ids.to(DEV), rows)
    want, err = ref.embed_grad(ids, grad, (rows,), 1.0)
    assert np.isnan(want[0, 3]) and np.isnan(want[1, 4]) and want[1, 7] == -np.inf and np.isfinite(want[2:]).all()
    ref.close(dw, want, np.where(np.isfinite(err), err, 0.0), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows", [(64, 24), (5000, 24), (5000, 700)])
def test_embed_grad_of_small_numbers(policy, n, rows, dtype):
    """Gradients among a type's smallest normal and subnormal numbers are summed, not flushed."""
    g = gen(n)
    ids = torch.randint(0, rows, (n,), generator=g)
    tiny = torch.finfo(dtype).tiny if dtype == torch.float16 else 2.0 ** -100
    grad = (randn(g, n, 32) * tiny * 0.25).to(dtype)
    dw = policy.embed_grad(grad.to(DEV), ids.to(DEV), rows)
    ref.close(dw, *ref.embed_grad(ids, grad, (rows,), 1.0), dtype)


def test_embed_strides_shapes_and_streams(policy):
    g = gen(5)
    image = some_ids(g, 4 * 3 * 5 * 5, (11, 6, 7), torch.uint8, outside=False).view(4, 3, 5, 5, 3)
    big = randn(g, 24, 80).to(DEV)
    want, err = ref.embed(image, big[:, 8:72].cpu(), (11, 6, 7), 1.0)
    x = image.to(DEV)
    for table in (big[:, 8:72], big[:, 8:72].contiguous(), big.t().contiguous().t()[:, 8:72]):  # rows apart, adjacent, columns adjacent
        ref.close(policy.embed(x, table, fields=(11, 6, 7)).view(-1, 64), want, err, torch.float32)
    types = x[..., 0]  # every third byte
    got = policy.embed(types, big[:11])
    ref.close(got.reshape(-1, 80), *ref.embed(image[..., 0], big[:11].cpu(), (11,), 1.0), torch.float32)
    assert got.shape == (4, 3, 5, 5, 80)
    swapped = x.permute(1, 0, 2, 3, 4)
    assert torch.equal(policy.embed(swapped, big, fields=(11, 6, 7)), policy.embed(x, big, fields=(11, 6, 7)).permute(1, 0, 2, 3, 4))
    same = x[:1, :1, :1, :1].expand(2, 3, 4, 5, 3)  # one token for all
    assert torch.equal(policy.embed(same, big, fields=(11, 6, 7))[1, 2, 3, 4], policy.embed(x, big, fields=(11, 6, 7))[0, 0, 0, 0])
    grad = randn(g, 300, 2, 80).to(DEV)[:, 1, 4:36]
    expanded = randn(g, 32).to(DEV).expand(300, 32)  # the gradient of a sum: one row for all tokens
    transposed = randn(g, 32, 300).to(DEV).t()
    for d in (grad, expanded, transposed):
        ref.close(policy.embed_grad(d, x.view(-1, 3), 24, fields=(11, 6, 7)), *ref.embed_grad(image, d.cpu(), (11, 6, 7), 1.0), torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = policy.embed(x, big, fields=(11, 6, 7))
        b = policy.embed_grad(grad, x.view(-1, 3), 24, fields=(11, 6, 7))
    side.synchronize()
    assert torch.equal(a, policy.embed(x, big, fields=(11, 6, 7))) and torch.equal(b, policy.embed_grad(grad, x.view(-1, 3), 24, fields=(11, 6, 7)))


def test_embed_of_nothing(policy):
    table = torch.ones((5, 4), device=DEV, requires_grad=True)
    out = policy.embed(torch.empty((0, 3), dtype=torch.int64, device=DEV), table)
    assert out.shape == (0, 3, 4)
    out.sum().backward()
    assert torch.equal(table.grad, torch.zeros_like(table))
    one = policy.embed(torch.tensor(2, device=DEV), table)
    assert one.shape == (4,)


def test_embed_keeps_its_own_copy_of_the_ids(policy):
    """The simulator writes its images in place: a backward pass after the next step still belongs to the old image."""
    g = gen(9)
    ids = some_ids(g, 500, (11, 6, 7), torch.uint8, outside=False)
    table, grad = randn(g, 24, 16).to(DEV).requires_grad_(), randn(g, 500, 16)
    x = ids.to(DEV)
    out = policy.embed(x, table, fields=(11, 6, 7))
    x.zero_()
    dw, = torch.autograd.grad(out, table, grad.to(DEV))
    ref.close(dw, *ref.embed_grad(ids, grad, (11, 6, 7), 1.0), torch.float32)


@pytest.mark.parametrize("n,rows", [(40, 24), (3000, 24), (3000, 4000)])
def test_embed_gradient_against_differences(policy, n, rows):
    """out is linear in the table: <G, out(W + V) - out(W - V)> / 2 = <dW, V>, but for roundings of sums of n * 16 products."""
    g = gen(n)
    ids = torch.randint(0, rows, (n,), generator=g).to(DEV)
    w, v, up = (randn(g, *s).to(DEV) for s in ((rows, 16), (rows, 16), (n, 16)))
    w.requires_grad_()
    out = policy.embed(ids, w, scale=0.5)
    dw, = torch.autograd.grad(out, w, up)
    with torch.no_grad():
        diff = (up.double() * (policy.embed(ids, w + v, scale=0.5).double() - policy.embed(ids, w - v, scale=0.5).double())).sum() / 2
    size = float((up.double().abs() * policy.embed(ids, w.abs() + v.abs(), scale=0.5).detach().double()).sum())
    assert abs(float(diff) - float((dw.double() * v.double()).sum())) <= size * ref.U32 * (n + 8)


def test_embed_with_offsets_beyond_32_bits(policy):
    """The output and the gradient pass 2^32 bytes, and 2^31 elements: the tokens behind that point are right too."""
    n, dim = (1 << 21) + 5, 1032
    ids = torch.arange(n, device=DEV) % 7
    ids[n - 3:] = torch.tensor([8, 9, 8], device=DEV)
    table = torch.arange(10 * dim, device=DEV).view(10, dim).remainder(251).to(torch.bfloat16)
    out = policy.embed(ids, table)
    assert out.numel() > 1 << 31
    for at in (0, n // 2, n - 4, n - 3, n - 2, n - 1):
        assert torch.equal(out[at], table[ids[at]])
    out.zero_()
    out[n - 3:] = table[:3]
    dw = policy.embed_grad(out, ids, 10)
    assert torch.equal(dw[9], table[1]) and torch.equal(dw[8], (table[0].float() + table[2].float()).to(torch.bfloat16)) and not dw[:8].any()
    big_rows = (1 << 21) + 9
    wide = torch.zeros((big_rows, dim), dtype=torch.bfloat16, device=DEV)
    wide[big_rows - 1] = table[3]
    assert torch.equal(policy.embed(torch.tensor([big_rows - 1], device=DEV), wide)[0], table[3])
    dw = policy.embed_grad(table[4:6], torch.tensor([big_rows - 1, big_rows - 2], device=DEV), big_rows)
    assert torch.equal(dw[big_rows - 1], table[4]) and torch.equal(dw[big_rows - 2], table[5]) and not dw[:big_rows - 2].any()


def test_cell_embedding_is_the_one_hot_image_times_the_table(policy):
    from multigrid_amd import envs, layouts, views
    from multigrid_amd.batched import BatchedMultiGrid
    spec, make = envs.make_spec("MultiGrid-BlockedUnlockPickup-v0", num_agents=2, agent_view_size=7)
    sim = BatchedMultiGrid(spec, 33, device=0, one_hot=True)
    sim.upload_layouts(*layouts.make_pool(make, 8, seed0=3)[:3])
    out = sim.reset()
    table = torch.randint(-8, 9, (24, 32), generator=gen(1)).float().to(DEV)  # whole numbers: both sums are exact
    got = views.cell_embedding(out.image, table)
    assert got.shape == (33, 2, 7, 7, 32)
    assert torch.equal(got, out.onehot.float() @ table)
    sim.close()


# ---- adjustment ----------------------------------------------------------------------------------------------------------


ADJUST = [  # rows, tokens, history, mask
    (1, 1, 1, None), (1, 7, 0, "bool"), (3, 7, 5, "bits"), (1000, 7, 16, "bool"), (129, 32, 3, "bits"), (300, 8, 40, "bits"), (70, 9, 3, "bool"), (70, 16, 17, "bits"), (70, 17, 33, "bool"), (77, 33, 300, "bits"), (64, 63, 9, "bool"),
    (64, 64, 9, None), (65, 65, 70, "bits"), (9, 1000, 33, "bits"), (2, 4099, 1025, "bool"), (3, 8191, 40, "bits"), (2, 8192, 40, "bool"),
    (2, 8193, 3000, "bits"), (1, 40007, 512, "bits"), (300, 511, 2, None),
]


def adjust_args(seed, n, k, t, mask, history_type=torch.int64, shared=False):
    g = gen(seed)
    more = dict(repetition=(0.5 + torch.rand(n, generator=g)), presence=torch.rand(n, generator=g), frequency=0.3 * torch.rand(n, generator=g) - 0.1)
    rows = (1,) if shared else (n,)
    if t:
        h = torch.randint(-2, k + 2, rows + (t,), generator=g)
        h = h.clamp(0, 255) if history_type == torch.uint8 else h
        h[:, : t // 2] = h[:, :1].clone()  # one token many times
        more["history"] = h.to(history_type)[0] if shared else h.to(history_type)
        if not shared:
            more["lengths"] = torch.randint(-1, t + 2, (n,), generator=g).int()
    more["bias"] = randn(g, k) if shared or n < 3 else randn(g, n, k)
    if mask == "bool":
        m = torch.rand(rows + (k,), generator=g) < 0.7
        m[0] &= n < 3  # a row of nothing
        more["mask"] = m[0] if shared else m
    elif mask == "bits":
        m = torch.randint(-(1 << 31), 1 << 31, rows + ((k + 31) // 32,), generator=g)
        m[0] *= n < 3
        more["mask"] = (m[0] if shared else m).int()
    return more


def on_gpu(more):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in more.items()}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k,t,mask", ADJUST)
def test_adjust(policy, n, k, t, mask, dtype):
    for j, history_type in enumerate((torch.int64, torch.int32, torch.uint8)):
        for shared in (False, True):
            more = adjust_args(n * 31 + k + j, n, k, t, mask, history_type, shared)
            g = gen(k)
            x, up = (randn(g, n, k) * 3).to(dtype), randn(g, n, k).to(dtype)
            want, err, factor = ref.adjust(x, **more)
            leaf = x.to(DEV).requires_grad_()
            y = policy.adjust_logits(leaf, **on_gpu(more))
            assert y.dtype == dtype
            ref.close(y, want, err, dtype)
            dx, = torch.autograd.grad(y, leaf, up.to(DEV))
            ref.close(dx, ref.np64(up) * factor, np.abs(ref.np64(up) * factor) * ref.U32, dtype)
            with torch.no_grad():
                assert torch.equal(policy.adjust_logits(leaf, **on_gpu(more)), y)
                inplace = x.to(DEV)
                assert policy.adjust_logits(inplace, out=inplace, **on_gpu(more)) is inplace and torch.equal(inplace, y)


def test_adjust_of_special_values(policy):
    """What a barred place holds does not matter; elsewhere NaN stays NaN and infinities stay infinities, in the gradient as in
    the logits, and the type's lowest value is a number."""
    for dtype in DTYPES:
        low = torch.finfo(dtype).min
        x = torch.tensor([[math.nan, math.inf, -math.inf, low, 0.0, -0.0, 1.0, math.nan, math.inf, -math.inf]], dtype=dtype)
        mask = torch.tensor([[1, 1, 1, 1, 1, 1, 1, 0, 0, 0]], dtype=torch.bool)
        h = torch.tensor([[1, 2, 4, 5, 7, 8, 9]])
        more = dict(history=h, repetition=2.0, presence=0.25, frequency=0.5, mask=mask)
        leaf = x.to(DEV).requires_grad_()
        y = policy.adjust_logits(leaf, **on_gpu(more))
        want, err, factor = ref.adjust(x, **more)
        ref.close(y, want, err, dtype)
        up = torch.tensor([[1.0, 1.0, 1.0, math.nan, math.inf, 3.0, -math.inf, math.nan, math.inf, 2.0]], dtype=dtype)
        dx, = torch.autograd.grad(y, leaf, up.to(DEV))
        with np.errstate(invalid="ignore"):
            ref.close(dx, np.where(factor > 0, ref.np64(up) * factor, 0.0), np.zeros((1, 10)), dtype)


def test_adjust_strides(policy):
    g = gen(3)
    n, k, t = 37, 50, 12
    more = on_gpu(adjust_args(4, n, k, t, "bool"))
    x = randn(g, n, 2 * k + 3).to(DEV)
    h = torch.randint(0, k, (t, n), generator=g).to(DEV)
    wide = torch.zeros((n, 3 * k), dtype=torch.bool, device=DEV)
    wide[:, k:2 * k] = more["mask"]
    for logits in (x[:, 3:3 + k], x[:, :2 * k:2], randn(g, k, n).to(DEV).t()):
        plain = dict(more, history=h.t().contiguous(), lengths=None)
        odd = dict(more, history=h.t(), mask=wide[:, k:2 * k], bias=more["bias"].t().contiguous().t(), lengths=None)
        want = policy.adjust_logits(logits.contiguous(), **plain)
        assert torch.equal(policy.adjust_logits(logits, **odd), want)
        assert torch.equal(policy.adjust_logits(logits, **dict(odd, bias=more["bias"].double())), want)  # float32 numbers in another type
        leaf = logits.detach().requires_grad_()
        up = randn(g, n).to(DEV)[:, None].expand(n, k)
        dx, = torch.autograd.grad(policy.adjust_logits(leaf, **odd), leaf, up)
        flat = logits.contiguous().requires_grad_()
        assert torch.equal(dx, torch.autograd.grad(policy.adjust_logits(flat, **plain), flat, up.contiguous())[0])
    deep = randn(g, 3, 5, 7).to(DEV)  # [environments, agents, actions]
    mask = torch.rand((3, 5, 7), generator=g).to(DEV) < 0.5
    assert torch.equal(policy.adjust_logits(deep, mask=mask, presence=torch.ones((3, 5), device=DEV)),
                       policy.adjust_logits(deep.view(15, 7), mask=mask.view(15, 7), presence=1.0).view(3, 5, 7))
    one = randn(g, 9).to(DEV)
    assert torch.equal(policy.adjust_logits(one, bias=one), one + one)
    assert policy.adjust_logits(torch.empty((0, 9), device=DEV), mask=torch.empty((0, 9), dtype=torch.bool, device=DEV)).shape == (0, 9)


def test_adjust_gradient_against_differences(policy):
    """Linear where no logit changes its sign: |x| > 0.1 and a step of 2^-4."""
    g = gen(8)
    for n, k, t in ((50, 7, 9), (3, 9000, 700)):
        more = on_gpu(adjust_args(k, n, k, t, None))
        x, v, up = randn(g, n, k), torch.rand((n, k), generator=g) * 2 ** -4, randn(g, n, k)
        x = torch.where(x.abs() < 0.1, 0.5, x)
        leaf = x.to(DEV).requires_grad_()
        v, up = v.to(DEV), up.to(DEV)
        dx, = torch.autograd.grad(policy.adjust_logits(leaf, **more), leaf, up)
        with torch.no_grad():
            high, low = policy.adjust_logits(leaf + v, **more), policy.adjust_logits(leaf - v, **more)
        diff = ((high.double() - low.double()) * up.double()).sum() / 2
        # each of the two values is off by a few half steps of numbers below 100
        assert abs(float(diff - (dx.double() * v.double()).sum())) <= float(up.abs().sum()) * 8 * ref.U32 * 100


# ---- draw ----------------------------------------------------------------------------------------------------------------


ROWS = [(1, 1), (1, 2), (5, 7), (1000, 7), (4099, 7), (100, 8), (100, 9), (65, 15), (65, 16), (65, 17), (65, 32), (65, 33), (65, 63), (65, 64), (65, 65), (17, 255), (17, 256), (9, 257), (9, 1000),
        (3, 4097), (2, 8193), (1, 40007), (300, 2000), (2, 131072), (3, 20000), (2, 65537), (2, 131079), (1, 300001)]


def some_logits(g, n, k, dtype, barred=True):
    x = randn(g, n, k) * (3 if k > 64 else 1)
    if barred and k > 1:
        bar = torch.rand((n, k), generator=g) < 0.2
        bar[torch.arange(n), torch.randint(0, k, (n,), generator=g)] = False
        x = x.masked_fill(bar, -math.inf)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", ROWS)
def test_draw(policy, n, k, dtype):
    g = gen(n * 7 + k)
    x = some_logits(g, n, k, dtype)
    if n > 4:  # an even row, a row that has one token only, a row of two equal maxima, tokens that are far below
        x[0], x[1], x[1, k // 2], x[3] = 0.0, -math.inf, 0.0, torch.finfo(dtype).min
        x[2, 0] = x[2, k - 1] = x[2].max() + 1
    u64 = torch.rand(n, generator=g, dtype=torch.float64)
    if n > 2:
        u64[0], u64[n - 1] = 0.0, 1 - 2.0 ** -53
    t = 0.5 + torch.rand(n, generator=g)
    for u, temperature in ((u64, 1.0), (u64.float().clamp(max=1 - 2.0 ** -24), 0.7), (u64, t), (None, 1.0)):
        number = temperature if isinstance(temperature, torch.Tensor) else float(np.float32(temperature))
        tokens, lp, margin = ref.draw(x, u, number)
        got, got_lp = policy.draw(x.to(DEV), None if u is None else u.to(DEV),
                                  temperature=t.to(DEV) if isinstance(temperature, torch.Tensor) else temperature)
        assert got.dtype == torch.int64 and got_lp.dtype == torch.float32
        clear = margin > 1e-12  # nearer to a border than 64 bits say anything about
        assert clear.sum() >= n - 1
        got = got.cpu().numpy()
        assert np.array_equal(got[clear], tokens[clear])
        assert (np.abs(got - tokens)[~clear] <= k).all()
        bound = ref.logprobs(x, torch.from_numpy(tokens), number)[0][1]
        ref.close(got_lp[torch.from_numpy(clear)], lp[clear], bound[clear], torch.float32)


def test_draw_follows_the_probabilities(policy):
    """n evenly spaced numbers give every token its share to within one."""
    x = randn(gen(2), 7)
    n = 100000
    u = (torch.arange(n, dtype=torch.float64) + 0.5) / n
    tokens, _ = policy.draw(x.to(DEV).expand(n, 7), u.to(DEV))
    share = torch.softmax(x.double(), 0) * n
    assert (torch.bincount(tokens.cpu(), minlength=7) - share).abs().max() <= 1.0


@pytest.mark.parametrize("k", [1, 7, 64, 65, 1000, 70000])
def test_draw_from_rows_that_are_no_distribution(policy, k):
    for dtype in DTYPES:
        x = torch.zeros((6, k), dtype=dtype)
        x[0] = -math.inf
        x[1, k - 1] = math.nan
        x[2, 0] = math.inf
        x[3] = -math.inf
        x[3, k // 2] = math.nan
        x[4, k // 3], x[4, k - 1] = math.inf, math.nan
        for u in (torch.full((6,), 0.5, device=DEV), None):
            tokens, lp = policy.draw(x.to(DEV), u, dtype=torch.int32)
            assert tokens.dtype == torch.int32
            assert tokens[:5].tolist() == [-1] * 5 and lp[0].item() == -math.inf and torch.isnan(lp[1:5]).all()
            assert 0 <= tokens[5].item() < k and abs(lp[5].item() + math.log(k)) <= ref.U32 * (math.log(k) + k / 64 + 24)
            if k <= 255:
                small, _ = policy.draw(x.to(DEV), u, dtype=torch.uint8)
                assert small.dtype == torch.uint8 and small.tolist() == [255] * 5 + [tokens[5].item()]


def test_draw_strides_and_shapes(policy):
    g = gen(4)
    x = randn(g, 6, 5, 2 * 7).to(DEV)
    u = torch.rand((5, 6), generator=g).to(DEV).t()
    tokens, lp = policy.draw(x[..., ::2], u)
    want = policy.draw(x[..., ::2].contiguous(), u.contiguous())
    assert tokens.shape == (6, 5) and torch.equal(tokens, want[0]) and torch.equal(lp, want[1])
    wide = randn(g, 40, 3000).to(DEV)[:, 5:2005]
    for a, b in zip(policy.draw(wide), policy.draw(wide.contiguous())):
        assert torch.equal(a, b)
    tokens, lp = policy.draw(x[0, 0])
    assert tokens.shape == () and lp.shape == ()
    tokens, lp = policy.draw(torch.empty((0, 9), device=DEV))
    assert tokens.shape == (0,) and lp.shape == (0,)
    with torch.no_grad():
        same = randn(g, 9).to(DEV).expand(20, 9)
    assert (policy.draw(same)[0] == same[0].argmax()).all()


# ---- log-probabilities ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", ROWS)
def test_token_logprobs(policy, n, k, dtype):
    g = gen(n * 13 + k)
    x = some_logits(g, n, k, dtype)
    tokens = torch.randint(0, k, (n,), generator=g)
    if n > 8:
        x[0] = -math.inf  # nothing allowed
        x[1] = torch.finfo(dtype).min  # an even row of the type's lowest value
        x[2], x[2, k // 2] = -20.0, 0.0  # one token holds nearly everything
        tokens[2] = k // 2
        x[3], x[3, 0] = -math.inf, 3.0
        x[4], x[4, k - 1] = 0.0, 12.0
        tokens[5], tokens[6] = -1, k  # padding
        x[7] = x[7] * 30  # a steep row
    up, up_h = randn(g, n), randn(g, n)
    t = 0.5 + torch.rand(n, generator=g)
    kinds = [torch.int64, torch.int32] + ([torch.uint8] if k < 255 else [])
    for kind, temperature in zip(kinds, (1.0, t, 0.75)):
        tok = tokens.clamp(min=0).to(kind) if kind == torch.uint8 else tokens.to(kind)
        number = temperature if isinstance(temperature, torch.Tensor) else float(np.float32(temperature))
        want = ref.logprobs(x, tok, number, up, up_h)
        leaf = x.to(DEV).requires_grad_()
        lp, h = policy.token_logprobs(leaf, tok.to(DEV), temperature=t.to(DEV) if isinstance(temperature, torch.Tensor) else temperature)
        ref.close(lp, *want[0], torch.float32)
        ref.close(h, *want[1], torch.float32)
        dx, = torch.autograd.grad((lp, h), leaf, (up.to(DEV), up_h.to(DEV)), retain_graph=True)
        assert dx.dtype == dtype
        ref.close(dx, *want[2], dtype)
        dx, = torch.autograd.grad(lp, leaf, up.to(DEV), retain_graph=True)
        ref.close(dx, *ref.logprobs(x, tok, number, up, up_h * 0)[2], dtype)
        dx, = torch.autograd.grad(h.sum(), leaf)
        ref.close(dx, *ref.logprobs(x, tok, number, up * 0, up_h * 0 + 1)[2], dtype)
        with torch.no_grad():
            again = policy.token_logprobs(leaf, tok.to(DEV), temperature=t.to(DEV) if isinstance(temperature, torch.Tensor) else temperature)
        assert torch.equal(again[0], lp) and torch.equal(again[1], h)


@pytest.mark.parametrize("k", [3, 7, 64, 65, 1000, 70000])
def test_token_logprobs_of_nan_and_infinity(policy, k):
    """A NaN or +inf in a row makes that row's results NaN, and no other's."""
    x = torch.zeros((5, k))
    x[0, 1], x[1, 2] = math.nan, math.inf
    x[3] = -math.inf
    x[3, k - 1] = math.nan
    leaf = x.to(DEV).requires_grad_()
    lp, h = policy.token_logprobs(leaf, torch.zeros(5, dtype=torch.int64, device=DEV))
    dx, = torch.autograd.grad((lp, h), leaf, (torch.ones_like(lp), torch.ones_like(h)))
    for i, bad in enumerate((True, True, False, True, False)):
        assert bool(torch.isnan(h[i])) == bad and bool(torch.isnan(dx[i]).any()) == bad, i
        assert bool(torch.isnan(lp[i])) == bad, i


@pytest.mark.parametrize("n,k", [(40, 7), (5, 300), (2, 9001)])
def test_token_logprobs_gradient_against_differences(policy, n, k):
    """Third derivatives of log-probability and entropy along a direction of entries below 1 are below 64 (sums of products of up
    to three centred entries, each below 2, weighted with probabilities, times log-probabilities for the entropy, below 12 here)."""
    g = gen(k)
    x, v = randn(g, n, k).to(DEV), (torch.rand((n, k), generator=g) * 2 - 1).to(DEV)
    tokens = torch.randint(0, k, (n,), generator=g).to(DEV)
    c, d = randn(g, n).to(DEV), randn(g, n).to(DEV)
    leaf = x.requires_grad_()
    lp, h = policy.token_logprobs(leaf, tokens)
    dx, = torch.autograd.grad((lp, h), leaf, (c, d))
    step = 2.0 ** -6
    with torch.no_grad():
        (lp1, h1), (lp0, h0) = policy.token_logprobs(x + step * v, tokens), policy.token_logprobs(x - step * v, tokens)
    diff = ((lp1 - lp0).double() * c + (h1 - h0).double() * d) / (2 * step)
    slope = (dx.double() * v).sum(1)
    bound = (c.abs() * 64 + d.abs() * 64 * 12) * step ** 2 / 6 + (c.abs() + d.abs()) * 64 * ref.U32 * 16 / step
    assert ((diff - slope).abs() <= bound).all()


def test_token_logprobs_strides_and_shapes(policy):
    g = gen(6)
    x = randn(g, 4, 5, 21).to(DEV)
    tokens = torch.randint(0, 7, (5, 4), generator=g).to(DEV).t()
    up = randn(g, 5, 4).to(DEV).t()
    flat = x[..., ::3].contiguous().requires_grad_()
    leaf = x[..., ::3].detach().requires_grad_()
    a, b = policy.token_logprobs(leaf, tokens), policy.token_logprobs(flat, tokens.contiguous())
    assert a[0].shape == (4, 5) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    da, = torch.autograd.grad(a, leaf, (up, torch.ones((), device=DEV).expand(4, 5)))
    db, = torch.autograd.grad(b, flat, (up.contiguous(), torch.ones((4, 5), device=DEV)))
    assert torch.equal(da, db)
    lp, h = policy.token_logprobs(x[0, 0], torch.tensor(3, device=DEV))
    assert lp.shape == () and h.shape == ()
    one = x[0, 0].detach().requires_grad_()
    lp, h = policy.token_logprobs(one, torch.tensor(3, device=DEV))
    lp.backward()
    assert one.grad.shape == (21,)
    none = torch.empty((0, 9), device=DEV, requires_grad=True)
    lp, h = policy.token_logprobs(none, torch.empty((0,), dtype=torch.int64, device=DEV))
    (lp.sum() + h.sum()).backward()
    assert none.grad.shape == (0, 9)


# ---- together ------------------------------------------------------------------------------------------------------------


def small_policy(g):
    """Weights of a first layer by cell, and of a linear layer from a 7 x 7 view to seven actions."""
    return [(randn(g, 24, 8) * 0.3).to(DEV), (randn(g, 7 * 7 * 8, 7) * 0.05).to(DEV)]


def test_a_policy_acts_and_trains(policy):
    """Observation -> embedding -> logits -> adjustment -> draw -> step, then the log-probabilities of what was done; the gradients
    against the same network of one-hot cells in torch, in 64 bits."""
    from multigrid_amd import views
    from multigrid_amd.vector import MultiGridVectorEnv
    n, agents, steps = 64, 2, 6
    env = MultiGridVectorEnv("MultiGrid-BlockedUnlockPickup-v0", n, agents=agents, num_layouts=16, agent_view_size=7)
    g = gen(12)
    weights = [w.requires_grad_() for w in small_policy(g)]
    bias = randn(g, 7).to(DEV)
    obs, _ = env.reset(seed=3)
    past = torch.full((n, agents, 4), 255, dtype=torch.uint8, device=DEV)
    kept = []
    for _ in range(steps):
        image = obs["image"].clone()
        mask = torch.ones((n, agents, 7), dtype=torch.bool, device=DEV)
        mask[::3, 0, 2] = False
        mask[5, 1] = False  # may do nothing at all
        adjust = dict(history=past.clone(), repetition=1.2, presence=0.1, frequency=0.05, bias=bias, mask=mask)
        u = torch.rand((n, agents), generator=g).to(DEV)
        with torch.no_grad():
            logits = views.cell_embedding(image, weights[0]).reshape(n, agents, -1) @ weights[1]
        obs, reward, term, trunc, infos = env.step_logits(logits, u, temperature=0.9, **adjust)
        actions = infos["actions"]
        assert actions.dtype == torch.uint8 and actions[5, 1] == 255 and not (actions[::3, 0] == 2).any()
        kept.append((image, adjust, actions, infos["action_logprobs"]))
        past = torch.cat((past[..., 1:], actions[..., None]), -1)
    images, actions = torch.stack([k[0] for k in kept]), torch.stack([k[2] for k in kept]).long()
    actions = torch.where(actions == 255, -1, actions)
    more = {k: torch.stack([s[1][k] for s in kept]) for k in ("history", "mask")}
    # as the training step computes it
    logits = views.cell_embedding(images, weights[0]).reshape(steps, n, agents, -1) @ weights[1]
    adjusted = policy.adjust_logits(logits, repetition=1.2, presence=0.1, frequency=0.05, bias=bias, **more)
    lp, h = policy.token_logprobs(adjusted, actions, temperature=0.9)
    drawn = torch.stack([k[3] for k in kept])
    live = actions >= 0
    assert (drawn[~live] == -math.inf).all() and (lp[~live] == 0).all()
    assert torch.allclose(lp[live], drawn[live], rtol=0, atol=1e-4)  # the products before differ in shape, so in their roundings
    advantage = randn(g, steps, n, agents).to(DEV)
    loss = -(lp * advantage).sum() - 0.01 * h.sum()
    got = torch.autograd.grad(loss, weights)
    # in 64 bits
    ws = [w.detach().double().cpu().requires_grad_() for w in weights]
    im, off = images.cpu().long(), torch.tensor([0, 11, 17])
    hot = torch.nn.functional.one_hot(im + off, 24).sum(-2).double()
    x = (hot @ ws[0]).reshape(steps * n * agents, -1) @ ws[1]
    hist, m = more["history"].cpu().view(-1, 4), more["mask"].cpu().view(-1, 7)
    c = torch.from_numpy(ref.history_counts(hist, None, len(x), 7))
    rep = float(np.float32(1.2))
    y = torch.where(c > 0, torch.where(x > 0, x / rep, x * rep) - 0.1, x) - 0.05 * c + bias.cpu().double()
    y = y.masked_fill(~m, -math.inf)[m.any(1)] / 0.9
    logp = torch.log_softmax(y, -1)
    acts = actions.cpu().view(-1)[m.any(1)]
    taken = logp.gather(1, acts[:, None])[:, 0]
    entropy = -(logp.exp() * torch.where(logp == -math.inf, 0.0, logp)).sum(1)
    want = torch.autograd.grad(-(taken * advantage.cpu().double().view(-1)[m.any(1)]).sum() - 0.01 * entropy.sum(), ws)
    for a, b in zip(got, want):
        # sums of up to steps * n * agents * 49 products of 32-bit numbers; the library's product adds its own roundings
        assert (a.cpu().double() - b).norm() <= 1e-4 * b.norm()
    env.close()


def test_step_logits_single_agent_and_numpy(policy):
    from multigrid_amd.vector import MultiGridVectorEnv
    for numpy in (False, True):
        one, two = (MultiGridVectorEnv("MultiGrid-Empty-8x8-v0", 20, agents=1, num_layouts=8, single_agent=True, numpy=numpy) for _ in range(2))
        one.reset(seed=1), two.reset(seed=1)
        g = gen(3)
        for _ in range(5):
            logits, u = randn(g, 20, 7).to(DEV), torch.rand(20, generator=g).to(DEV)
            got = one.step_logits(logits, u)
            tokens, lp = policy.draw(logits, u, dtype=torch.uint8)
            want = two.step(tokens)
            acts = torch.as_tensor(got[4]["actions"]).cpu()
            assert torch.equal(acts, tokens.cpu()) and torch.equal(torch.as_tensor(got[4]["action_logprobs"]).cpu(), lp.cpu())
            for a, b in zip((got[0]["image"], got[1], got[2], got[3]), (want[0]["image"], want[1], want[2], want[3])):
                assert torch.equal(torch.as_tensor(a), torch.as_tensor(b))
        with pytest.raises(ValueError, match="logits"):
            one.step_logits(torch.zeros((20, 1, 7), device=DEV))
        one.close(), two.close()


def test_no_action_changes_nothing_but_the_step_count():
    """255 among the actions is what ``done`` is: the agent stays as it is."""
    from multigrid_amd import envs, layouts
    from multigrid_amd.batched import BatchedMultiGrid
    for name, agents in (("MultiGrid-Empty-8x8-v0", 2), ("MultiGrid-LockedHallway-4Rooms-v0", 4), ("MultiGrid-Empty-16x16-v0", 8)):
        spec, make = envs.make_spec(name, num_agents=agents, agent_view_size=7)
        sims = [BatchedMultiGrid(spec, 40, device=0) for _ in range(2)]
        pool = layouts.make_pool(make, 8, seed0=2)[:3]
        g = gen(agents)
        for s in sims:
            s.upload_layouts(*pool)
            s.reset()
        for _ in range(10):
            acts = torch.randint(0, 6, (40, agents), generator=g, dtype=torch.uint8)
            none = torch.rand((40, agents), generator=g) < 0.4
            order = torch.argsort(torch.rand((40, agents), generator=g), 1).to(torch.uint8)
            outs = [s.step(acts.masked_fill(none, v), order) for s, v in zip(sims, (255, 6))]
            torch.cuda.synchronize()
            assert torch.equal(outs[0].image, outs[1].image) and torch.equal(outs[0].reward, outs[1].reward)
        a, b = (s.get_state() for s in sims)
        assert all(torch.equal(a[k], b[k]) for k in a)
        for s in sims:
            s.close()


@pytest.mark.parametrize("n,k,rows,dim", [(130, 7, 24, 16), (9000, 7, 24, 16), (33, 9001, 3000, 72), (5000, 300, 2000, 40)])
def test_captured_and_replayed(policy, n, k, rows, dim):
    """Every operator in one graph, replayed on new inputs with other work in between; two graphs whose replays take turns."""
    g = gen(n + k)

    def inputs():
        return dict(ids=torch.randint(0, rows, (n,), generator=g).to(DEV), table=randn(g, rows, dim).to(DEV), up=randn(g, n, dim).to(DEV),
                    logits=some_logits(g, n, k, torch.float32).to(DEV), u=torch.rand(n, generator=g, dtype=torch.float64).to(DEV),
                    history=torch.randint(0, k, (n, 11), generator=g).to(DEV), tokens=torch.randint(0, k, (n,), generator=g).to(DEV),
                    gl=randn(g, n).to(DEV))

    def work(s):
        out = policy.embed(s["ids"], s["table"])
        dw = policy.embed_grad(s["up"], s["ids"], rows)
        y = policy.adjust_logits(s["logits"], history=s["history"], repetition=1.3, frequency=0.1)
        tokens, lp = policy.draw(y, s["u"], temperature=0.8)
        with torch.enable_grad():  # of a tensor that only this call sees
            leaf = y.detach().requires_grad_()
            lps, h = policy.token_logprobs(leaf, s["tokens"])
            dl, = torch.autograd.grad((lps, h), leaf, (s["gl"], s["gl"]))
        return [out, dw, y, tokens, lp, lps.detach(), h.detach(), dl]

    graphs = []
    for _ in range(2):
        s = inputs()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work(s)
        graphs.append((graph, s, outs))
    for _ in range(3):
        for graph, s, outs in graphs:
            fresh = inputs()
            for key in s:
                s[key].copy_(fresh[key])
            want = work(fresh)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
        for graph, s, outs in graphs:  # one behind the other, nothing between
            graph.replay()
        torch.cuda.synchronize()
        for graph, s, outs in graphs:
            for a, b in zip(outs, work(s)):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(policy):
    g = gen(1)
    sets = [dict(ids=torch.randint(0, 3000, (6000,), generator=g).to(DEV), up=randn(g, 6000, 64).to(DEV), x=randn(g, 12, 70001).to(DEV),
                 u=torch.rand(12, generator=g).to(DEV), h=torch.randint(0, 70001, (12, 300), generator=g).to(DEV)) for _ in range(2)]

    def work(s):
        return [policy.embed_grad(s["up"], s["ids"], 3000), policy.adjust_logits(s["x"], history=s["h"], presence=1.0), *policy.draw(s["x"], s["u"]),
                *policy.token_logprobs(s["x"], s["h"][:, 0].contiguous())]

    want = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(work(s))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


# ---- what no argument check can see, and what one refuses --------------------------------------------------------------------


@pytest.mark.parametrize("k", [7, 33, 64, 600, 2000, 9000, 70000])
def test_temperatures_and_uniforms_out_of_range(policy, k):
    g = gen(k)
    inf, nan = math.inf, math.nan
    x = randn(g, 7, k)
    x[:, : k // 3] = -inf
    x[:, -(k // 3):] = -inf
    temperature = torch.tensor([0.0, -1.0, nan, inf, 1e-40, 1.0, 2.0 ** -126])
    x, t = x.to(DEV), temperature.to(DEV)
    for u in (torch.full((7,), 0.5, device=DEV), None):
        tokens, lp = policy.draw(x, u, temperature=t)
        assert (tokens[:5] == -1).all() and lp[:5].isnan().all()
        assert (tokens[5:] >= k // 3).all() and (tokens[5:] < k - k // 3).all() and lp[5:].isfinite().all()
        assert tokens[6] == x[6].argmax()  # next to nothing beside it
    leaf = x.clone().requires_grad_()
    lp, h = policy.token_logprobs(leaf, torch.full((7,), k // 2, device=DEV), temperature=t)
    assert lp[:5].isnan().all() and h[:5].isnan().all() and lp[5].isfinite() and not lp[6].isnan() and h[5:].isfinite().all()
    grad, = torch.autograd.grad(lp[:6].sum() + h[:6].sum(), leaf)
    barred = x.isinf()
    assert (grad[barred] == 0).all() and grad[:5][~barred[:5]].isnan().all() and grad[5].isfinite().all()
    # uniform numbers below, above and none at all: the first and the last token that has a probability
    low, _ = policy.draw(x, torch.tensor([-1.0, nan, -inf, 0.0, -1e-30, -0.0, -5.0], device=DEV))
    high, _ = policy.draw(x, torch.tensor([1.0, 2.0, inf, 1e30, 1.0, 1.0, 1.5], device=DEV))
    assert (low == k // 3).all() and (high == k - k // 3 - 1).all()


@pytest.mark.parametrize("k", [7, 300, 70000])
def test_token_logprobs_of_infinite_gradients(policy, k):
    x = randn(gen(k), 4, k)
    x[:, ::2] = -math.inf
    x = x.to(DEV).requires_grad_()
    lp, h = policy.token_logprobs(x, torch.ones(4, dtype=torch.int64, device=DEV))
    up = torch.tensor([math.inf, -math.inf, math.nan, 1.0], device=DEV)
    grad, = torch.autograd.grad((lp, h), x, (up, torch.zeros_like(up)))
    assert (grad[:, ::2] == 0).all() and grad[3].isfinite().all()


def test_embed_of_many_tokens_from_one_field(policy):
    # finished rows and the table itself, side by side, would pass the LDS that a launch may ask for
    n, rows, dim = 16 * 256 * 1001 + 3, 1000, 12
    g = gen(3)
    ids = torch.randint(0, rows + 1, (n,), generator=g, dtype=torch.int32).to(DEV)
    table = randn(g, rows, dim).to(DEV)
    got = policy.embed(ids, table, scale=2.0)
    want = torch.where((ids < rows)[:, None], 2.0 * table[ids.clamp(max=rows - 1).long()], 0.0)
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [24, 100])
def test_embed_of_the_widest_rows(policy, rows):
    dim, n = 1 << 20, 40
    g = gen(rows)
    ids = torch.randint(0, rows, (n,), generator=g)
    table = torch.arange(rows * dim, device=DEV, dtype=torch.float32).reshape(rows, dim) % 1021
    up = torch.arange(n * dim, device=DEV, dtype=torch.float32).reshape(n, dim) % 1019
    assert torch.equal(policy.embed(ids.to(DEV), table), table[ids.to(DEV)])
    want = torch.zeros(rows, dim, device=DEV)  # whole numbers: every order gives the same sum
    for i, r in enumerate(ids.tolist()):
        want[r] += up[i]
    assert torch.equal(policy.embed_grad(up, ids.to(DEV), rows), want)
    with pytest.raises(ValueError, match="not supported"):
        policy.embed_grad(torch.empty(1, dim + 1, device=DEV), ids[:1].to(DEV), rows)


def test_refusals(policy):
    f = lambda *shape, dtype=torch.float32: torch.zeros(shape, device=DEV, dtype=dtype)
    x, table, ids = f(4, 9), f(24, 8), f(5, dtype=torch.int64)
    asks = lambda t: t.clone().requires_grad_()
    refused = [
        (lambda: policy.embed(ids.cpu(), table), "GPU"), (lambda: policy.embed(ids, table.cpu()), "GPU"), (lambda: policy.embed(ids.float(), table), "ids must be"),
        (lambda: policy.embed(ids, table.double()), "table must be"), (lambda: policy.embed(ids, f(8)), "table must be"), (lambda: policy.embed(ids, f(0, 8)), "hold something"),
        (lambda: policy.embed(f(5, 3, dtype=torch.uint8), table, fields=(11, 6, 8)), "add up"), (lambda: policy.embed(f(5, 2, dtype=torch.uint8), table, fields=(11, 6, 7)), "fields"),
        (lambda: policy.embed(f(5, 9, dtype=torch.uint8), table, fields=(1,) * 8 + (16,)), "fields"), (lambda: policy.embed(f(5, 2, dtype=torch.uint8), table, fields=(24, 0)), "positive"),
        (lambda: policy.embed_grad(f(6, 8), ids, 24), "shape"), (lambda: policy.embed_grad(f(5, 8), ids, 0), "hold something"),
        (lambda: policy.adjust_logits(x.double()), "logits must be"), (lambda: policy.adjust_logits(x, history=f(3, 2, dtype=torch.int64)), "history must be"),
        (lambda: policy.adjust_logits(x, history=f(4, 2)), "history must be"), (lambda: policy.adjust_logits(x, lengths=f(4, dtype=torch.int32)), "without a history"),
        (lambda: policy.adjust_logits(x, history=f(4, 2, dtype=torch.int32), lengths=f(3, dtype=torch.int32)), "lengths must be"),
        (lambda: policy.adjust_logits(x, mask=f(4, 8, dtype=torch.bool)), "mask must be"), (lambda: policy.adjust_logits(x, mask=f(4, 9)), "mask must be"),
        (lambda: policy.adjust_logits(x, mask=f(4, 2, dtype=torch.int32)), "mask must be"), (lambda: policy.adjust_logits(x, bias=f(8)), "bias must be"),
        (lambda: policy.adjust_logits(x, presence=f(3)), "presence must be"), (lambda: policy.adjust_logits(x, out=f(4, 8)), "out must be"),
        (lambda: policy.adjust_logits(x, out=f(9, 4).t()), "out must be"), (lambda: policy.adjust_logits(x, out=x.half()), "out must be"),
        (lambda: policy.adjust_logits(asks(x), out=f(4, 9)), "not differentiable"), (lambda: policy.adjust_logits(f(5, 9)[:4], out=f(4, 9).cpu()), "GPU"),
        (lambda: policy.draw(x, f(3)), "uniforms must be"), (lambda: policy.draw(x, f(4, dtype=torch.float16)), "uniforms must be"),
        (lambda: policy.draw(x, dtype=torch.int16), "dtype must be"), (lambda: policy.draw(f(2, 256), dtype=torch.uint8), "uint8"), (lambda: policy.draw(x, temperature=f(2)), "temperature must be"),
        (lambda: policy.token_logprobs(x, f(3, dtype=torch.int64)), "tokens must be"), (lambda: policy.token_logprobs(x, f(4)), "tokens must be"), (lambda: policy.token_logprobs(x[0, 0], ids), "logits must be"),
        # gradients that would be lost without a word
        (lambda: policy.adjust_logits(asks(x), bias=asks(f(9))), "bias passes no"), (lambda: policy.adjust_logits(x, bias=asks(f(9))), "bias passes no"),
        (lambda: policy.adjust_logits(asks(x), repetition=asks(f(4))), "repetition passes no"), (lambda: policy.adjust_logits(asks(x), presence=asks(f(4))), "presence passes no"),
        (lambda: policy.adjust_logits(x, frequency=asks(f(4))), "frequency passes no"), (lambda: policy.draw(x, temperature=asks(f(4))), "temperature passes no"),
        (lambda: policy.token_logprobs(asks(x), f(4, dtype=torch.int64), temperature=asks(f(4))), "temperature passes no"),
    ]
    for call, text in refused:
        with pytest.raises(ValueError, match=text):
            call()
    # out across what the call reads
    whole = f(10, 9)
    for more in (dict(out=whole[1:5]), dict(out=whole[4:8], bias=whole[7]), dict(out=whole[4:8], presence=whole.view(-1)[36:40])):
        with pytest.raises(ValueError, match="across"):
            policy.adjust_logits(whole[:4], **more)
    from multigrid_amd._lib import MgError
    for call in (lambda: policy.draw(x, temperature=0.0), lambda: policy.draw(x, temperature=1e-40), lambda: policy.token_logprobs(x, f(4, dtype=torch.int64), temperature=math.nan),
                 lambda: policy.adjust_logits(x, repetition=0.0)):
        with pytest.raises(MgError, match="temperature must be|repetition must be"):
            call()
    # differentiable once
    for out, leaf in ((lambda t: policy.embed(ids, t), table), (lambda t: policy.adjust_logits(t, presence=1.0), x), (lambda t: policy.token_logprobs(t, ids[:4])[0], x)):
        leaf = asks(leaf)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(out(leaf).sum(), leaf, create_graph=True)


def test_capture_beside_an_eager_graph_of_the_same_leaf(policy):
    table = randn(gen(1), 24, 8).to(DEV).requires_grad_()
    w = randn(gen(2), 6, 9).to(DEV).requires_grad_()
    ids, tokens, x = torch.arange(24, device=DEV), torch.arange(4, device=DEV), randn(gen(3), 4, 6).to(DEV)
    calls = [lambda: policy.embed(ids, table), lambda: policy.adjust_logits(x @ w, presence=1.0), lambda: policy.token_logprobs(x @ w, tokens)[0]]
    with torch.no_grad():
        x @ w  # the library's own first call
    held = [call().sum() for call in calls]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mark = x + 1  # (a graph of nothing is reported)
        for call in calls:
            with pytest.raises(RuntimeError, match="eager graph"):
                call()
    graph.replay()
    del held, graph
    # with that graph gone the same is captured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, = torch.autograd.grad(calls[0]().square().sum(), table)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(calls[0]().square().sum(), table)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert torch.equal(mark, x + 1)


@pytest.mark.parametrize("t", [65535, 65536, 70001])
@pytest.mark.parametrize("k", [20, 40])
def test_adjust_counts_beyond_16_bits(policy, t, k):
    # one token throughout, in one row; its neighbours' counts must not see it
    x = randn(gen(t), 2, k)
    history = torch.full((2, t), 3)
    history[1] = torch.arange(t) % k
    y = policy.adjust_logits(x.to(DEV), history=history.to(DEV), repetition=1.25, presence=0.5, frequency=2.0 ** -12)
    want, err, _ = ref.adjust(x, history, None, 1.25, 0.5, 2.0 ** -12)
    ref.close(y, want, err, torch.float32)


def test_the_longest_rows(policy):
    k = 1 << 24
    x = torch.zeros((1, k), dtype=torch.bfloat16)
    x[0, 5], x[0, k - 1] = 3.0, 17.0
    total = (k - 2) + math.exp(3.0) + math.exp(17.0)
    d = x.to(DEV).requires_grad_()
    # a border in the middle of the equal ones, and one behind them
    for u, token in ((0.25 * (k - 2) / total, None), (0.9, k - 1), (None, k - 1)):
        got, lp = policy.draw(d.detach(), None if u is None else torch.tensor([u], dtype=torch.float64, device=DEV))
        if token is None:  # tokens 0 .. j hold j plus the sixth's surplus
            token = math.floor(u * total - (math.exp(3.0) - 1.0))
            assert abs(int(got) - token) <= 1  # (one step where the product above is rounded the other way)
            assert abs(float(lp) + math.log(total)) < 1e-5
        else:
            assert int(got) == token
    lp, h = policy.token_logprobs(d, torch.tensor([k - 1], device=DEV))
    # relative to the sum: 32 additions in a thread, 8 levels of a block, 38 merges of four roundings, which make 192; an exponent of
    # up to 17 log2(e), rounded twice, 50 more: 256 half steps; the entropy is a mean of exponents of up to 17 on top of it
    off = 256 * 2.0 ** -24
    assert abs(float(lp.detach()) - (17.0 - math.log(total))) < off
    p = (math.exp(17.0) / total, math.exp(3.0) / total, 1.0 / total)
    entropy = -(p[0] * math.log(p[0]) + p[1] * math.log(p[1]) + (k - 2) * p[2] * math.log(p[2]))
    assert abs(float(h.detach()) - entropy) < off * (1.0 + 2 * 17.0)
    grad, = torch.autograd.grad(lp, d)
    assert grad.shape == d.shape and abs(float(grad[0, k - 1]) - (1.0 - p[0])) < 2.0 ** -8 and abs(float(grad[0, 7]) + p[2]) < p[2] * 2.0 ** -7
    y = policy.adjust_logits(d.detach(), history=torch.tensor([[5, k - 1, k, -1]], device=DEV), presence=2.0)
    assert float(y[0, 5]) == 1.0 and float(y[0, k - 1]) == 15.0 and float(y.float().sum()) == 16.0
    with pytest.raises(ValueError, match="not supported"):
        policy.draw(torch.empty((1, k + 1), dtype=torch.bfloat16, device=DEV))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int64])
@pytest.mark.parametrize("n,sizes", [(1, (5,)), (101, (11, 6, 7)), (140003, (11, 6, 7)), (60005, (2, 3)), (60007, (7,)), (501, (200, 30))])
def test_the_backward_pass_has_the_ids_of_the_forward_pass(policy, n, sizes, dtype):
    # every way of embedding writes the copy itself: ids side by side, apart, and the same for all tokens
    g = gen(n)
    wide = torch.stack([torch.randint(0, r + 1, (n, 2), generator=g) for r in sizes], -1).to(dtype).to(DEV)  # [n, 2, fields]
    w, up = randn(g, sum(sizes), 16).to(DEV).requires_grad_(), randn(g, n, 16).to(DEV)
    for ids in (wide[:, 0].contiguous(), wide[:, 1], wide[:1, 0].expand(n, -1)):
        want = policy.embed_grad(up, ids.clone(), sum(sizes), fields=sizes)
        y = policy.embed(ids, w, fields=sizes)
        with torch.no_grad():
            assert torch.equal(policy.embed(ids, w, fields=sizes), y)
        kept = wide.clone()
        ids[:1].fill_(0) if ids.stride(0) == 0 else ids.fill_(0)
        assert torch.equal(torch.autograd.grad(y, w, up)[0], want)
        wide.copy_(kept)
