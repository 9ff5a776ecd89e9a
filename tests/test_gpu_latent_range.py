"""Attention over the quantised latent cache where probabilities and scales span many powers of two: one key that holds
nearly all of a head's probability over a broad tail (an attention sink), groups of dims whose scales lie far apart.

Bounds: check_attend's (a probability is off by at most a bf16 half step, 2^-8 of itself, however small it is), and for
the queries, which up to 16 heads are two e4m3 numbers, the second lifted by 16, 2^-21 of a row's largest latent value
(half of e4m3's smallest step, 2^-10, over 16, of values whose largest is between 224 and 448)."""
import pytest
import torch

from oracle import latent_oracle as L
from tests.test_gpu_latent_cache import BF16, DEV, F32, _status, run_attend

pytestmark = pytest.mark.gpu
QUERY = 2.0 ** -21


def check_range(c, ctx, lse, items, query=QUERY):
    """Every item of `items` against the 64-bit definition."""
    for i in items:
        slots = L.item_keys(c["idx"][i], c["table"][int(c["req"][i])], c["page"], int(c["qpos"][i]))
        rows, q = L.cache_rows(c["cache"], slots), c["q"][i].double()
        ref, ref_lse, mass, qk = L.attend(q, rows, c["scale"])
        k = slots.numel()
        q_off = query * q[:, :512].abs().amax(1) * rows[:, :512].abs().sum(1).max() * c["scale"] * (q.shape[0] <= 16)
        d = (576 * F32 * qk + q_off).view(-1, 1) + 1e-6           # error of a score; exp of it is relative
        step = BF16 if ctx.dtype == torch.bfloat16 else F32
        bound = (BF16 + 2 * d + k * F32) * mass + step * ref.abs() + 1e-30
        got = ctx[i].double().cpu()
        assert bool(((got - ref).abs() <= bound).all()), (i, float(((got - ref).abs() / bound).max()))
        lim = d.view(-1) + k * F32 + 8 * F32 * ref_lse.abs() + 2e-7
        assert bool(((lse[i].double().cpu() - ref_lse).abs() <= lim).all())


def range_case(seed, H, nats, at, k=2048, items=1, scales=(0, 0, 0, 0)):
    """k keys whose codes share a mean, their scores decided by the first position dim: key number `at` of the list lies
    `nats` above the others, which are within one of each other.  scales: powers of two of the four groups."""
    g = torch.Generator().manual_seed(seed)
    page = 64
    pages = (k + page - 1) // page
    cache = torch.zeros(pages * page, 656, dtype=torch.uint8)
    codes = (torch.randn(k, 512, generator=g) * 40 + 90).clamp(-448, 448)
    cache[:k, :512] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    cache[:k, 512:528] = torch.exp2(torch.tensor(scales).float() - 7).repeat(k, 1).view(torch.uint8)
    pe = torch.zeros(k, 64)
    pe[:, 0] = torch.rand(k, generator=g)
    order = torch.randperm(k, generator=g)
    pe[order[at], 0] = nats + 0.5
    cache[:k, 528:] = pe.bfloat16().view(torch.uint8)
    q = 2.0 ** -6 * torch.randn(items, H, 576, generator=g)
    q[:, :, 512:] = 0
    q[:, :, 512] = 16                                              # times 1/16: nats
    return {"cache": cache, "page": page, "scale": 1 / 16, "table": torch.arange(pages, dtype=torch.int32).view(1, -1),
            "q": q.bfloat16(), "req": torch.zeros(items, dtype=torch.int32), "idx": order.to(torch.int32).repeat(items, 1),
            "qpos": torch.full((items,), k, dtype=torch.int32), "lens": torch.tensor([k]), "mask": None}


@pytest.mark.parametrize("H", [1, 8, 16, 17])
@pytest.mark.parametrize("nats", [6.0, 8.0, 9.5, 10.0, 12.0, 15.0])
def test_one_key_over_a_broad_tail(H, nats):
    """In the first and in the last tile of the list, one CTA an item and several; 17 heads take the other kernel."""
    for at in (3, 2045):
        c = range_case(int(nats * 2) + H + at, H, nats, at)
        for splits in (1, 5):
            ws = (splits, torch.empty(splits * H * 513, device=DEV) if splits > 1 else None)
            out, lse = run_attend(c, ctx=torch.empty(1, H, 512, device=DEV), workspace=ws)
            check_range(c, out, lse, [0])
    assert _status() == 0


@pytest.mark.parametrize("scales", [(0, -6, -8, -14), (-8, 0, 0, -6), (3, -3, -11, 0)])
@pytest.mark.parametrize("H", [1, 8, 16])
def test_groups_of_uneven_scales(H, scales):
    """A group keeps its precision whatever the scales of the others."""
    for nats, at in ((0.0, 0), (9.5, 1000)):
        c = range_case(31 + H, H, nats, at, k=1500, scales=scales)
        out, lse = run_attend(c, ctx=torch.empty(1, H, 512, device=DEV), workspace=(1, None))
        check_range(c, out, lse, [0])
    assert _status() == 0


def test_tail_in_items_behind_the_last_full_wave():
    """Whole items and items cut into runs in one call, the default result type."""
    n = torch.cuda.get_device_properties(0).multi_processor_count + 3
    c = range_case(77, 16, 10.0, 600, k=700, items=n)
    out, lse = run_attend(c, workspace=(-3, torch.empty(3 * 3 * 16 * 513, device=DEV)))
    assert _status() == 0
    check_range(c, out, lse, [0, 1, n - 4, n - 3, n - 1])


@pytest.mark.parametrize("ratio,nats", [(8, 12.0), (14, 12.0), (14, 30.0), (30, 30.0), (40, 60.0)])
@pytest.mark.parametrize("H", [1, 16])
def test_a_key_of_large_scales_and_no_weight(H, ratio, nats):
    """A key whose scales are 2^ratio times the others' but whose probability is e^-nats of theirs: its latent dims and the
    queries' do not meet, so that its score is the position dims' alone."""
    for at in (0, 700, 1499):
        c = range_case(90 + H + at, H, 2.0, (at + 5) % 1500, k=1500)
        lone = int(c["idx"][0, at])
        row = c["cache"][lone]
        row[512:528] = torch.full((4,), 2.0 ** (ratio - 7)).view(torch.uint8)
        row[:512:2] = 0                                           # the odd latent dims hold its values,
        c["q"][:, :, 1:512:2] = 0                                 # the even ones the queries'
        row[528:] = 0
        row[528:530] = torch.tensor([-nats], dtype=torch.bfloat16).view(torch.uint8)
        for splits in (1, 4):
            ws = (splits, torch.empty(splits * H * 513, device=DEV) if splits > 1 else None)
            out, lse = run_attend(c, ctx=torch.empty(1, H, 512, device=DEV), workspace=ws)
            check_range(c, out, lse, [0], query=0)
    assert _status() == 0


@pytest.mark.parametrize("H", [3, 16])
def test_scores_and_scales_that_grow_in_turn(H):
    """Tile by tile the score, or one group's scale by any factor, takes the lead: references of heads and groups are renewed
    at different times; then the same keys in falling order."""
    g = torch.Generator().manual_seed(H)
    k = 1280
    c = range_case(5 + H, H, 0.0, 0, k=k)
    tile = torch.arange(k) // 128
    up = torch.stack([tile * 3 % 7 - 9, tile - 12, -2 * tile, (tile % 2) * 9 - 14], 1).float()
    c["cache"][:k, 512:528] = torch.exp2(up).view(torch.uint8)
    pe = torch.zeros(k, 64)
    pe[:, 0] = tile * 1.5 + torch.rand(k, generator=g)
    pe[:, 1] = -tile.float()                                      # for the heads that look there scores fall
    c["cache"][:k, 528:] = pe.bfloat16().view(torch.uint8)
    c["q"][:, 1::2, 512], c["q"][:, 1::2, 513] = 0, 16
    c["qpos"][:] = k
    for order in (torch.arange(k), torch.arange(k).flip(0)):
        c["idx"] = order.to(torch.int32).view(1, -1)
        out, lse = run_attend(c, ctx=torch.empty(1, H, 512, device=DEV), workspace=(1, None))
        check_range(c, out, lse, [0])
    assert _status() == 0


def test_scales_of_zero_and_of_the_smallest_numbers():
    """Rows of zeros (a cache that nobody wrote), a group of tiny scales beside ordinary ones."""
    c = range_case(8, 16, 3.0, 40, k=300)
    c["cache"][:150] = 0
    c["cache"][200:, 512:516] = torch.tensor([2.0 ** -126]).view(torch.uint8)
    out, lse = run_attend(c, ctx=torch.empty(1, 16, 512, device=DEV), workspace=(1, None))
    check_range(c, out, lse, [0])
    c["cache"][:300] = 0                                          # nothing but zeros: scores 0, the mean of zeros
    out, lse = run_attend(c)
    assert _status() == 0 and bool((out == 0).all())
    assert bool(((lse.cpu() - torch.log(torch.tensor(300.0))).abs() < 1e-5).all())


@pytest.mark.parametrize("H", [1, 16, 17])
@pytest.mark.parametrize("top", [64.0, 4096.0])
def test_queries_with_one_large_dim(H, top):
    """A query dim far above the others that meets nothing in the cache takes no precision from them: values of 1.75 * 2^-18 of
    it, which two terms hold exactly (the row's power of two makes 256 and 1.75 * 2^-10 of them, and the second term, 16 times
    that, is a normal number)."""
    c = range_case(3 + H, H, 2.0, 9, k=600)
    c["q"][:, :, :512] = 1.75 * 2.0 ** -18 * top
    c["q"][:, :, 5:512:128] = top
    c["cache"][:, 5:512:128] = 0
    out, lse = run_attend(c, ctx=torch.empty(1, H, 512, device=DEV), workspace=(1, None))
    check_range(c, out, lse, [0], query=0)
    assert _status() == 0


@pytest.mark.parametrize("H", [2, 16])
def test_plain_scales_over_a_broad_tail(H):
    """Scales that are no powers of two: up to 16 heads no row is widened, so nothing more is rounded."""
    g = torch.Generator().manual_seed(50 + H)
    for nats, at in ((10.0, 3), (12.0, 1020)):
        c = range_case(60 + H, H, nats, at, k=1024, scales=(0, -3, 2, -9))
        sc = c["cache"][:, 512:528].contiguous().view(torch.float32) * (1 + torch.rand(1024, 4, generator=g))
        c["cache"][:, 512:528] = sc.view(torch.uint8)
        out, lse = run_attend(c, ctx=torch.empty(1, H, 512, device=DEV), workspace=(1, None))
        check_range(c, out, lse, [0])
    assert _status() == 0


def test_a_committed_key_over_a_tree_and_a_drafted_one_over_the_selection():
    """The drafted tokens are one more tile: a key that dominates from either side of it."""
    for at in (10, 600):                                          # 600: the first drafted position
        c = range_case(70 + at, 16, 11.0, 0, k=608)
        pe = torch.rand(608, 1, generator=torch.Generator().manual_seed(at))
        pe[at] = 11.5
        c["cache"][:608, 528:530] = pe.bfloat16().view(torch.uint8)
        sel = torch.arange(600).flip(0).to(torch.int32).view(1, -1)
        d = dict(c, idx=sel, lens=torch.tensor([600], dtype=torch.int32), mask=torch.tensor([0b10110101]))
        out, lse = run_attend(d, ctx=torch.empty(1, 16, 512, device=DEV), workspace=(1, None))
        flat = dict(c, idx=torch.cat([sel, torch.tensor([[600, 602, 604, 605, 607]], dtype=torch.int32)], 1))
        check_range(flat, out, lse, [0])
    assert _status() == 0
