"""Quantised latent cache: written, read back, and attended (also by trees of drafted tokens), against 64-bit
definitions.  Bounds are derived: a stored or returned number is off by half a step of its type, a product of bf16
probabilities by 2^-8 of the mass it sums, fp32 sums by their length times 2^-24."""
import pytest
import torch

from oracle import latent_oracle as L

pytestmark = pytest.mark.gpu

E4M3, BF16, F32 = 2.0 ** -4, 2.0 ** -8, 2.0 ** -24
DEV = "cuda"


def _status():
    from transarch_b200 import _lib
    return _lib.read_status(torch.device(DEV))


def random_cache(slots, g, pow2=True):
    sc = torch.exp2(torch.randint(-9, -6, (slots, 4), generator=g).float())
    if not pow2:
        sc = sc * (1 + torch.rand(slots, 4, generator=g))
    codes = (torch.randn(slots, 512, generator=g) * 110).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    pe = (0.5 * torch.randn(slots, 64, generator=g)).bfloat16().view(torch.uint8)
    return torch.cat([codes, sc.view(torch.uint8), pe], 1)


def check_written(cache, slots, n, r):
    """Rows of the cache against the 64-bit latent n and position dims r."""
    v = L.cache_rows(cache, slots)
    sc = L.cache_scales(cache, slots).double().repeat_interleave(128, 1)
    assert bool(((v[:, :512] - n).abs() <= E4M3 * n.abs() * (1 + 1e-5) + sc * 2.0 ** -10 + 1e-6 * n.abs()).all())
    # fp32 products of the rotation: two roundings of terms no larger than the pair's norm
    size = torch.sqrt((r * r).sum(1, keepdim=True))
    assert bool(((v[:, 512:] - r).abs() <= BF16 * r.abs() + 4 * F32 * size + 2.0 ** -133).all())
    return sc


@pytest.mark.parametrize("n,width,f32,norm,rope,offset", [
    (1, 576, False, True, "pairs", 0), (5, 576, True, True, "half", 0), (64, 2112, False, True, "pairs", 1536),
    (33, 700, False, False, "half", 13), (130, 600, True, True, None, 24), (7, 577, True, False, "pairs", 1)])
def test_write(n, width, f32, norm, rope, offset):
    """All forms, rows aligned and not, padding tokens; rows of other slots stay as they were."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(n + width)
    page, pages = 16, n // 16 + 3
    before = random_cache(pages * page, g)
    raw = torch.randn(n, width, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))
    raw = raw if f32 else raw.bfloat16()
    kv = raw[:, offset:offset + 576]
    slots = torch.randperm(pages * page, generator=g)[:n]
    if n > 4:
        slots[2] = -1
    gain = torch.randn(512, generator=g).to(torch.float32 if f32 else torch.bfloat16) if norm else None
    pos = torch.randint(0, 160000, (n, 1), generator=g).double()
    a = pos * 10000.0 ** (-torch.arange(32).double() / 32)
    a = torch.cat([a, a], 1)
    cos, sin = (a.cos().float(), a.sin().float()) if rope else (None, None)
    cache = before.clone().to(DEV).view(pages, page * 656)
    on = lambda t: None if t is None else t.to(DEV)
    K.latent_quant_and_cache(raw.to(DEV)[:, offset:offset + 576], cache, slots.to(DEV), page, norm_weight=on(gain),
                             eps=1e-5, cos=on(cos), sin=on(sin), interleaved=rope == "pairs")
    assert _status() == 0
    after = cache.cpu().view(-1, 656)
    live = slots[slots >= 0]
    other = torch.ones(pages * page, dtype=torch.bool)
    other[live] = False
    assert torch.equal(after[other], before[other])
    nn, rr = L.norm_rotate(kv, gain, 1e-5, cos, sin, rope == "pairs")
    keep = slots >= 0
    sc = check_written(after, live, nn[keep], rr[keep])[:, ::128]
    # power-of-two scales, the smallest that holds the group's largest value (fp32 arithmetic: 2^-20 either way)
    top = nn[keep].view(-1, 4, 128).abs().amax(2).clamp_min(1e-4) / 448
    assert torch.equal(torch.exp2(torch.log2(sc).round()), sc)
    assert bool((sc >= top * (1 - 2.0 ** -20)).all()) and bool((sc < 2 * top * (1 + 2.0 ** -20)).all())


def test_write_plain_scales_and_specials():
    """scale_fmt None; a row of zeros, tiny and huge rows, NaN and infinity, a slot behind the cache."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(3)
    kv = torch.randn(8, 576, generator=g)
    kv[1] = 0
    kv[2] *= 1e-30
    kv[3] *= 1e30
    kv[4, 7] = float("nan")
    kv[5, 200] = float("inf")
    slots = torch.tensor([9, 0, 3, 8, 5, 15, 16, 1])
    cache = random_cache(16, g).to(DEV)
    before = cache.cpu().clone()
    K.latent_quant_and_cache(kv.to(DEV), cache, slots.to(DEV), 16, scale_fmt=None)
    assert _status() == 2                                      # slot 16 does not exist
    after = cache.cpu()
    fine = [0, 1, 2, 3, 7]
    check_written(after, slots[fine], kv[fine, :512].double(), kv[fine, 512:].double())
    sc = L.cache_scales(after, slots[[0, 7]]).double()
    top = kv[[0, 7], :512].double().view(2, 4, 128).abs().amax(2) / 448
    assert bool(((sc - top).abs() <= F32 * top * 2).all())
    v = L.cache_rows(after, slots[[4, 5]])
    assert bool(torch.isnan(v[0, 7])) and bool(torch.isfinite(v[0, 128:512]).all())
    assert bool(torch.isnan(v[1, 200])) and bool(torch.isfinite(v[1, :128]).all())
    untouched = [s for s in range(16) if s not in slots.tolist()]
    assert torch.equal(after[untouched], before[untouched])


@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("pow2", [True, False])
def test_rows_read_back(n, pow2):
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(n)
    cache = random_cache(96, g, pow2)
    slots = torch.randint(0, 96, (n,), generator=g)            # the same slot may be read twice
    slots[0] = -1
    out = K.latent_cache_rows(cache.to(DEV), slots.to(DEV), 32).cpu()
    ref = L.cache_rows(cache, slots.clamp_min(0)).float().bfloat16()
    ref[slots < 0] = 0
    assert _status() == 0 and torch.equal(out, ref)
    bad = slots.clone()
    bad[-1] = 96
    out = K.latent_cache_rows(cache.to(DEV), bad.to(DEV), 32).cpu()
    assert _status() == 2 and bool((out[-1] == 0).all()) and torch.equal(out[:-1], ref[:-1])


def test_gather_requests():
    """Ragged requests, an empty one, a page outside the cache, rows behind the last request left alone."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(8)
    page, lens = 16, [33, 0, 1, 16, 50] + [3] * 40
    each = 4
    pages = len(lens) * each
    cache = random_cache(pages * page, g)
    table = torch.randperm(pages, generator=g).view(len(lens), each).to(torch.int32)
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lens).cumsum(0)
    total = int(cu[-1])
    refs = []
    for r, n in enumerate(lens):
        p = torch.arange(n)
        refs.append(L.cache_rows(cache, table[r, p // page].long() * page + p % page).float().bfloat16())
    ref = torch.cat(refs)
    out = torch.full((total + 5, 576), 7.0, dtype=torch.bfloat16, device=DEV)
    K.latent_cache_gather(cache.to(DEV), page, table.to(DEV), cu.to(DEV), total + 5, out=out)
    assert _status() == 0
    assert torch.equal(out[:total].cpu(), ref) and bool((out[total:] == 7).all())
    # a wider table's slice as the block table; a page that does not exist
    wide = torch.cat([table, torch.full((len(lens), 3), -5, dtype=torch.int32)], 1).to(DEV)
    wide[4, 1] = pages
    out = K.latent_cache_gather(cache.to(DEV), page, wide[:, :each], cu.to(DEV), total).cpu()
    assert _status() == 2
    hole = slice(int(cu[4]) + 16, int(cu[4]) + 32)
    ref[hole] = 0
    assert torch.equal(out, ref)


def _tree(n, g):
    parents = torch.full((n,), -1, dtype=torch.int32)
    for j in range(1, n):
        parents[j] = int(torch.randint(-1, j, (1,), generator=g))
    return parents


@pytest.mark.parametrize("trees,nodes", [(1, 1), (3, 7), (5, 64)])
def test_tree_masks(trees, nodes):
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(nodes)
    parents = torch.stack([_tree(nodes, g) for _ in range(trees)])
    ref = torch.zeros(trees, nodes, dtype=torch.int64)
    for r in range(trees):
        for j in range(nodes):
            at = j
            while at >= 0:
                ref[r, j] |= (1 << at) if at < 63 else -(1 << 63)
                at = int(parents[r, at])
    assert torch.equal(K.draft_tree_masks(parents.to(DEV)).cpu(), ref) and _status() == 0
    if nodes > 2:
        parents[0, 1] = 2                                      # a child before its parent: reported, the path ends
        m = K.draft_tree_masks(parents.to(DEV)).cpu()
        assert _status() == 2 and int(m[0, 1]) == 2


def attend_case(seed, requests, per, H, k, ctx, page, drafts=0, holes=True, pow2=True):
    g = torch.Generator().manual_seed(seed)
    each = (ctx + drafts + page - 1) // page
    pages = requests * each + 1
    c = {"cache": random_cache(pages * page, g, pow2), "page": page, "scale": 192 ** -0.5,
         "table": (torch.randperm(pages - 1, generator=g) + 1)[:requests * each].view(requests, each).to(torch.int32),
         "q": torch.randn(requests * per, H, 576, generator=g).bfloat16(),
         "req": torch.arange(requests, dtype=torch.int32).repeat_interleave(per),
         "lens": torch.randint(1, ctx + 1, (requests,), generator=g).to(torch.int32)}
    idx = torch.full((requests * per, k), -1, dtype=torch.int32)
    for i in range(requests * per):
        pick = torch.randperm(ctx, generator=g)[:k].to(torch.int32)
        idx[i, :pick.numel()] = pick
    if holes:
        idx[:, 3::7] = -1
    c["idx"] = idx
    c["qpos"] = c["lens"][c["req"].long()] - 1 - torch.arange(per, dtype=torch.int32).repeat(requests) * (drafts == 0)
    c["mask"] = None
    if drafts:
        masks = torch.zeros(requests * per, dtype=torch.int64)
        for r in range(requests):
            parents = _tree(drafts, g)
            for j in range(per):
                at = j % drafts
                while at >= 0:
                    masks[r * per + j] |= (1 << at) if at < 63 else -(1 << 63)
                    at = int(parents[at])
        c["mask"] = masks
    return c


def run_attend(c, **kw):
    from transarch_b200 import kernels as K
    d = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    return K.sparse_mla_decode_cached(d["q"], d["cache"], d["page"], d["idx"], d["scale"], block_table=d["table"],
                                      row_request=d["req"], q_pos=d["qpos"], tree_mask=d["mask"],
                                      tree_base=d["lens"] if d["mask"] is not None else None, **kw)


def check_attend(c, ctx, lse, items=None, limit=None, pow2=True):
    n, H, _ = c["q"].shape
    widen = 0.0 if pow2 else BF16                             # a plain scale rounds the widened row once
    for i in items if items is not None else range(n):
        r = int(c["req"][i])
        idx = c["idx"][i] if limit is None else c["idx"][i, :max(0, int(limit[i]))]
        base = int(c["lens"][r]) if c["mask"] is not None else None
        slots = L.item_keys(idx, c["table"][r], c["page"], int(c["qpos"][i]), base,
                            None if c["mask"] is None else int(c["mask"][i]))
        ref, ref_lse, mass, qk = L.attend(c["q"][i], L.cache_rows(c["cache"], slots), c["scale"])
        k = max(1, slots.numel())
        d = (576 * F32 + widen) * qk.view(-1, 1) + 1e-6       # error of a score; exp of it is relative
        step = BF16 if ctx.dtype == torch.bfloat16 else F32
        bound = (BF16 + widen + 2 * d + k * F32) * mass + step * ref.abs() + 1e-30
        got = ctx[i].double().cpu()
        assert bool(((got - ref).abs() <= bound).all()), (i, float(((got - ref).abs() / bound).max()))
        got_lse = lse[i].double().cpu()
        if slots.numel() == 0:
            assert bool((got == 0).all()) and bool((got_lse == float("-inf")).all())
        else:
            lim = d.view(-1) + k * F32 + 8 * F32 * ref_lse.abs() + 2e-7
            assert bool(((got_lse - ref_lse).abs() <= lim).all()), (i, float(((got_lse - ref_lse).abs() / lim).max()))


@pytest.mark.parametrize("requests,per,H,k,ctx,page", [
    (1, 1, 128, 1, 5, 16), (1, 1, 128, 2048, 4000, 64), (3, 1, 64, 64, 200, 16), (2, 3, 16, 100, 300, 32),
    (5, 1, 1, 33, 50, 16), (40, 2, 128, 65, 130, 64), (2, 1, 65, 700, 900, 128), (160, 1, 128, 200, 400, 16)])
def test_attend(requests, per, H, k, ctx, page):
    c = attend_case(requests + k, requests, per, H, k, ctx, page)
    out, lse = run_attend(c)
    assert _status() == 0 and out.dtype == torch.bfloat16
    check_attend(c, out, lse, items=range(0, requests * per, max(1, requests * per // 8)))


@pytest.mark.parametrize("requests,nodes,H,k", [(1, 1, 128, 64), (2, 24, 16, 300), (3, 64, 128, 40), (2, 5, 64, 0)])
def test_attend_tree(requests, nodes, H, k):
    c = attend_case(nodes + k, requests, nodes, H, k, 400, 32, drafts=nodes)
    out, lse = run_attend(c)
    assert _status() == 0
    check_attend(c, out, lse, items=range(0, requests * nodes, max(1, requests * nodes // 10)))


@pytest.mark.parametrize("splits", [1, 2, 5, 32])
def test_attend_splits_and_fp32(splits):
    """Every number of splits gives the same attention; runs without a single key among them; fp32 result."""
    from transarch_b200 import kernels as K
    c = attend_case(11, 2, 2, 128, 1000, 1500, 64)
    c["idx"][1, 64:640] = -1                                  # whole tiles without a key
    c["idx"][2] = -1                                          # an item without keys
    ws = (splits, torch.empty(splits * 4 * 128 * 513, device=DEV))
    out32 = torch.empty(4, 128, 512, device=DEV)
    out, lse = run_attend(c, ctx=out32, workspace=ws)
    assert _status() == 0 and out.dtype == torch.float32
    check_attend(c, out, lse)
    out16, lse16 = run_attend(c, workspace=ws)
    assert torch.equal(out16, out.bfloat16()) and torch.equal(lse16, lse)


def test_attend_lengths_per_item():
    """n_idx_item: only the first entries of a list count, none at all for a negative length."""
    c = attend_case(12, 4, 1, 32, 300, 400, 16)
    limit = torch.tensor([0, 1, 150, 999], dtype=torch.int32)
    out, lse = run_attend(c, n_idx_item=limit.to(DEV))
    assert _status() == 0
    check_attend(c, out, lse, limit=limit)
    limit[0] = -3
    out2, lse2 = run_attend(c, n_idx_item=limit.to(DEV))
    assert torch.equal(out2, out) and torch.equal(lse2, lse)


def test_attend_plain_scales():
    """Scales that are no powers of two: the widened row is rounded to bf16 once."""
    c = attend_case(13, 2, 1, 128, 500, 900, 64, pow2=False)
    out, lse = run_attend(c)
    assert _status() == 0
    check_attend(c, out, lse, pow2=False)


def test_attend_growing_maximum():
    """Keys whose scores keep growing: the accumulator is rescaled again and again."""
    c = attend_case(14, 1, 1, 128, 512, 512, 64, holes=False)
    c["lens"][:] = 512
    c["qpos"][:] = 511
    sc = torch.exp2(torch.linspace(-10, -4, 512).floor()).view(-1, 1).repeat(1, 4)
    slots = L.item_keys(torch.arange(512), c["table"][0], 64, 511)
    rows = c["cache"].clone()
    rows[slots, 512:528] = sc.contiguous().view(torch.uint8)
    c["cache"], c["scale"] = rows, 0.3
    c["idx"] = torch.arange(512, dtype=torch.int32).view(1, -1)
    out, lse = run_attend(c)
    assert _status() == 0
    check_attend(c, out, lse)
    one = (1, None)                                           # and without splitting, where one CTA sees them all
    out, lse = run_attend(c, workspace=one)
    check_attend(c, out, lse)


def test_attend_masked_places_may_hold_anything():
    """NaN and infinities in rows that no item selects, and behind the mask, do not reach the result."""
    c = attend_case(15, 2, 2, 64, 200, 300, 16, drafts=2)
    used = set()
    for i in range(4):
        r = int(c["req"][i])
        used |= set(L.item_keys(c["idx"][i], c["table"][r], 16, int(c["qpos"][i]), int(c["lens"][r]), int(c["mask"][i])).tolist())
    rest = [s for s in range(c["cache"].shape[0]) if s not in used]
    c["cache"][rest, :512] = 0x7f
    c["cache"][rest, 512:528] = torch.full((1, 4), float("inf")).view(torch.uint8)
    c["cache"][rest, 528:] = torch.full((1, 64), float("nan"), dtype=torch.bfloat16).view(torch.uint8)
    out, lse = run_attend(c)
    assert _status() == 0 and bool(torch.isfinite(out).all())
    check_attend(c, out, lse)


def test_attend_bad_pages_and_requests():
    """A page outside the cache, a position outside the table and a request that does not exist: left out, reported."""
    c = attend_case(16, 3, 1, 32, 100, 200, 16, holes=False)
    c["lens"][:] = 200
    c["qpos"][:] = 2 ** 30
    pages = c["cache"].shape[0] // 16
    bad = dict(c, table=c["table"].clone(), idx=c["idx"].clone(), req=c["req"].clone())
    bad["table"][0, 2] = pages
    bad["table"][0, 4] = -1
    bad["idx"][1, 5] = 4000                                    # beyond the table
    bad["req"][2] = 3
    out, lse = run_attend(bad)
    assert _status() == 2
    good = dict(c, idx=c["idx"].clone())
    lost = (good["idx"][0] // 16 == 2) | (good["idx"][0] // 16 == 4)
    good["idx"][0][lost] = -1
    good["idx"][1, 5] = -1
    good["idx"][2] = -1
    check_attend(good, out, lse)


def test_cache_written_attended_and_read_in_one_stream():
    """As a decode step uses it: new tokens written, then attended and read back, captured in a graph and replayed on
    new inputs; another stream gives the same; two captured graphs do not share a workspace."""
    from transarch_b200 import kernels as K
    g = torch.Generator().manual_seed(21)
    B, H, page, ctx = 4, 128, 64, 700
    each = (ctx + page) // page
    cache = random_cache(B * each * page, g).to(DEV)
    table = torch.arange(B * each, dtype=torch.int32).view(B, each).to(DEV)
    lens = torch.tensor([700, 1, 333, 64], dtype=torch.int32)
    slots = torch.tensor([(int(table[b, (int(lens[b]) - 1) // page]) * page + (int(lens[b]) - 1) % page) for b in range(B)])
    idx = torch.arange(704, dtype=torch.int32).repeat(B, 1).to(DEV)
    kv = torch.randn(B, 576, generator=g).bfloat16()
    q = torch.randn(B, H, 576, generator=g).bfloat16()
    s_kv, s_q, s_slots, s_lens = kv.to(DEV), q.to(DEV), slots.to(DEV), lens.to(DEV)

    def step():
        K.latent_quant_and_cache(s_kv, cache, s_slots, page)
        out, lse = K.sparse_mla_decode_cached(s_q, cache, page, idx, 0.1, block_table=table, q_pos=s_lens, q_pos_bias=-1)
        return out, lse, K.latent_cache_rows(cache, s_slots, page)

    def verify(out, lse, rows):
        host = cache.cpu()
        c = {"q": q, "idx": idx.cpu(), "req": torch.arange(B), "lens": lens, "qpos": lens - 1, "mask": None,
             "table": table.cpu(), "page": page, "cache": host, "scale": 0.1}
        check_attend(c, out, lse)
        check_written(host, slots, kv[:, :512].double(), kv[:, 512:].double())
        assert torch.equal(rows.cpu(), L.cache_rows(host, slots).float().bfloat16())

    verify(*step())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    verify(*got)
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for turn in range(2):
        kv.copy_(torch.randn(B, 576, generator=g).bfloat16())
        q.copy_(torch.randn(B, H, 576, generator=g).bfloat16())
        s_kv.copy_(kv)
        s_q.copy_(q)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            verify(*outs)
    assert _status() == 0


def test_long_cache_offsets():
    """Slots whose byte offset passes 32 bits (a cache of 6.6 million tokens, 4.3 GB)."""
    from transarch_b200 import kernels as K
    slots_n = 6_600_000 // 64 * 64
    cache = torch.zeros(slots_n, 656, dtype=torch.uint8, device=DEV)
    g = torch.Generator().manual_seed(5)
    kv = torch.randn(70, 576, generator=g).bfloat16()
    slots = slots_n - 1 - torch.arange(70) * 3
    K.latent_quant_and_cache(kv.to(DEV), cache, slots.to(DEV), 64)
    part = cache[slots_n - 512:].cpu()
    local = slots - (slots_n - 512)
    check_written(part, local, kv[:, :512].double(), kv[:, 512:].double())
    rows = K.latent_cache_rows(cache, slots.to(DEV), 64).cpu()
    assert torch.equal(rows, L.cache_rows(part, local).float().bfloat16())
    table = torch.tensor([[slots_n // 64 - 4 + i for i in range(4)]], dtype=torch.int32)
    pos = (slots - (slots_n - 256)).to(torch.int32)
    q = torch.randn(1, 128, 576, generator=g).bfloat16()
    out, lse = K.sparse_mla_decode_cached(q.to(DEV), cache, 64, pos.view(1, -1).to(DEV), 0.05, block_table=table.to(DEV))
    ref, ref_lse, mass, qk = L.attend(q[0], L.cache_rows(part, local), 0.05)
    assert bool(((out[0].double().cpu() - ref).abs() <= (2 * BF16 + 1e-3) * mass + BF16 * ref.abs()).all())
    assert _status() == 0


# ------------------------------------------------------------------------------------------------------------------
# up to 16 heads: codes multiplied as they are, queries and probabilities as two e4m3 numbers
# ------------------------------------------------------------------------------------------------------------------
def check_few(c, ctx, lse, items=None, limit=None):
    """check_attend with what two e4m3 numbers add: a query value is off by at most 2^-18 of its row's largest, and a
    probability by 2^-14 (half of e4m3's smallest step, of 16 p), times the largest scale over the key's own."""
    n, H, _ = c["q"].shape
    for i in items if items is not None else range(n):
        r = int(c["req"][i])
        idx = c["idx"][i] if limit is None else c["idx"][i, :max(0, int(limit[i]))]
        base = int(c["lens"][r]) if c["mask"] is not None else None
        slots = L.item_keys(idx, c["table"][r], c["page"], int(c["qpos"][i]), base,
                            None if c["mask"] is None else int(c["mask"][i]))
        rows = L.cache_rows(c["cache"], slots)
        ref, ref_lse, mass, qk = L.attend(c["q"][i], rows, c["scale"])
        if slots.numel() == 0:
            assert bool((ctx[i] == 0).all()) and bool((lse[i] == float("-inf")).all())
            continue
        k = slots.numel()
        sc = L.cache_scales(c["cache"], slots).double().repeat_interleave(128, 1)
        loose = (rows[:, :512].abs() / sc * sc.max()).sum(0)                       # sum |code| * largest scale
        top = torch.exp((c["q"][i].double() @ rows.t() * c["scale"]).amax(1) - ref_lse).view(-1, 1)
        q_off = 2.0 ** -18 * c["q"][i].double().abs().amax(1) * rows.abs().sum(1).max() * c["scale"]
        d = (576 * F32 * qk + q_off).view(-1, 1) + 1e-6
        step = BF16 if ctx.dtype == torch.bfloat16 else F32
        bound = (BF16 + 2 * d + k * F32) * mass + 2.0 ** -14 * loose * top + step * ref.abs() + 1e-30
        got = ctx[i].double().cpu()
        assert bool(((got - ref).abs() <= bound).all()), (i, float(((got - ref).abs() / bound).max()))
        lim = d.view(-1) + k * F32 + 8 * F32 * ref_lse.abs() + 2e-7
        assert bool(((lse[i].double().cpu() - ref_lse).abs() <= lim).all())


@pytest.mark.parametrize("requests,per,H,k,ctx,page", [
    (1, 1, 16, 1, 5, 16), (1, 1, 9, 2048, 4000, 64), (3, 2, 8, 128, 300, 16), (2, 1, 16, 129, 400, 32), (200, 1, 1, 300, 500, 64)])
def test_few_heads(requests, per, H, k, ctx, page):
    c = attend_case(requests + k, requests, per, H, k, ctx, page)
    out, lse = run_attend(c)
    assert _status() == 0
    check_few(c, out, lse, items=range(0, requests * per, max(1, requests * per // 8)))


@pytest.mark.parametrize("splits", [1, 3, 16])
def test_few_heads_splits_fp32_and_lengths(splits):
    c = attend_case(61, 2, 3, 12, 900, 1200, 32)
    c["idx"][1, 128:640] = -1                                  # whole tiles without a key
    c["idx"][2] = -1                                           # an item without keys
    limit = torch.tensor([900, 900, 900, 0, 1, 300], dtype=torch.int32)
    ws = (splits, torch.empty(splits * 6 * 12 * 513, device=DEV))
    out, lse = run_attend(c, ctx=torch.empty(6, 12, 512, device=DEV), workspace=ws, n_idx_item=limit.to(DEV))
    assert _status() == 0
    check_few(c, out, lse, limit=limit)
    out16, lse16 = run_attend(c, workspace=ws, n_idx_item=limit.to(DEV))
    assert torch.equal(out16, out.bfloat16()) and torch.equal(lse16, lse)


def test_few_heads_growing_scores_and_scales():
    """Scores and scales that grow from tile to tile: both references are renewed, the accumulators rescaled."""
    c = attend_case(62, 1, 1, 16, 640, 640, 64, holes=False)
    c["lens"][:], c["qpos"][:] = 640, 639
    sc = torch.exp2(torch.linspace(-12, -3, 640).floor()).view(-1, 1).repeat(1, 4)
    slots = L.item_keys(torch.arange(640), c["table"][0], 64, 639)
    c["cache"] = c["cache"].clone()
    c["cache"][slots, 512:528] = sc.contiguous().view(torch.uint8)
    c["scale"], c["idx"] = 0.3, torch.arange(640, dtype=torch.int32).view(1, -1)
    for ws in (None, (1, None)):
        out, lse = run_attend(c, workspace=ws)
        assert _status() == 0
        check_few(c, out, lse)
    c["idx"] = c["idx"].flip(1).contiguous()                    # and falling ones
    out, lse = run_attend(c, workspace=(1, None))
    check_few(c, out, lse)


def test_few_heads_plain_scales_mixed_sizes_and_foreign_rows():
    """Scales that are no powers of two, differing by group; NaN in rows that nobody selects; a row of NaN that one item
    selects reaches that item alone."""
    c = attend_case(63, 2, 2, 16, 300, 500, 16, pow2=False, drafts=2)
    used = set()
    for i in range(4):
        r = int(c["req"][i])
        used |= set(L.item_keys(c["idx"][i], c["table"][r], 16, int(c["qpos"][i]), int(c["lens"][r]), int(c["mask"][i])).tolist())
    rest = [s for s in range(c["cache"].shape[0]) if s not in used]
    c["cache"][rest, :512] = 0x7f
    c["cache"][rest, 512:528] = torch.full((1, 4), float("nan")).view(torch.uint8)
    c["cache"][rest, 528:] = torch.full((1, 64), float("inf"), dtype=torch.bfloat16).view(torch.uint8)
    out, lse = run_attend(c)
    assert _status() == 0
    check_few(c, out, lse)
    clean = out.clone()
    own = L.item_keys(c["idx"][0], c["table"][0], 16, int(c["qpos"][0]), int(c["lens"][0]), None)
    others = L.item_keys(c["idx"][1], c["table"][0], 16, int(c["qpos"][1]), int(c["lens"][0]), int(c["mask"][1]))
    lone = next(int(s) for s in own if int(s) not in set(others.tolist()))
    c["cache"][lone, 512:516] = torch.full((1,), float("nan")).view(torch.uint8)
    out, lse = run_attend(c)
    assert bool(torch.isnan(out[0]).all()) and torch.equal(out[1:], clean[1:])


@pytest.mark.parametrize("H", [16, 128])
def test_calls_in_flight_on_two_streams(H):
    """Two split calls at once: each has a workspace of its own."""
    cases = [attend_case(70 + i, 2, 1, H, 1500, 2000, 64) for i in range(2)]
    alone = [run_attend(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for c, st in zip(cases, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(run_attend(c))
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, alone[i % 2][0]) and torch.equal(lse, alone[i % 2][1])
    assert _status() == 0


@pytest.mark.parametrize("H", [3, 16, 40, 128])
def test_items_that_share_a_request_equal_calls_of_their_own(H):
    """Many items a request (rows are not prefetched then) against one item a call (they are), bit for bit."""
    c = attend_case(90 + H, 2, 8, H, 700, 900, 32)
    one = (1, None)
    out, lse = run_attend(c, workspace=one)
    assert _status() == 0
    if H <= 16:
        check_few(c, out, lse, items=(0, 7, 15))
    else:
        check_attend(c, out, lse, items=(0, 7, 15))
    for i in range(16):
        alone = dict(c, q=c["q"][i:i + 1], idx=c["idx"][i:i + 1], req=c["req"][i:i + 1], qpos=c["qpos"][i:i + 1])
        got, got_lse = run_attend(alone, workspace=one)
        assert torch.equal(got[0], out[i]) and torch.equal(got_lse[0], lse[i])


def test_few_heads_long_cache_and_missing_rows_among_four():
    """Slots whose byte offset passes 32 bits; of four rows that come in one copy any may be missing, the cache's first and
    last slot among the others."""
    from transarch_b200 import kernels as K
    slots_n, page = 6_600_000 // 64 * 64, 64
    cache = torch.zeros(slots_n, 656, dtype=torch.uint8, device=DEV)
    g = torch.Generator().manual_seed(6)
    own = random_cache(2 * page, g)
    cache[:page] = own[:page].to(DEV)
    cache[slots_n - page:] = own[page:].to(DEV)
    table = torch.tensor([[0, slots_n // page - 1]], dtype=torch.int32)
    n = 16
    idx = torch.stack([torch.randperm(2 * page, generator=g) for _ in range(n)]).to(torch.int32)
    for i in range(n):                             # every pattern of missing rows among four
        for j in range(4):
            if i >> j & 1:
                idx[i, j::4] = -1
    q = torch.randn(n, 16, 576, generator=g).bfloat16()
    out, lse = K.sparse_mla_decode_cached(q.to(DEV), cache, page, idx.to(DEV), 0.05, block_table=table.to(DEV),
                                          row_request=torch.zeros(n, dtype=torch.int32, device=DEV))
    assert _status() == 0
    local = dict(cache=own, page=page, scale=0.05, table=torch.tensor([[0, 1]], dtype=torch.int32), q=q, idx=idx,
                 req=torch.zeros(n, dtype=torch.int32), qpos=torch.full((n,), 2 * page, dtype=torch.int32), mask=None)
    check_few(local, out, lse)


@pytest.mark.parametrize("H,over,own,tree", [(16, 9, True, False), (16, 3, False, True), (8, 0, False, False),
                                             (40, 5, True, False), (128, 3, False, False)])
def test_items_behind_the_last_full_wave_are_cut_into_runs(H, over, own, tree):
    """splits = -3: whole waves of items as splits = 1, the others as splits = 3, bit for bit; `own`: item i is request i."""
    from transarch_b200 import kernels as K
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    whole = sms // 2 if H > 64 else sms
    n = whole + over
    c = attend_case(120 + H + over, n if own else 1, 1 if own else n, H, 400, 600, 32, drafts=7 if tree else 0)
    if not tree:
        c["qpos"].fill_(500)
    if own:
        c["req"] = None
    limit = torch.randint(0, 401, (n,), generator=torch.Generator().manual_seed(H), dtype=torch.int32).to(DEV)
    got = {}
    for splits in (1, 3, -3):
        ws = None if splits == 1 else torch.full((abs(splits) * n * H * 513,), float("nan"), device=DEV)
        got[splits] = run_attend(c, workspace=(splits, ws), n_idx_item=limit)
    assert _status() == 0
    for x, a, b in zip(got[-3], got[1], got[3]):
        assert torch.equal(x[:whole], a[:whole]) and torch.equal(x[whole:], b[whole:])
    # a smaller call takes the same workspace, one that does not hold its runs is refused
    splits, ws = K.sparse_mla_cached_workspace(n, H, 400, DEV, tree=tree)
    small = {k: (v[:5] if k in ("q", "idx", "qpos", "req", "mask") and v is not None else v) for k, v in c.items()}
    out, _ = run_attend(small, workspace=(splits, ws))
    assert out.shape[0] == 5 and bool(torch.isfinite(out).all())
    if over:
        from transarch_b200._lib import B200DSAError
        with pytest.raises(B200DSAError, match="workspace"):
            run_attend(c, workspace=(-3, torch.empty(3 * over * H * 513 - 1, device=DEV)))


def test_plan_of_items_behind_the_last_full_wave():
    """192 items of 16 heads are more than one wave: planned, allocated and captured."""
    from transarch_b200 import kernels as K
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = sms + 44
    splits, ws = K.sparse_mla_cached_workspace(n, 16, 2048, DEV)
    assert splits < -1 and ws.numel() <= -splits * n * 16 * 513
    c = attend_case(140, 2, n // 2, 16, 2048, 2500, 64)
    out, lse = run_attend(c)
    held = run_attend(c, workspace=(splits, ws))
    d = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in c.items()}
    ctx, l2 = torch.zeros_like(out), torch.zeros_like(lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.sparse_mla_decode_cached(d["q"], d["cache"], 64, d["idx"], d["scale"], block_table=d["table"], row_request=d["req"],
                                   q_pos=d["qpos"], ctx=ctx, lse=l2, workspace=(splits, ws))
    for _ in range(2):
        ctx.zero_()
        graph.replay()
        for a, b in ((held[0], out), (ctx, out), (held[1], lse), (l2, lse)):
            assert torch.equal(a, b)
    assert _status() == 0
    check_few(c, out, lse, items=(0, 1, n // 2, n - 1))
