"""The 8-bit path where the framework uses it: the decode step over the quantised latent cache (eager, captured,
replayed), a verification pass over drafted trees, and the indexer's projections in 8 bits."""
import pytest
import torch

from oracle import dsa_oracle as O
from oracle import latent_oracle as L
from tests.decode_cases import make_global_problem, shard_state
from tests.test_gpu_latent_cache import attend_case, check_attend, run_attend

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _latent_pages(prob, page):
    """The problem's latents written into a quantised cache: (cache, block table)."""
    from transarch_b200 import kernels as K
    each = max((c + page - 1) // page for c in prob["ctxs"])
    B = len(prob["ctxs"])
    table = torch.randperm(B * each, generator=torch.Generator().manual_seed(3)).view(B, each).to(torch.int32)
    cache = torch.zeros(B * each, page * 656, dtype=torch.uint8, device=DEV)
    for b, kv in enumerate(prob["kv"]):
        p = torch.arange(kv.shape[0])
        slots = table[b, p // page].long() * page + p % page
        K.latent_quant_and_cache(kv.to(DEV), cache, slots.to(DEV), page)
    return cache, table


def test_decode_step_over_the_quantised_cache():
    from transarch_b200 import _lib
    from transarch_b200.decode import GraphedDecodeStep, SparseDecodeStep
    prob, topk, page = make_global_problem(17, [1500, 700, 64]), 256, 32
    st = shard_state(prob, 0, 1, 1500, DEV)
    cache, table = _latent_pages(prob, page)

    def check(idx, ctx, lse):
        c = {"q": prob["q_lat"], "idx": idx.cpu(), "req": torch.arange(3), "lens": st["lens"].cpu(),
             "qpos": st["lens"].cpu() - 1, "mask": None, "table": table, "page": page,
             "cache": cache.cpu().view(-1, 656), "scale": 192 ** -0.5}
        check_attend(c, ctx, lse)

    for dtype in (torch.bfloat16, torch.float32):
        step = SparseDecodeStep(3, st["table"].shape[1] * 64, topk=topk, device=torch.device(DEV, 0), ctx_dtype=dtype,
                                latent_page_size=page, sorted_topk=True)
        args = (st["cache"], st["lens"], st["table"], cache, table.to(DEV))
        q = (prob["q_idx"].to(DEV), prob["w"].to(DEV), prob["q_lat"].to(DEV))
        idx, ctx, lse = step.run(*q, *args)
        assert ctx.dtype == dtype and _lib.read_status(ctx.device) == 0
        check(idx, ctx, lse)
        eager = (idx.clone(), ctx.clone(), lse.clone())
        graphed = GraphedDecodeStep(step, *args).capture()
        out = graphed.replay(*q)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
    # the selection does not depend on the latent cache
    plain = SparseDecodeStep(3, st["table"].shape[1] * 64, topk=topk, device=torch.device(DEV, 0), sorted_topk=True)
    ref_idx, ref_ctx, _ = plain.run(*q, st["cache"], st["lens"], st["table"], st["kv"], st["base"])
    assert torch.equal(ref_idx, eager[0])
    # and the attention differs from the bf16 cache's by the quantisation alone: each latent by at most 2^-4 of itself
    for b in range(3):
        rows = prob["kv"][b][ref_idx[b][ref_idx[b] >= 0].cpu().long()].double()
        _, _, mass, qk = L.attend(prob["q_lat"][b], rows, 192 ** -0.5)
        moved = 2.0 ** -4 * mass * 1.1 + 4 * 2.0 ** -4 * qk.view(-1, 1) * mass
        assert bool(((eager[1][b].double().cpu() - ref_ctx[b].double().cpu()).abs() <= moved).all())
    assert _lib.read_status(torch.device(DEV)) == 0


def test_drafted_tree_written_and_verified():
    """A speculative step: drafted tokens written behind the committed ones, masks from their parents, one attention
    over selection and tree; a chain (each node the child of the one before) equals ordinary causal queries."""
    from transarch_b200 import _lib, kernels as K
    R, n, page, H = 3, 6, 16, 32
    c = attend_case(51, R, n, H, 120, 200, page, drafts=n)
    g = torch.Generator().manual_seed(52)
    drafts = torch.randn(R * n, 576, generator=g).bfloat16()
    parents = torch.arange(-1, n - 1, dtype=torch.int32).repeat(R, 1)
    pos = c["lens"].repeat_interleave(n).long() + torch.arange(n).repeat(R)
    req = c["req"].long()
    slots = c["table"][req, pos // page].long() * page + pos % page
    cache = c["cache"].to(DEV)
    K.latent_quant_and_cache(drafts.to(DEV), cache, slots.to(DEV), page)
    c["cache"] = cache.cpu()
    masks = K.draft_tree_masks(parents.to(DEV))
    assert masks.cpu().tolist() == [[2 ** (j + 1) - 1 for j in range(n)]] * R
    c["mask"] = masks.cpu().view(-1)
    out, lse = run_attend(c)
    check_attend(c, out, lse)
    # the same keys as positions: the selection and the chain's prefix
    flat = dict(c, mask=None)
    own = torch.arange(n).repeat(R, 1).reshape(-1)
    idx = torch.where(c["idx"] < c["lens"][req].view(-1, 1), c["idx"], torch.full_like(c["idx"], -1))
    tail = c["lens"][req].view(-1, 1) + torch.arange(n)
    tail = torch.where(torch.arange(n) <= own.view(-1, 1), tail, torch.full_like(tail, -1)).to(torch.int32)
    flat["idx"] = torch.cat([torch.where(idx <= c["qpos"].view(-1, 1), idx, torch.full_like(idx, -1)), tail], 1).contiguous()
    flat["qpos"] = torch.full((R * n,), 2 ** 30, dtype=torch.int32)
    out2, lse2 = run_attend(flat)
    check_attend(flat, out2, lse2)
    assert _lib.read_status(out.device) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_indexer_projections_in_8_bits(dtype):
    from transarch_b200 import _lib, kernels as K
    from transarch_b200._lib import B200DSAError
    from transarch_b200.indexer_module import LightningIndexer
    g = torch.Generator().manual_seed(33)
    T, hidden, q_in, H, page = 37, 272, 144, 64, 64
    mod = LightningIndexer(hidden, n_heads=H, q_input_dim=q_in, dtype=dtype).to(DEV)
    h = torch.randn(T, hidden, generator=g).to(dtype).to(DEV)
    qi = torch.randn(T, q_in, generator=g).to(dtype).to(DEV)
    ang = torch.rand(T, 32, generator=g) * 6.28
    cos, sin = torch.cat([ang.cos()] * 2, -1).to(DEV), torch.cat([ang.sin()] * 2, -1).to(DEV)
    slots = torch.randperm(2 * page, generator=g)[:T].to(DEV)

    def serve():
        cache = torch.zeros(2, page * 132, dtype=torch.uint8, device=DEV)
        return (*mod.forward_quantised(h, qi, cos, sin, cache, slots, page), cache)

    plain = serve()
    mod.quantise_projections()
    q8, w8, c8 = serve()
    assert _lib.read_status(h.device) == 0
    # exactly the fused tails on the block-scaled products ...
    q = K.fp8_block_linear(qi, *K.fp8_quantise_blocks(mod.wq.weight.detach()), out_dtype=dtype)
    q_ref, w_ref = K.indexer_q_rope(q.view(T, H, 128), cos, sin, rope_first=True, want_rows=False, w=mod.w_proj(h),
                                    fold=mod.softmax_scale * H ** -0.5, ue8m0=True)
    assert torch.equal(q8.view(torch.uint8), q_ref.view(torch.uint8)) and torch.equal(w8, w_ref)
    # ... whose operands are off by at most 2^-4 each
    exact = qi.double().cpu() @ mod.wq.weight.detach().double().cpu().t()
    mass = qi.double().cpu().abs() @ mod.wq.weight.detach().double().cpu().abs().t()
    assert bool(((q.double().cpu() - exact).abs() <= (2 * 2.0 ** -4 + 2.0 ** -8 + 2.0 ** -7) * mass + 2.0 ** -8 * exact.abs()).all())
    assert not torch.equal(c8, plain[2])
    # stale copies are refused: changed in place, replaced, loaded, cast
    with torch.no_grad():
        mod.wk.weight.mul_(2.0)
    with pytest.raises(B200DSAError, match="wk has changed"):
        serve()
    mod.quantise_projections("ue8m0")
    serve()
    mod.load_state_dict({k: v.clone() for k, v in mod.state_dict().items()})
    with pytest.raises(B200DSAError, match="changed"):
        serve()
    mod.quantise_projections()
    mod.wq.weight = torch.nn.Parameter(mod.wq.weight.detach().clone())
    with pytest.raises(B200DSAError, match="wq has changed"):
        serve()
    assert set(mod.state_dict()) == {"wq.weight", "wk.weight", "k_norm.weight", "k_norm.bias", "w_proj.weight"}
    # the training-side forward keeps its parameters
    mod.quantise_projections()
    c4 = cos.view(1, T, 64), sin.view(1, T, 64)
    a = mod(h.view(1, T, -1), qi.view(1, T, -1), *c4)
    mod._fp8 = {}
    b = mod(h.view(1, T, -1), qi.view(1, T, -1), *c4)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_indexer_projections_of_a_module_made_for_inference():
    """Parameters made under inference_mode carry no version counter."""
    from transarch_b200.indexer_module import LightningIndexer
    g = torch.Generator().manual_seed(34)
    T, hidden, H, page = 5, 144, 8, 64
    h = torch.randn(T, hidden, generator=g).bfloat16().to(DEV)
    cos, sin = torch.ones(T, 64, device=DEV), torch.zeros(T, 64, device=DEV)
    slots = torch.arange(T, device=DEV)
    outs = []
    for inference in (False, True):
        torch.manual_seed(35)
        with torch.inference_mode(inference):
            mod = LightningIndexer(hidden, n_heads=H).to(DEV)
            mod.quantise_projections()
            cache = torch.zeros(1, page * 132, dtype=torch.uint8, device=DEV)
            q, w = mod.forward_quantised(h, h, cos, sin, cache, slots, page)
            outs.append((q.view(torch.uint8).clone(), w.clone(), cache))
    for x, y in zip(*outs):
        assert torch.equal(x.cpu(), y.cpu())
