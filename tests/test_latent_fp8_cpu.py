"""What the quantised latent cache, the attention over it and the 8-bit products refuse, before anything is launched:
through the wrappers (CPU tensors: a call that passes every check ends at "need CUDA tensors") and through the C ABI."""
import pytest
import torch

from transarch_b200 import _lib, build, kernels as K
from transarch_b200._lib import B200DSAError

bf16, f32, i32, i64, u8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()
    return _lib.load()


def refuses(match, f, *a, **kw):
    with pytest.raises(B200DSAError, match=match):
        f(*a, **kw)


def test_write():
    z = torch.zeros
    ok = dict(kv=z(3, 576, dtype=bf16), cache=z(4, 16 * 656, dtype=u8), slot_mapping=z(3, dtype=i64), page_size=16)
    call = lambda **kw: K.latent_quant_and_cache(**{**ok, **kw})
    refuses("need CUDA", call)
    refuses("need CUDA", call, kv=z(3, 700, dtype=f32)[:, 50:626], norm_weight=z(512), cos=z(3, 64), sin=z(3, 64, dtype=bf16))
    refuses("kv must be", call, kv=z(3, 575, dtype=bf16))
    refuses("kv must be", call, kv=z(3, 576, dtype=torch.float16))
    refuses("kv must be", call, kv=z(3, 1152, dtype=bf16)[:, ::2])
    refuses("overlap", call, kv=z(1, 576, dtype=bf16).expand(3, 576))
    refuses("slot_mapping", call, slot_mapping=z(3, dtype=i32))
    refuses("slot_mapping", call, slot_mapping=z(2, dtype=i64))
    refuses("cache must be", call, cache=z(4, 16 * 655, dtype=u8))
    refuses("cache must be", call, cache=z(0, 16 * 656, dtype=u8))
    refuses("norm_weight", call, norm_weight=z(511))
    refuses("norm_weight", call, norm_weight=z(512, dtype=torch.float16))
    refuses("cos and sin", call, cos=z(3, 64))
    refuses("cos and sin", call, cos=z(3, 64), sin=z(3, 32))
    refuses("scale_fmt", call, scale_fmt="e8m0")


def test_read():
    z = torch.zeros
    cache = z(4, 16 * 656, dtype=u8)
    refuses("need CUDA", K.latent_cache_rows, cache, z(5, dtype=i64), 16)
    refuses("int64", K.latent_cache_rows, cache, z(5, dtype=i32), 16)
    refuses("out must be", K.latent_cache_rows, cache, z(5, dtype=i64), 16, out=z(4, 576, dtype=bf16))
    refuses("cache must be", K.latent_cache_rows, cache, z(5, dtype=i64), 17)
    table, cu = z(2, 2, dtype=i32), z(3, dtype=i32)
    refuses("need CUDA", K.latent_cache_gather, cache, 16, table, cu, 7)
    refuses("block_table", K.latent_cache_gather, cache, 16, table.long(), cu, 7)
    refuses("block_table", K.latent_cache_gather, cache, 16, z(2, 4, dtype=i32)[:, ::2], cu, 7)
    refuses("cu_rows", K.latent_cache_gather, cache, 16, table, z(2, dtype=i32), 7)
    refuses("negative", K.latent_cache_gather, cache, 16, table, cu, -1)
    refuses("parents", K.draft_tree_masks, z(2, 65, dtype=i32))
    refuses("int32", K.draft_tree_masks, z(2, 6, dtype=i64))


def test_attend():
    z = torch.zeros
    ok = dict(q=z(2, 16, 576, dtype=bf16), cache=z(4, 16 * 656, dtype=u8), page_size=16, indices=z(2, 8, dtype=i32),
              sm_scale=0.1, block_table=z(2, 2, dtype=i32))
    call = lambda **kw: K.sparse_mla_decode_cached(**{**ok, **kw})
    refuses("need CUDA", call)
    refuses("need CUDA", call, indices=z(2, 0, dtype=i32), tree_mask=z(2, dtype=i64), tree_base=z(2, dtype=i32))
    refuses("q must be", call, q=z(2, 129, 576, dtype=bf16))
    refuses("q must be", call, q=z(2, 16, 576))
    refuses("q must be", call, q=z(2, 576, dtype=bf16))
    refuses("q must be", call, q=z(2, 16, 640, dtype=bf16)[..., :576])
    refuses("indices", call, indices=z(3, 8, dtype=i32))
    refuses("indices", call, indices=z(2, 8, dtype=i64))
    refuses("indices", call, indices=z(2, 16, dtype=i32)[:, ::2])
    refuses("block table", call, block_table=z(1, 2, dtype=i32))
    refuses("need CUDA", call, block_table=z(1, 2, dtype=i32), row_request=z(2, dtype=i32))
    refuses("row_request", call, row_request=z(3, dtype=i32))
    refuses("q_pos", call, q_pos=z(2, dtype=i64))
    refuses("n_idx_item", call, n_idx_item=z(1, dtype=i32))
    refuses("tree_base", call, tree_mask=z(2, dtype=i64))
    refuses("tree_mask", call, tree_base=z(2, dtype=i32))
    refuses("tree_mask", call, tree_mask=z(2, dtype=i32), tree_base=z(2, dtype=i32))
    refuses("tree_base", call, tree_mask=z(2, dtype=i64), tree_base=z(3, dtype=i32))
    refuses("ctx must", call, ctx=z(2, 16, 512, dtype=torch.float16))
    refuses("lse must", call, lse=z(2, 16, dtype=bf16))
    refuses("positive", call, sm_scale=0.0)
    refuses("positive", call, sm_scale=float("nan"))


def test_products():
    z = torch.zeros
    refuses("need CUDA", K.fp8_quantise_rows, z(3, 144, dtype=bf16))
    refuses("multiple of 16", K.fp8_quantise_rows, z(3, 140, dtype=bf16))
    refuses("multiple of 16", K.fp8_quantise_rows, z(3, 0, dtype=bf16))
    refuses("bf16 or fp32", K.fp8_quantise_rows, z(3, 144, dtype=torch.float16))
    refuses("bf16 or fp32", K.fp8_quantise_rows, z(144, 3, dtype=bf16).t())
    refuses("overlap", K.fp8_quantise_rows, z(1, 144, dtype=bf16).expand(3, 144))
    refuses("scale_fmt", K.fp8_quantise_rows, z(3, 144, dtype=bf16), scale_fmt="fp32")
    refuses("multiple of 16", K.fp8_quantise_blocks, z(3, 24))
    a, sa, w, sw = z(3, 272).to(E4M3), z(3, 3), z(200, 272).to(E4M3), z(2, 3)
    refuses("need CUDA", K.fp8_block_matmul, a, sa, w, sw)
    refuses("a must be", K.fp8_block_matmul, z(3, 272), sa, w, sw)
    refuses("a must be", K.fp8_block_matmul, z(3, 264).to(E4M3), sa, w, sw)
    refuses("w must be", K.fp8_block_matmul, a, sa, z(272, 200).to(E4M3).t(), sw)
    refuses("same number", K.fp8_block_matmul, a, sa, z(200, 256).to(E4M3), sw)
    refuses("a_scale", K.fp8_block_matmul, a, z(3, 2), w, sw)
    refuses("w_scale", K.fp8_block_matmul, a, sa, w, z(1, 3))
    refuses("bf16 or fp32", K.fp8_block_matmul, a, sa, w, sw, out_dtype=torch.float16)
    refuses("out must be", K.fp8_block_matmul, a, sa, w, sw, out=z(3, 199))
    refuses("out must be", K.fp8_block_matmul, a, sa, w, sw, out=z(1, 200).expand(3, 200))
    refuses("need CUDA", K.fp8_block_linear, z(3, 272, dtype=bf16), w, sw)
    refuses("same number", K.fp8_block_linear, z(3, 256, dtype=bf16), w, sw)


def test_c_abi_rejects_without_launching(lib):
    p = 4096                                   # an aligned address that nothing reads
    err = lambda rc, text: (rc, text in lib.b200dsa_last_error().decode())
    assert err(lib.b200dsa_latent_quant_and_cache(p, 0, 500, 3, None, 0, 1e-6, None, None, 0, p, p, 64, 1, p, None),
               "latent_quant_and_cache") == (-1, True)
    assert lib.b200dsa_latent_quant_and_cache(p, 0, 576, 3, None, 0, 1e-6, None, None, 0, p, p + 8, 64, 1, p, None) == -2
    assert lib.b200dsa_latent_quant_and_cache(p, 0, 576, 0, None, 0, 1e-6, None, None, 0, p, p, 64, 1, p, None) == 0
    assert lib.b200dsa_latent_cache_rows(p, 0, p, 3, p, p, None) == -1
    assert lib.b200dsa_latent_cache_rows(p, 8, p, 3, p + 2, p, None) == -2
    assert lib.b200dsa_latent_cache_gather(p, 64, 16, p, 1, 2, p, 1, 5, p, p, None) == -1
    assert lib.b200dsa_draft_tree_masks(p, 1, 65, p, p, None) == -1
    base = [p, p, 64, 16, p, 4, 4, 2, None, p, 8, 8, None, None, 0, None, None, 2, 16, 0.1, p, 1, p, 1, None, 0, p, None]

    def attend(**at):
        a = list(base)
        for k, v in at.items():
            a[int(k[1:])] = v
        return lib.b200dsa_sparse_mla_decode_cached(*a)

    assert attend(_18=129) == -1 and attend(_18=0) == -1          # heads
    assert attend(_10=7) == -1                                    # index stride
    assert attend(_19=0.0) == -1 and attend(_19=float("nan")) == -1
    assert attend(_7=1) == -1                                     # a request for every item
    assert attend(_15=p) == -1                                    # a mask without its base
    assert attend(_23=33) == -1 and attend(_23=0) == -1           # splits
    assert attend(_23=2, _24=p, _25=2 * 2 * 16 * 513 * 4 - 1) == -1
    assert attend(_2=2 ** 31) == -1                               # slots
    assert attend(_20=p + 4) == -2
    assert attend(_17=0) == 0
    assert lib.b200dsa_fp8_quantise_rows(p, 0, 144, 3, 140, 0, p, p, 3, None) == -1
    assert lib.b200dsa_fp8_quantise_rows(p, 0, 144, 3, 144, 0, p + 8, p, 3, None) == -2
    assert lib.b200dsa_fp8_quantise_blocks(p, 0, 100, 3, 144, 0, p, p, None) == -1
    mm = [p, 272, p, 3, 1, p, 272, p, 3, 1, 3, 200, 272, p, 0, 200, p, None]
    for at, v, rc in ((12, 270, -1), (1, 271, -1), (15, 199, -1), (0, p + 8, -2), (6, 280, -2), (13, p + 1, -2), (10, 0, 0)):
        a = list(mm)
        a[at] = v
        assert lib.b200dsa_fp8_block_matmul(*a) == rc, (at, v)
    ln = [p, 0, 272, 0, p, 272, p, 3, 1, 3, 200, 272, p, 0, 200, p, 3 * (272 + 12), p, None]
    for at, v, rc in ((16, 3 * 284 - 1, -1), (15, p + 4, -2), (5, 280, -2), (11, 264, -1), (9, 0, 0)):
        a = list(ln)
        a[at] = v
        assert lib.b200dsa_fp8_block_linear(*a) == rc, (at, v)


def test_decode_step_refuses_a_sharded_latent_cache():
    from tests import cpu_backend
    from transarch_b200.decode import ShardInfo, SparseDecodeStep
    with pytest.raises(ValueError, match="key-sharded"):
        SparseDecodeStep(2, 128, device=torch.device("cpu"), backend=cpu_backend, combine="nccl",
                         shard=ShardInfo(rank=0, world_size=2, shard_len=64), latent_page_size=64)


def test_oracle_scales_and_codes():
    """The 64-bit definitions against torch's e4m3 and against a search for the power of two."""
    from oracle import latent_oracle as L
    t = L.e4m3_table()
    ref = torch.arange(256, dtype=torch.uint8).view(E4M3).double()
    assert torch.equal(torch.isnan(t), torch.isnan(ref)) and torch.equal(t[~torch.isnan(t)], ref[~torch.isnan(ref)])
    v = torch.linspace(-460, 460, 20011, dtype=torch.float64)
    assert torch.equal(L.round_e4m3(v), v.clamp(-448, 448).float().to(E4M3).double())
    x = torch.randn(50, 300, generator=torch.Generator().manual_seed(1)) * 10
    _, s = L.quantise_groups(x, True)
    top = torch.stack([x[:, k:k + 128].abs().amax(1) for k in (0, 128, 256)], 1).double() / 448
    assert torch.equal(torch.exp2(torch.log2(s).round()), s) and bool((s >= top).all()) and bool((s < 2 * top).all())
