"""The 8-bit path with dependent launches on (B200DSA_PDL=1, read once by a process): kernels of one stream overlap, and
each still sees what the one before it wrote."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu

STEPS = """
import torch
from tests.test_gpu_latent_cache import _status, _tree, attend_case, check_attend
from transarch_b200 import kernels as K

# masks of new parents, attention under them, then the next masks into the memory that these leave behind
g = torch.Generator().manual_seed(4)
cases = [attend_case(200 + i, 2, 8, H, 150, 300, 32, drafts=8) for i, H in enumerate((16, 64, 128))]
trees = [[torch.stack([_tree(8, g) for _ in range(2)]) for _ in cases] for _ in range(6)]
on = lambda t: t.to("cuda")
d = [{k: on(v) if isinstance(v, torch.Tensor) else v for k, v in c.items()} for c in cases]
parents = [[on(t) for t in turn] for turn in trees]
torch.cuda.synchronize()
got = []
for turn in parents:
    for c, par in zip(d, turn):
        masks = K.draft_tree_masks(par)
        out = K.sparse_mla_decode_cached(c["q"], c["cache"], c["page"], c["idx"], c["scale"], block_table=c["table"],
                                         row_request=c["req"], q_pos=c["qpos"], tree_mask=masks.view(-1), tree_base=c["lens"])
        got.append((masks.clone(), *out))
        del masks
torch.cuda.synchronize()
assert _status() == 0
at = iter(got)
for turn in trees:
    for c, par in zip(cases, turn):
        masks, out, lse = next(at)
        want = torch.zeros(2, 8, dtype=torch.int64)
        for r in range(2):
            for j in range(8):
                node = j
                while node >= 0:
                    want[r, j] |= 1 << node
                    node = int(par[r, node])
        assert torch.equal(masks.cpu(), want)
        check_attend(dict(c, mask=want.view(-1)), out, lse, items=(0, 7, 11))
"""


def _run(args):
    r = subprocess.run([sys.executable, *args], cwd=ROOT, env={**os.environ, "B200DSA_PDL": "1"}, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


def test_masks_and_attention_in_turn():
    _run(["-c", STEPS])


def test_the_paths_own_tests():
    _run(["-m", "pytest", "-x", "-q", "tests/test_gpu_latent_step.py", "tests/test_gpu_latent_cache.py",
          "tests/test_gpu_fp8_block.py", "-k", "step or stream or tree or splits or written or linear or wave"])
