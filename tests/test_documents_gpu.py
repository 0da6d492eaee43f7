"""The documents' examples run, with operands of the layouts that they state."""

import re
from pathlib import Path

import pytest
import torch

import dwarf_amd

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def layouts(line):
    """{name: (letters)} of "q, out [B,H,T,D], k, v [B,H_kv,T,D]; ..."."""
    res = {}
    for names, letters in re.findall(r"((?:\w+, )*\w+) \[([^\]]+)\]", line):
        for n in names.split(", "):
            res[n] = tuple(x.strip() for x in letters.split(","))
    return res


CALL = "cache.tree_step(q, k, v, parents)"
DOCUMENTS = [p for p in sorted(ROOT.glob("*.md")) if CALL in p.read_text()]


def test_documents_are_found():
    assert len(DOCUMENTS) >= 2


@pytest.mark.parametrize("document", DOCUMENTS, ids=lambda p: p.stem)
def test_drafted_tokens(gpu_device, document):
    text = document.read_text()
    line = next(x for x in text.splitlines() if CALL in x)
    block = next((b for b in re.findall(r"```python\n(.*?)```", text, re.S) if line in b), None)
    shapes = layouts(line.split("#", 1)[1])
    sizes = dict(B=3, H=4, H_kv=2, T=5, D=32)  # (all of them different)
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn([sizes[x] for x in shapes[n]], generator=g).to(torch.bfloat16).to(gpu_device) for n in "qkv")
    space = dict(sizes, q=q, k=k, v=v, parents=torch.tensor([[-1, 0, 0, 1, 3]] * 3, device=gpu_device), u=torch.rand(3, 5, generator=g).to(gpu_device),
                 drafted=torch.randint(0, 9, (3, 5), generator=g).to(gpu_device), logits=lambda x: x.float() @ weights,
                 sample_tokens=dwarf_amd.sample_tokens, draft_tree_accept=dwarf_amd.draft_tree_accept,
                 cache=dwarf_amd.PagedKVCache(3, 2, 32, 64, torch.bfloat16, gpu_device))
    weights = torch.randn(4 * 32, 9, generator=g).to(gpu_device)
    exec(line.strip() if block is None else block, space)
    if block is not None:
        assert space["picks"].shape == (3, 5)
        assert (space["cache"].pos == space["n"]).all() and (space["n"] >= 1).all()
    assert space["out"].shape == tuple(sizes[x] for x in shapes["out"])
