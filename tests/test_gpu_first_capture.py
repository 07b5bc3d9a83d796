"""The first call of each first-order operator in a process, made inside a graph capture."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

CODE = """
import sys
sys.path.insert(0, {path!r})
import torch
from dsmezo_b200 import AdamW, grouped, scoring
dev = "cuda"
x = torch.randn(300, 512, device=dev).bfloat16()
w = torch.randn(2, 512, 48, device=dev).bfloat16()
dy = torch.randn(300, 48, device=dev).bfloat16()
off = torch.tensor([0, 100, 300], dtype=torch.int32, device=dev)
logits, targets = torch.randn(6, 5000, device=dev), torch.zeros(6, dtype=torch.int32, device=dev)
p, g = torch.randn(1000, device=dev), torch.randn(1000, device=dev)
opt = AdamW([p], grads=[g], state_bits=8, capturable=True)
calls = dict(product=lambda: grouped.grouped_matmul(x, w, off), weight_grad=lambda: grouped.grouped_weight_grad(x, dy, off),
             loss=lambda: scoring.contrastive_loss_grad(logits, [2, 4], [1.0, -1.0], targets)[1], adamw=opt.step)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = calls[{op!r}]()
graph.replay()
torch.cuda.synchronize()
if out is not None:
    assert torch.equal(out, calls[{op!r}]())
else:
    assert int(opt.step_counter) == 1
print("ok")
"""


@pytest.mark.parametrize("op", ["product", "weight_grad", "loss", "adamw"])
def test_first_call_inside_a_capture(op):
    r = subprocess.run([sys.executable, "-c", CODE.format(path=str(ROOT / "ds-mezo_b200"), op=op)], capture_output=True,
                       text=True, timeout=240)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]
