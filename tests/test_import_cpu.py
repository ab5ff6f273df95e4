"""The package on a torch built without CUDA: import, routing to SDPA, and refusals of the kernel calls."""
import os
import subprocess
import sys

PROGRAM = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import rdna4_sage, sageattention
q, k, v = (torch.randn(1, 2, 8, 64, dtype=torch.bfloat16) for _ in range(3))
want = torch.nn.functional.scaled_dot_product_attention(q, k, v)
assert torch.equal(rdna4_sage.sageattn(q, k, v), want) and torch.equal(sageattention.sageattn(q, k, v), want)
kv = rdna4_sage.PagedKV.empty(4, 16, 2, 64, device="cpu")
table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
rope = rdna4_sage.Rotary(64, device="cpu")
for call in (lambda: rdna4_sage.attention(q, k, v), lambda: rdna4_sage.attention_paged_kv(q, kv, table, lens),
             lambda: rdna4_sage.paged_kv_append(kv, k, v, table, lens), lambda: rdna4_sage.paged_kv_read(kv, table, lens, 4),
             lambda: rdna4_sage.rotary(q, k, torch.arange(8), rope)):
    try:
        call()
    except rdna4_sage.Unsupported:
        continue
    raise AssertionError("not refused")
print("done")
"""


def test_import_without_cuda_in_torch():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = {**os.environ, "PYTHONPATH": os.path.join(root, "rdna4-sageattention_b200")}
    r = subprocess.run([sys.executable, "-c", PROGRAM], env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]
