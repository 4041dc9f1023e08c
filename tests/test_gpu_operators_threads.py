"""The operators from several threads at once, each on its own stream and tensors, in a process that has not called
them before: what they look up once is shared (needs a B200)."""
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys, threading
sys.path.insert(0, "tests")
import torch
from conftest import load_package
ops = load_package().ops
# (n_rows, n_q, head_dim, keys): one- and few-row tiles, 64-row tiles, tcgen05 tiles with the key axis whole and split
shapes = [(1, 8, 128, 700), (9, 8, 64, 300), (60, 2, 128, 4000), (300, 8, 128, 400), (300, 8, 64, 20000), (2, 2, 64, 9000), (40, 8, 128, 30), (700, 2, 64, 1000)]

def work(i, out, gate):
    rows, n_q, hd, keys = shapes[i % len(shapes)]
    g = torch.Generator(device="cuda").manual_seed(i)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c = ops.PagedKV.empty(-(-keys // 64), 2, hd, torch.arange(-(-keys // 64), dtype=torch.int32, device="cuda")[None])
        k, v = (torch.randn((keys, 2, hd), generator=g, device="cuda").half() for _ in range(2))
        q = torch.randn((rows, n_q, hd), generator=g, device="cuda").half()
        x = torch.randn((rows, 5000), generator=g, device="cuda")
        off, lens, none = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, rows], [keys], [0]))
        koff = torch.tensor([0, keys], dtype=torch.int32, device="cuda")
        st.synchronize()
        gate.wait()
        for _ in range(5):
            ops.kv_append(c, k, v, koff, none, max_rows=keys)
            a = ops.kv_attention(c, q, off, lens, max_rows=rows, max_keys=keys)
            p = ops.token_logprobs(x, top_k=5)
        st.synchronize()
        out[i] = [a.clone(), p[1].clone(), p[2].clone(), c.k.view(torch.uint8).clone()]
        st.synchronize()

n = 2 * len(shapes)
torch.zeros(1, device="cuda")
together, alone = {}, {}
gate = threading.Barrier(n)
threads = [threading.Thread(target=work, args=(i, together, gate)) for i in range(n)]
[t.start() for t in threads]
[t.join() for t in threads]
one = threading.Barrier(1)
for i in range(n):
    work(i, alone, one)
assert len(together) == n and all(bool((a == b).all()) for i in range(n) for a, b in zip(together[i], alone[i]))
print("same")
"""


def test_threads():
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), (r.stdout[-500:], r.stderr[-2000:])
