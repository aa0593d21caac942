"""CPU: no queries over any number of keys is a call like any other (in a process of its own: a division by zero ends it)."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = """
from image_generator_amd._lib import lib
for keys in (0, 1, 383, 384, 5000, 1 << 24):
    for heads, kv in ((8, 8), (8, 2), (1, 1), (32, 1), (128, 1)):
        for docs in (1, 2, 1000):
            assert lib.mi355_doc_attention_fwd_workspace_bytes(0, keys, heads, kv, 96, docs) == 0, (keys, heads, kv, docs)
            assert lib.mi355_doc_attention_bwd_workspace_bytes(0, keys, heads, kv, 96, docs, 0) == 16, (keys, heads, kv, docs)
            assert lib.mi355_doc_attention_fwd(None, 16, 16, None, None, 16, 16, docs, None, None, 0.0, 0, 0, 0, keys, heads, kv, 96, 96 * heads, 96 * kv,
                                               96 * kv, 96 * heads, 1.0, 0.0, 0, None, 0, None) == 0
print("answered")
"""


def test_sizes_without_queries():
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "answered", (r.returncode, r.stdout, r.stderr)
