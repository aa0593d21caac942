"""CPU: the code that a counter profile of the benchmarked step belongs to."""
import os
import re
import shutil

import bench

PKG = os.path.join(bench.ROOT, "image_generator_amd")


def read(*parts):
    return open(os.path.join(PKG, *parts)).read()


def test_sources_outside_the_step_leave_it_alone(tmp_path):
    shutil.copytree(os.path.join(PKG, "csrc"), tmp_path / "image_generator_amd" / "csrc", ignore=shutil.ignore_patterns("build"))
    for f in ("ops.py", "unet.py", "trainer.py"):
        shutil.copy(os.path.join(PKG, f), tmp_path / "image_generator_amd" / f)
    want = bench.source_fingerprint()
    assert bench.source_fingerprint(str(tmp_path)) == want
    for f in sorted(bench.NOT_IN_STEP):
        (tmp_path / "image_generator_amd" / "csrc" / f).write_text("changed")         # (each of them exists: copied above)
        assert os.path.exists(os.path.join(PKG, "csrc", f)), f
    assert bench.source_fingerprint(str(tmp_path)) == want
    for f in ("csrc/gemm.hip", "csrc/wgrad.hip", "csrc/common.h", "trainer.py"):
        with open(tmp_path / "image_generator_amd" / f, "a") as out:
            out.write("\n")
        now = bench.source_fingerprint(str(tmp_path))
        assert now != want, f
        want = now


def test_the_step_launches_nothing_of_what_is_left_out():
    entries = set()
    for f in bench.NOT_IN_STEP:
        entries |= set(re.findall(r"^\w[\w *]*\b(mi355_\w+)\(", read("csrc", f), flags=re.M))
    assert {"mi355_doc_attention_fwd", "mi355_embedding_bwd", "mi355_multi_adamw_step", "mi355_lmdb_open"} <= entries
    for module in ("ops.py", "unet.py", "trainer.py"):
        called = set(re.findall(r"lib\.(mi355_\w+)", read(module)))
        assert not called & entries, (module, called & entries)
    for module in ("unet.py", "trainer.py"):                 # ... nor by way of the wrappers
        assert not re.search(r"doc_attention|ops\.embedding|TensorAdamW|host\(\)", read(module)), module
