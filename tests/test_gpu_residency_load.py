"""Loading with an expert budget ends: in a process of its own, which a load that does not return cannot stop."""
import os
import subprocess
import sys

import pytest

import eahmmf_b200 as eb

pytestmark = pytest.mark.gpu


def test_a_budgeted_load_ends_and_copies_by_dma(tmp_path):
    code = """
import sys; sys.path[:0] = [%r]
import eahmmf_b200 as eb, synth
cfg = synth.config_kquant_small(n_layer=24)
small = synth.write_gguf(%r, cfg)
path = small + ".once"
open(path, "wb").write(open(small, "rb").read())  # 100 MB in one write: large pages of the file cache
tg, tu, td = cfg.expert_types
foot = sum((n + 255) // 256 * 256 for n in (cfg.FF * synth.row_bytes(tg, cfg.D), cfg.FF * synth.row_bytes(tu, cfg.D),
                                             cfg.D * synth.row_bytes(td, cfg.FF)))
e = eb.Engine(path, 64, expert_vram_bytes=2 * cfg.n_expert * foot)
assert e.greedy([1, 2, 3], 4, 32)[0] == 0
print("dma", e.cache_stats()["dma"])
e.close()
""" % (os.path.dirname(eb.__file__), str(tmp_path / "m.gguf"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=150)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "dma 1" in r.stdout or "dma True" in r.stdout, r.stdout
