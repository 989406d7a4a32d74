"""Greedy speculative decoding needs librq alone: no torch, no torch binding."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys
sys.modules.update(dict.fromkeys({missing}))
from rustyllm_b200.spec import SpecDecoder

class Counter:
    "says n + 1 after n; the draft is wrong about every third"
    def __init__(self, wrong):
        self.wrong, self.pos = wrong, 0
    def after(self, t, pos):
        return t + 2 if self.wrong and pos % 3 == 0 else t + 1
    def forward(self, ids, pos, want_logits=True):
        return None, self.after(ids[-1], pos)
    def forward_all(self, ids, pos):
        return None, [t + 1 for t in ids]
    def truncate_caches(self, n):
        self.pos = n

dec = SpecDecoder(Counter(False), Counter(True), k=4)
assert dec.generate([1, 2, 3], 20) == list(range(4, 24))
assert 0 < dec.stats["accepted"] < dec.stats["proposed"]
"""


def run(missing):
    return subprocess.run([sys.executable, "-c", SCRIPT.format(missing=missing)], cwd=ROOT, capture_output=True, text=True)


def test_greedy_decoding_without_the_torch_binding():
    r = run(["rustyllm_b200._rqtorch"])
    assert r.returncode == 0, r.stderr


def test_greedy_decoding_without_torch():
    r = run(["torch", "rustyllm_b200._rqtorch"])
    assert r.returncode == 0, r.stderr
