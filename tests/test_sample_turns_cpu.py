"""The rule by which the sampling kernel's exchanges between threads and between blocks take turns, compiled for the
host from the kernel's header (CPU only)."""
import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG, REPO


@pytest.mark.skipif(shutil.which("nvcc") is None, reason="nvcc not available")
def test_exchanges_never_share_a_set(tmp_path):
    exe = str(tmp_path / "sample_turns_check")
    src = os.path.join(REPO, "tests", "sample_turns_check.cu")
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17",
                           "-I" + os.path.join(PKG, "csrc"), "-o", exe, src])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "unsound orders 0" in r.stdout, r.stdout + r.stderr


def test_words_of_a_cluster_take_the_clusters_turn():
    """Each set that other blocks read is taken by the next_cluster() right before it, and each that only the block's
    threads read by next_block()."""
    with open(os.path.join(PKG, "csrc", "eii_sample.cuh")) as f:
        text = re.sub(r"//.*", "", f.read())
    text = text[text.index("k_sample("):]
    taken = {}
    uses = 0
    for m in re.finditer(r"const int (\w+) = turns\.next_(block|cluster)\(\)|sh\.(warp|block)_(?:max|mass|n)\[(\w+)\]", text):
        if m[1]:
            taken[m[1]] = m[2]
        else:
            assert taken[m[4]] == {"warp": "block", "block": "cluster"}[m[3]], text[m.start() - 200:m.end()]
            uses += 1
    assert uses > 20
