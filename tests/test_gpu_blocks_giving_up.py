"""A block-scaled product that gives up waits for its own copies and MMAs, and only for them: beside ``test_gpu_blocks_late`` (whose build of the
library and child process these are), products whose ring of stages has gone round a few times, or is not full, when the wait runs out."""

import os
import subprocess
import sys
import time
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from tests.test_gpu_blocks_late import MARK, product  # noqa: E402

pytestmark = pytest.mark.gpu


def few_rows(qb):
    """Three experts of few tokens each: of A only boxes of 32 rows are fetched."""
    from tests import util
    from tests.test_gpu_blocks import Operands, T

    M, N, K = 384, 200, 1200
    op = Operands(util.rng([97, M]), M, N, K, experts=3)
    y = T(qb, np.full((M, N), MARK["bf16"], np.uint16), "bf16")
    qb.qf.gemm_grouped_blocks(*op.tensors(qb), T(qb, np.arange(3, dtype=np.int32)), T(qb, np.array([9, 32, 17], np.int32)), n_experts=3, out=y, tile_n=128)
    return y.to_numpy(), np.zeros((1, 1), np.float32)


# name -> (call, rows and columns of the last CTA's last tile)
CASES = {
    "one block": (product(100, 64, 128, tile_n=64, split_k=1), np.s_[:, :64]),
    "two blocks, 256 columns": (product(100, 256, 256, tile_n=256), np.s_[:, :256]),
    "64 blocks, 64 columns": (product(200, 192, 8192, tile_n=64, split_k=1), np.s_[128:200, 128:192]),
    "9 blocks, 256 columns": (product(200, 328, 1152, tile_n=256), np.s_[128:200, 256:328]),
    # 20 x 16 tiles on 148 CTAs: the last one's second tile is number 295, the 40th of the third group of (4) row tiles
    "second tile of a CTA, 5 blocks, narrowed": (product(2500, 2048, 640, out="e4m3", tile_n=128), np.s_[2432:2500, 1152:1280]),
    "few rows of experts": (few_rows, np.s_[256:273, 128:200]),
}


def run_all(qb):
    results = {}
    for name, (call, _) in CASES.items():
        call(qb)  # (what a first call loads is not timed)
        qb._lib.device_status()
        t = time.perf_counter()
        results[name], results[name + " scales"] = call(qb)
        results[name + " seconds"] = time.perf_counter() - t
        results[name + " status"] = qb._lib.device_status()
    return results


@pytest.fixture(scope="module")
def results(tmp_path_factory):
    import quark_b200 as qb

    qb._lib.require_device(0)
    tmp = tmp_path_factory.mktemp("late")
    env = dict(os.environ, QB_BUILD_DIR=str(tmp), QB_BUILD_FLAGS="-DQB_LATE_WAIT")
    subprocess.run(["bash", str(ROOT / "quark_b200/csrc/build.sh")], env=env, check=True, timeout=600)
    env = dict(os.environ, QUARK_B200_LIB_PATH=str(tmp / "libquark_b200.so"))
    subprocess.run([sys.executable, __file__, str(tmp / "late.npz")], env=env, check=True, timeout=300)
    return run_all(qb), np.load(tmp / "late.npz")


@pytest.mark.parametrize("name", list(CASES))
def test_giving_up_waits_for_what_is_in_flight_only(results, name):
    usual, late = results
    assert usual[name + " status"] == 0 and late[name + " status"] != 0
    # a wait for something that does not come would take a second
    assert late[name + " seconds"] < 0.5 + usual[name + " seconds"]
    mark = MARK["bf16" if usual[name].dtype == np.uint16 else "e4m3"]
    rows, cols = CASES[name][1]
    want = usual[name].copy()
    assert not (want[rows, cols] == mark).any()
    want[rows, cols] = mark
    np.testing.assert_array_equal(late[name], want)
    scales = usual[name + " scales"].copy()
    if mark == MARK["e4m3"]:
        scales[cols.start // 128 : -(-cols.stop // 128), rows] = -5.0
    np.testing.assert_array_equal(late[name + " scales"], scales)


if __name__ == "__main__":
    import quark_b200

    np.savez(sys.argv[1], **run_all(quark_b200))
