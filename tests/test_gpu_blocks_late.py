"""What a block-scaled product leaves of a call in which a wait ran out: the tile that the late work belongs to stays as it was, whole, all
others are what they always are, and the status says so.

The library is built once more with QB_LATE_WAIT (``late`` in csrc/sm100.cuh): the MMA thread of the last CTA of a grid, its last tile's work
done, waits half a millisecond for a flag that nothing sets and gives up.  A child process loads it and makes the calls below."""

import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

pytestmark = pytest.mark.gpu

MARK = {"bf16": 0x7FC1, "e4m3": 0x7F}  # NaN that no call computes


def product(M, N, K, out="bf16", experts=0, **kw):
    """The result, and the scales of a narrowed one."""

    def run(qb):
        from tests import util
        from tests.test_gpu_blocks import Operands, T, blocks

        op = Operands(util.rng([95, M, N]), M, N, K, experts=max(experts, 1))
        y = T(qb, np.full((M, N), MARK[out], np.uint16 if out == "bf16" else np.uint8), out)
        s = T(qb, np.full((blocks(N), M), -5.0, np.float32)) if out == "e4m3" else None
        if experts:
            tables = (T(qb, np.array([0] * (M // 128 - 1) + [experts - 1], np.int32)), T(qb, np.full(M // 128, 128, np.int32)))
            qb.qf.gemm_grouped_blocks(*op.tensors(qb), *tables, n_experts=experts, out=y, scale_out=s, **kw)
        else:
            if out == "bf16":
                r = util.rng(96)
                kw.update(gate=T(qb, util.bf16_randn(r, (1, N)), "bf16"), residual=T(qb, util.bf16_randn(r, (M, N)), "bf16"))
            qb.qf.gemm_blocks(*op.tensors(qb), out=y, scale_out=s, **kw)
        return y.to_numpy(), s.to_numpy() if s else np.zeros((1, 1), np.float32)

    return run


# name -> (call, rows and columns of the last CTA's last tile)
CASES = {
    "64 columns": (product(200, 192, 512, tile_n=64, split_k=1), np.s_[128:200, 128:192]),
    "128 columns, remainder": (product(200, 200, 528, tile_n=128), np.s_[128:200, 128:200]),
    "256 columns, remainder": (product(200, 328, 512, tile_n=256), np.s_[128:200, 256:328]),
    "cluster of 4 slices": (product(200, 192, 2048, tile_n=64, split_k=4), np.s_[128:200, 128:192]),
    "cluster of 8 slices": (product(100, 192, 2048, tile_n=64, split_k=8), np.s_[:, 128:192]),
    "narrowed, 128 columns": (product(200, 264, 512, out="e4m3", tile_n=128), np.s_[128:200, 256:264]),
    "narrowed, 256 columns": (product(200, 392, 512, out="e4m3", tile_n=256), np.s_[128:200, 256:392]),
    # 19 x 16 tiles on 148 CTAs: the last one's second tile is number 295, the 40th of the third group of (3) row tiles
    "second tile of a CTA": (product(2400, 2048, 256, tile_n=128), np.s_[2048:2176, 1664:1792]),
    "experts": (product(512, 192, 512, experts=2, tile_n=64), np.s_[384:, 128:192]),
    "experts, narrowed": (product(512, 264, 512, experts=2, out="e4m3", tile_n=128), np.s_[384:, 256:264]),
}


def run_all(qb):
    results = {}
    for name, (call, _) in CASES.items():
        qb._lib.device_status()
        results[name], results[name + " scales"] = call(qb)
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
def test_the_late_tile_stays_as_it_was(results, name):
    usual, late = results
    assert usual[name + " status"] == 0 and late[name + " status"] != 0
    mark = MARK["bf16" if usual[name].dtype == np.uint16 else "e4m3"]
    assert not (usual[name] == mark).any()
    rows, cols = CASES[name][1]
    want = usual[name].copy()
    want[rows, cols] = mark
    np.testing.assert_array_equal(late[name], want)
    scales = usual[name + " scales"].copy()
    if mark == MARK["e4m3"]:
        assert not (scales == -5.0).any()
        scales[cols.start // 128 : -(-cols.stop // 128), rows] = -5.0
    np.testing.assert_array_equal(late[name + " scales"], scales)


if __name__ == "__main__":
    import quark_b200

    np.savez(sys.argv[1], **run_all(quark_b200))
