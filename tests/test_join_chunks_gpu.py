"""The join of a row's chunks (csrc/score_head.cu) on lists as the kernel before leaves them, and on lists that hold anything, as where a wait of that kernel ran out."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
DEV = "cuda:0"


@pytest.fixture(scope="module")
def join(tmp_path_factory):
    from infer_b200.csrc import build
    so = str(tmp_path_factory.mktemp("join") / "join_check.so")
    subprocess.run([build._find_nvcc()] + build.NVCC_FLAGS + ["-I", build.HERE, "-o", so, os.path.join(HERE, "join_check.cu")], check=True, capture_output=True, timeout=300)
    f = ctypes.CDLL(so).join_check
    f.argtypes = [ctypes.c_int64] * 2 + [ctypes.c_int] * 3 + [ctypes.c_void_p] * 9

    def run(keys, top, vocab):
        chunks, rows, n = keys.shape
        stats = torch.zeros(chunks, rows, 4, device=DEV)
        stats[..., 1] = 1.0
        lists, at = torch.from_numpy(keys.view(np.int64)).to(DEV), torch.zeros(rows, device=DEV)
        lp, ent = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
        ids, best = torch.full((rows + 2, top), -7, dtype=torch.int32, device=DEV), torch.full((rows + 2, top), 7.0, device=DEV)
        assert f(rows, vocab, chunks, n, top, stats.data_ptr(), lists.data_ptr(), at.data_ptr(), lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), best.data_ptr(), None,
                 torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert (ids[rows:] == -7).all() and (best[rows:] == 7.0).all()
        return ids[:rows].cpu().numpy(), best[:rows].cpu().numpy()
    return run


def _key(z, i):
    bits = np.asarray(z, np.float32).view(np.uint32)
    order = np.where(bits & 0x80000000, ~bits, bits | 0x80000000).astype(np.uint64)
    return (order << np.uint64(32)) | (np.uint64(0xffffffff) - np.asarray(i, np.uint64))


@pytest.mark.parametrize("chunks,n,top", [(1, 8, 5), (3, 8, 8), (20, 20, 20), (148, 8, 1), (592, 20, 20)])
def test_lists_of_a_row(join, chunks, n, top):
    rng = np.random.default_rng(chunks)
    rows, V = 5, chunks * 40
    z = np.round(rng.normal(size=(rows, V)) * 4).astype(np.float32) + np.float32(0)           # many ties
    keys = np.zeros((chunks, rows, n), np.uint64)
    for c in range(chunks):
        k = _key(z[:, c::chunks], np.arange(V)[c::chunks])
        keys[c] = np.sort(k, 1)[:, ::-1][:, :n]
    ids, _ = join(keys, top, V)
    for r in range(rows):
        assert ids[r].tolist() == sorted(range(V), key=lambda i: (-z[r, i], i))[:top]


@pytest.mark.parametrize("chunks,n,top", [(21, 20, 20), (148, 8, 1), (148, 8, 8), (592, 20, 20), (592, 8, 3)])
@pytest.mark.parametrize("fill", ["one key", "all bits", "two keys", "noise"])
def test_lists_that_hold_anything(join, chunks, n, top, fill):
    """More lists than `top` pass the bound where keys are not distinct; the results are in their places, whatever they say, and nothing beside them is written."""
    rng = np.random.default_rng(3)
    shape = (chunks, 4, n)
    keys = {"one key": np.full(shape, int(_key(1.0, 9)), np.uint64), "all bits": np.full(shape, 0xffffffffffffffff, np.uint64),
            "two keys": rng.choice(np.array([int(_key(1.0, 9)), int(_key(2.0, 3))], np.uint64), shape),
            "noise": rng.integers(0, 1 << 64, shape, np.uint64, endpoint=False)}[fill]
    join(keys, top, 1000)
