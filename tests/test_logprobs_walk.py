"""The walk over a long row's best classes on the host, thread by thread: what a workgroup finds must not depend on how its
waves run between two barriers.  The kernel's own source is compiled for the host (host_waves) and each wave run as far
as the next barrier lets it, in one order after the other."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import helpers_logprobs as ref
from imagesegmentation_amd import build

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_waves")
CLANG = os.path.join(os.path.dirname(build.HIPCC), "amdclang++")
ORDERS = [(0, 1, 2, 3), (3, 2, 1, 0), (1, 2, 3, 0), (2, 0, 3, 1)]


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no %s" % CLANG)
    folder = tmp_path_factory.mktemp("walk")
    with open(os.path.join(build.CSRC, "isg_logprobs.hip")) as f:
        text = f.read()
    kernels = str(folder / "kernels.h")
    with open(kernels, "w") as f:  # up to the walk; the namespace it stands in is closed here
        f.write(text[:text.index("// Joins the parts of a row")] + "}\n")
    out = str(folder / "walk.so")
    subprocess.run([CLANG, "-x", "c++", "-std=c++20", "-O1", "-w", "-fPIC", "-shared", "-I", HERE, "-I", build.CSRC,
                    "-DKERNELS=\"%s\"" % kernels, os.path.join(HERE, "walk.cpp"), "-o", out], check=True)
    entry = ctypes.CDLL(out).walk

    def call(row, top, order):
        row = np.ascontiguousarray(row, np.float32)
        entropy, logp, classes = np.zeros([1], np.float32), np.zeros([top], np.float32), np.full([top], -2, np.int32)
        p = lambda a: a.ctypes.data_as(ctypes.c_void_p)
        rc = entry(p(row), row.size, top, p(np.asarray(order, np.int32)), p(entropy), p(logp), p(classes))
        return rc, entropy, logp, classes
    return call


def _rows(cols):
    rs = np.random.RandomState(cols)
    ramp = np.linspace(-8, 8, cols)
    return {"random": rs.randn(cols) * 3, "rising": ramp, "rising steps": np.floor(ramp * 4) / 4, "falling": ramp[::-1],
            "constant": np.zeros(cols), "few": np.where(np.arange(cols) % (cols // 7) == 3, ramp, -np.inf),
            "overrun": np.where(np.arange(cols) < 4096, rs.randn(cols), np.arange(cols) // 700 + 10.0)}


@pytest.mark.parametrize("top", [1, 20, 64])
@pytest.mark.parametrize("kind", sorted(_rows(13001)))
def test_the_best_classes_do_not_depend_on_the_order_of_the_waves(walk, kind, top):
    z = _rows(13001)[kind].astype(np.float32)
    want = ref.token_logprobs(z[None].astype(np.float64), 1.0, None, top)
    for order in ORDERS:
        rc, entropy, logp, classes = walk(z, top, order)
        assert rc == 0, "order %s: %s" % (order, {-1: "lanes of a wave at different places", -2: "waves at different barriers",
                                                  -3: "a barrier that some waves never come to"}[rc])
        assert np.array_equal(classes, want["top_classes"][0]), order
        ref.close(logp[None], want["top_logprobs"], want["top_logprobs_tol"])
        ref.close(entropy, want["entropy"], want["entropy_tol"])
