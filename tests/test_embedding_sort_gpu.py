"""The embedding gradient on a device that has no room for a cluster of CTAs, such as a partition of a GPU. The device of the test has: the
library's source is compiled once more with a stand-in for the runtime's question, which answers that no cluster fits."""
import ctypes as C
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

from conftest import ROOT
from test_training_ops_gpu import assert_guards, guarded, normal

pytestmark = pytest.mark.gpu

STAND_IN = """
#include <cuda_runtime.h>
static int asked = 0;
extern "C" int times_asked() { return asked; }
extern "C" cudaError_t CUDARTAPI no_cluster_fits(int* clusters, const void*, const cudaLaunchConfig_t*) {
    *clusters = 0;
    return ++asked % 2 ? cudaSuccess : cudaErrorInvalidClusterSize;
}
"""


@pytest.fixture(scope="module")
def clusterless(cgb, tmp_path_factory):
    d = tmp_path_factory.mktemp("clusterless")
    (d / "stand_in.cu").write_text(STAND_IN)
    csrc, nvcc = os.path.join(ROOT, "cantors-gift_b200", "csrc"), os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    lib = str(d / "clusterless.so")
    r = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O3", "-Xcompiler", "-fPIC", "-shared", "-o", lib,
                        "-I" + os.path.join(ROOT, "include"), "-I" + csrc, "-DcudaOccupancyMaxActiveClusters=no_cluster_fits",
                        os.path.join(csrc, "embedding.cu"), os.path.join(csrc, "runtime.cu"), str(d / "stand_in.cu")],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    L = C.CDLL(lib)
    for name in ("cg_b200_embedding_backward", "cg_b200_embedding_backward_workspace_bytes"):
        fn = getattr(L, name)
        fn.restype, fn.argtypes = cgb.capi.SIGNATURES[name]
    return L


@pytest.mark.parametrize("n,vocab,cols", [(1, 3, 8), (1024, 90, 16), (1025, 90, 16), (5000, 300, 264), (9000, 300000, 33), (70000, 50000, 24),
                                          (131072, 700, 12)])
def test_gradient_without_clusters(ops, cgb, clusterless, n, vocab, cols):
    """Ids of up to 131072 tokens are sorted by the launches that sort more of them otherwise: the same order, so the same bits."""
    dy = normal(n, cols, seed=n)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    ids = (torch.rand(n, device="cuda", generator=g) ** 2 * (vocab + 2)).long() - 1
    want = ops.embedding_backward(dy, ids, vocab, scale=0.5, padding_id=1)
    need = C.c_size_t(0)
    assert clusterless.cg_b200_embedding_backward_workspace_bytes(n, vocab, cols, C.byref(need)) == cgb.capi.OK
    ws = torch.full((need.value,), 255, dtype=torch.uint8, device="cuda")
    buf, out = guarded((vocab, cols), torch.float32)
    before = clusterless.times_asked()
    for accumulate in (0, 1):
        st = clusterless.cg_b200_embedding_backward(cgb.capi.F32, cgb.capi.F32, dy.data_ptr(), ids.data_ptr(), 8, n, 0.5, 1, accumulate, out.data_ptr(),
                                                    vocab, cols, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert st == cgb.capi.OK
        if not accumulate:
            assert torch.equal(out, want)
    assert torch.equal(out, 2 * want)   # the same sum on top of itself: exact
    assert_guards(buf, out, "gradient")
    assert clusterless.times_asked() == before + (2 if n > 1024 else 0)   # one CTA is no cluster
