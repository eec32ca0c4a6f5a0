"""Embedding rows' gradient by the sort of four CTAs: more than 2048 tokens and a
table of more than 16 KB for each."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import ttfoil as tf  # noqa: E402
from test_token_path_gpu import BF, F32, close, embed_grad, embed_ref, gen, make_ids, randn  # noqa: E402


@pytest.fixture(autouse=True, scope="module")
def device():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    tf.device_error()


@pytest.mark.parametrize("T,V,D,kind", [(2500, 50000, 256, "frequent"), (2049, 9000, 1001, "any"),
                                        (4099, 40001, 514, "frequent"), (2300, 20000, 512, "one"),
                                        (9000, 300000, 129, "sorted")])
@pytest.mark.parametrize("fp32,long_ids", [(False, True), (True, False)])
def test_gradient_sorted_by_four_ctas(T, V, D, kind, fp32, long_ids):
    assert T > 2048 and V * D > 4096 * T
    g = gen(T + V)
    ids = make_ids(g, T, V, kind).to(torch.int64 if long_ids else torch.int32)
    dout = randn(g, T, D, dtype=F32 if fp32 else BF)
    got = embed_grad(ids.cuda(), dout.cuda(), V, 1.7)
    ref, slack = embed_ref(ids.long(), dout, V, 1.7)
    close(got, ref, slack, F32)
    assert torch.equal(got, embed_grad(ids.cuda(), dout.cuda(), V, 1.7))
    assert tf.device_error() == 0
