"""The packed attention beside other calls and at the edge of what it accepts,
on the GPU."""
import pytest
import torch

from oracle import packed as O
from test_packed_gpu import SPEC, call, check, offsets, problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import mergenet_b200  # noqa: F401
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _status_stays_clear():
    import mergenet_b200
    d = torch.device("cuda", 0)
    mergenet_b200.attention.attention_status(d, reset=True)
    yield
    assert mergenet_b200.attention.attention_status(d, reset=True) == 0


@pytest.mark.parametrize("bad", ["past_the_end", "descending", "first", "length"])
def test_a_call_with_bad_offsets_leaves_later_calls_alone(dev, bad):
    """Bad offsets are recorded in a word that other attention calls share and
    that stays set; what those calls return is what they return without it."""
    import mergenet_b200 as mn
    from mergenet_b200 import _lib as L
    from mergenet_b200 import attention as local
    train = problem(dev, [2500, 1, 600], heads=16, kv_heads=4, dim=128, dtype=torch.bfloat16)
    images = problem(dev, [785, 393, 500], heads=6, kv_heads=6, dtype=torch.float16, spec=SPEC)
    cache = problem(dev, [1, 1], [30000, 700], heads=8, kv_heads=2, dim=128)
    gen = torch.Generator(device=dev).manual_seed(0)
    q, k, v = (torch.randn(4, 785, 6, 64, generator=gen, device=dev).half() for _ in range(3))
    qkv = torch.randn(4, 785, 3 * 384, generator=gen, device=dev).half()
    latent = torch.randn(4, 100, 6, 64, generator=gen, device=dev).half()

    def valid():
        got = [call(train, True, True), call(images, False, True), call(cache, True, False)]
        got.append({"local": local.unbiased_local_attention(q, k, v, 16),
                    "wide": local.unbiased_local_attention(q, k, v, 64),
                    "packed": local.local_attention_packed(qkv, 6, 16)})
        got.append({"latent": local.local_attention_packed(qkv, 6, -1), "cross": local.cross_attention(latent, k, v)})
        return got

    want = valid()
    p = problem(dev, [30, 40])
    cu, lens = {"past_the_end": ([0, 30, 900], None), "descending": ([0, 50, 20], None), "first": ([3, 30, 70], None),
                "length": ([0, 30, 70], [31, -1])}[bad]
    leaf = p["q"].detach().requires_grad_(True)
    mn.packed_attention(leaf, p["k"], p["v"], torch.tensor(cu, dtype=torch.int32, device=dev),
                        lengths_k=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)).sum().backward()
    assert mn.attention.attention_status(dev) == L.MN_STATUS_BAD_LENGTHS
    for _ in range(3):
        for a, b in zip(valid(), want):
            for name in b:
                assert torch.equal(a[name], b[name]), name
    assert mn.attention.attention_status(dev, reset=True) == L.MN_STATUS_BAD_LENGTHS
