"""The 8-bit form of LaplacianBlock beside weights that change after it was laid out."""
import copy
import io

import pytest
import torch

from laplacianformer_b200.block import LaplacianBlock

pytestmark = pytest.mark.gpu


def eight_bit(b, x):
    """What a block of b's weights gives that was quantised just now."""
    c = LaplacianBlock(64, heads=2, grid=8, device="cuda")
    c.load_state_dict({k: v.clone() for k, v in b.state_dict().items()})
    with torch.no_grad():
        return c.quantize_()(x)


def new_weights(b, k):
    g = torch.Generator().manual_seed(k)
    return (torch.randn(b.w_qkv.shape, generator=g) * 0.125).bfloat16().cuda()


CHANGES = {
    "in place": lambda b: b.w_qkv.mul_(1.5),
    "optimizer step": lambda b: (setattr(b.w_qkv, "grad", torch.ones_like(b.w_qkv)), torch.optim.SGD([b.w_qkv], lr=0.25).step()),
    "load_state_dict": lambda b: b.load_state_dict({**b.state_dict(), "w_qkv": new_weights(b, 1)}),
    "load_state_dict by assignment": lambda b: b.load_state_dict({**b.state_dict(), "w_qkv": new_weights(b, 2)}, assign=True),
    "new data": lambda b: setattr(b.w_qkv, "data", new_weights(b, 3)),
    "new parameter": lambda b: setattr(b, "w_qkv", torch.nn.Parameter(new_weights(b, 4))),
    "new parameter of the old storage": lambda b: (setattr(b, "w_qkv", torch.nn.Parameter(b.w_qkv.data)), b.w_qkv.neg_()),
    "there and back": lambda b: (b.to("cpu"), b.w_qkv.mul_(0.5), b.to("cuda")),
    "data in place before eval()": lambda b: (b.w_qkv.data.mul_(-2), b.eval()),
}


@pytest.mark.parametrize("change", list(CHANGES))
@pytest.mark.parametrize("used", [False, True])
def test_block_quantized_follows_its_weights(change, used):
    """Whatever changes the 16-bit weights after quantize_(), the 8-bit form is of the weights that there are."""
    torch.manual_seed(2)
    b = LaplacianBlock(64, heads=2, grid=8, device="cuda").quantize_()
    x = torch.randn(2, 64, 64, device="cuda").bfloat16()
    with torch.no_grad():
        before = eight_bit(b, x)
        if used:
            assert torch.equal(b(x), before)
        CHANGES[change](b)
        got = b(x)
        assert torch.equal(got, eight_bit(b, x)) and not torch.equal(got, before)
        assert torch.equal(b(x), got)


def test_block_quantized_copies_and_modes():
    """Copies are quantised too, inference mode works, and a captured forward follows the weights when replayed."""
    torch.manual_seed(3)
    b = LaplacianBlock(64, heads=2, grid=8, device="cuda").quantize_()
    x = torch.randn(2, 64, 64, device="cuda").bfloat16()
    with torch.no_grad():
        want = b(x)
        c = copy.deepcopy(b)
        assert torch.equal(c(x), want)
        c.w_qkv.mul_(2)
        assert torch.equal(c(x), eight_bit(c, x)) and torch.equal(b(x), want)
    with torch.inference_mode():
        assert torch.equal(b(x), want)
        d = LaplacianBlock(64, heads=2, grid=8, device="cuda")
        d.load_state_dict(b.state_dict())
        assert torch.equal(d.quantize_()(x), want)
        d.w_qkv.mul_(0.5)
        assert torch.equal(d(x), eight_bit(d, x))
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = b(x)
        b.w_qkv.mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eight_bit(b, x)) and torch.equal(b(x), y)
    assert set(b.state_dict()) == set(LaplacianBlock(64, heads=2, grid=8).state_dict())


def test_block_quantized_on_another_stream():
    """A forward on one stream lays the weights out late; one on another stream waits for that, and keeps them alive."""
    torch.manual_seed(4)
    b = LaplacianBlock(64, heads=2, grid=8, device="cuda").quantize_()
    x = torch.randn(2, 64, 64, device="cuda").bfloat16()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.no_grad():
        for _ in range(3):
            b.w_qkv.mul_(1.25)
            want = eight_bit(b, x)
            torch.cuda.synchronize()
            with torch.cuda.stream(one):
                torch.cuda._sleep(50_000_000)
                first = b(x)
            with torch.cuda.stream(two):
                second = b(x)
                b.eval()  # drops what stream two still reads
                third = b(x)
            torch.cuda.synchronize()
            for y in (first, second, third):
                assert torch.equal(y, want)


def test_block_quantized_copies_by_pickle():
    torch.manual_seed(5)
    b = LaplacianBlock(64, heads=2, grid=8, device="cuda").quantize_()
    x = torch.randn(2, 64, 64, device="cuda").bfloat16()
    with torch.no_grad():
        want = b(x)
        f = io.BytesIO()
        torch.save(b, f)
        f.seek(0)
        c = torch.load(f, weights_only=False)
        assert c.quantized and torch.equal(c(x), want)
        c.w_qkv.neg_()
        assert torch.equal(c(x), eight_bit(c, x))
