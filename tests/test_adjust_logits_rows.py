"""adjust_logits on many rows, whose workgroups are dealt to the XCDs row by row, in every width, captured, and with the ends of what one row may hold."""
import pytest
import torch

from test_adjust_logits import TYPES, check, launch, make, plain


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [(63, 1500, 9, 2, True), (64, 1025, 40, 0, True), (65, 8191, 7, 3, False), (71, 8193, 60, 0, True), (131, 5000, 200, 5, True), (200, 33, 3, 1, True)])
def test_gpu_many_rows(ct, dev, dtype, rows, vocab, history, biases, mask):
    x = make(rows, vocab, dtype, history, biases, mask, rows + vocab)
    on = {k: v.to(dev) for k, v in x.items()}
    want, size = plain(**x)
    for v in (None, 1024, 4096, 8192):
        wide = torch.full((rows + 2, vocab + 5), 7.0, dtype=TYPES[dtype], device=dev)     # rows at odd places, and some that are nobody's around them
        out = wide[1:-1, 2:-3]
        launch(ct, on, out, variant=v and f"{dtype}_{v}")
        check(out.cpu(), want, size, biases)
        out.fill_(7.0)
        assert bool((wide == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 70])
def test_gpu_captured(ct, dev, rows):
    """a graph replayed for other logits, histories and lengths, with eager work between"""
    x = make(rows, 9001, "bf16", 50, 6, True, rows)
    on = {k: v.to(dev) for k, v in x.items()}
    out, eager = torch.zeros_like(on["logits"]), torch.zeros_like(on["logits"])
    launch(ct, on, out)
    torch.cuda.synchronize()
    g = ct.CapturedGraph().capture(lambda s: launch(ct, on, out, stream=s))
    for i in range(3):
        other = make(rows, 9001, "bf16", 50, 6, True, 100 + i)
        for k, v in other.items():
            on[k].copy_(v)
        torch.cuda.synchronize()
        g.launch()
        g.synchronize()
        launch(ct, on, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        want, size = plain(**other)
        check(out.cpu(), want, size, 6)
    g.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 66])
def test_gpu_one_token_all_along(ct, dev, rows):
    """every token and every bias of a row the same one"""
    vocab, n = 4097, 5000
    x = {"logits": torch.ones(rows, vocab), "tokens": torch.full((rows, n), 4096, dtype=torch.int32), "frequency": torch.full((rows,), 0.5), "repetition": torch.full((rows,), 2.0),
         "bias_ids": torch.full((rows, 1024), 4096, dtype=torch.int32), "bias_values": torch.full((rows, 1024), 0.25)}
    on = {k: v.to(dev) for k, v in x.items()}
    out = torch.zeros_like(on["logits"])
    launch(ct, on, out)
    assert bool((out[:, :-1] == 1.0).all()) and bool((out[:, -1] == 0.5 - 0.5 * n + 256.0).all())
