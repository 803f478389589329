"""The operators together, as they are used: a small bf16 model trained with
its gradients clipped in place, then its weights quantized to 4 bits and one
token after another run through them; a captured step included."""
import pytest

pytestmark = pytest.mark.gpu


def _model(cuda):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(0)
    shapes = [(200, 72), (72, 200), (72,)]
    return [(torch.randn(s, generator=gen, device=cuda) * 0.1).to(torch.bfloat16).requires_grad_() for s in shapes]


def _forward(p, x):
    import torch
    return (torch.relu(x @ p[0].t()) @ p[1].t()) * (1 + p[2])


def test_train_clip_quantize_decode(cuda, qrc):
    import torch
    p = _model(cuda)
    gen = torch.Generator(device="cuda").manual_seed(1)
    lists, master = None, [v.detach().float() for v in p]
    for step in range(6):
        x = torch.randn(33, 72, generator=gen, device=cuda).to(torch.bfloat16)
        loss = (_forward(p, x).float() - 3 * x.float()).square().sum()
        for v in p:
            if v.grad is not None:
                v.grad.zero_()                               # the gradients stay where they are
        loss.backward()
        if lists is None:
            lists = qrc.TensorList([v.grad for v in p])
        raw = [v.grad.double() for v in p]
        want = float(sum((g * g).sum() for g in raw).sqrt())
        norm = lists.clip_norm(1.0)
        assert abs(float(norm) - want) <= 5 * 2.0 ** -24 * want
        assert want > 1.0
        for v, g in zip(p, raw):                             # factor and product in float, rounded once to bf16
            y = g / (want + 1e-6)
            assert ((v.grad.double() - y).abs() <= (2.0 ** -8 * 1.001) * y.abs() + 1e-40).all()
        with torch.no_grad():
            for v, m in zip(p, master):
                m -= 0.05 * v.grad.float()
                v.copy_(m)
    w = [qrc.quant_w4(v.detach(), group=32) for v in p[:2]]
    for _ in range(4):
        x = torch.randn(1, 72, generator=gen, device=cuda).to(torch.bfloat16)
        h = torch.relu(w[0].matvec(x))
        y = w[1].matvec(h, out_dtype=torch.float32)
        v = [a.dequant(dtype=torch.float32).double() for a in w]
        first = x.double() @ v[0].t()
        # bf16 hidden values: half a step each, and the float sums before it
        assert ((w[0].matvec(x).double() - first).abs() <= 2.0 ** -8 * first.abs() + 90 * 2.0 ** -23 * (x.double().abs() @ v[0].abs().t())).all()
        second = h.double() @ v[1].t()
        assert ((y.double() - second).abs() <= 220 * 2.0 ** -23 * (h.double().abs() @ v[1].abs().t())).all()


def test_captured_training_step(cuda, qrc):
    """backward and clip in one graph, replayed on new data."""
    import torch
    p = _model(cuda)
    x = torch.randn(33, 72, device=cuda).to(torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            for v in p:
                v.grad = None
            _forward(p, x).float().square().sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    grads = [torch.zeros_like(v) for v in p]
    for v, g in zip(p, grads):
        v.grad = g
    tensors = qrc.TensorList(grads)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for v in grads:
            v.zero_()
        _forward(p, x).float().square().sum().backward()
        norm = tensors.clip_norm(0.5)
    for seed in range(3):
        x.copy_(torch.randn(33, 72, device=cuda, generator=torch.Generator(device="cuda").manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        clipped = float(torch.stack([v.double().square().sum() for v in grads]).sum().sqrt())
        assert float(norm) > 0.5
        # every element is off by half a bf16 step at most, so the norm is too
        assert abs(clipped - 0.5) <= 0.5 * (2.0 ** -8 + 2.0 ** -20)
