"""The operators of msplat.ops together with the training step: learned colours and labels of a scene's Gaussians (GPU).

A feature vector per Gaussian goes through a hidden layer (GELU), dropout and a second layer (sigmoid) to the [N, 3] colours
that msplat_shard_forward_backward_rgb takes; its gradient records give dL/dcolour (columns 10 .. 12 of [N, 16]), which goes
back through the same operators to the weights, and msplat_fused_adam updates those. A label loss on the hidden features
does the same against a table of label embeddings.
"""
import pytest

torch = pytest.importorskip("torch")

import _ops_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu

F, H = 24, 40  # features per Gaussian, hidden width


class Network:
    """Features, two layers and a label table, in 32 bits, with Adam's moments."""

    def __init__(self, n, labels, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s, std=1.0: torch.randn(*s, generator=g, device="cuda") * std  # noqa: E731
        self.p = {"x": r(n, F), "w1": r(H, F, std=F ** -0.5), "b1": r(H, std=0.1), "w2": r(3, H, std=H ** -0.5),
                  "b2": r(3, std=0.1), "table": r(labels, H, std=0.3)}
        self.m = {k: torch.zeros_like(v) for k, v in self.p.items()}
        self.v = {k: torch.zeros_like(v) for k, v in self.p.items()}

    def forward(self, seed, step):
        from msplat import ops
        p, n = self.p, self.p["x"].shape[0]
        self.z1, self.z2 = torch.empty(n, H, device="cuda"), torch.empty(n, 3, device="cuda")
        h = ops.linear_forward(p["x"], p["w1"], p["b1"], activation="gelu", preact=self.z1)
        self.h = ops.dropout(h, 0.2, seed, step)
        return ops.linear_forward(self.h, p["w2"], p["b2"], activation="sigmoid", preact=self.z2)

    def backward(self, dcolour, seed, step, targets=None, weight=0.0):
        """Gradients by name, and the label loss."""
        from msplat import ops
        p, grads = self.p, {}
        dh, grads["w2"], grads["b2"] = ops.linear_backward(self.h, p["w2"], dcolour, preact=self.z2, activation="sigmoid")
        loss = None
        if targets is not None:
            loss, _, dl, grads["table"] = ops.loss_cross_entropy(self.h, p["table"], targets, weight=weight)
            dh += dl
        dh = ops.dropout(dh, 0.2, seed, step)
        grads["x"], grads["w1"], grads["b1"] = ops.linear_backward(p["x"], p["w1"], dh, preact=self.z1, activation="gelu")
        return grads, loss

    def update(self, grads, step, lr=1e-2):
        from msplat import _backend as B
        for k, g in grads.items():
            B.fused_adam(self.p[k], g.contiguous(), self.m[k], self.v[k], lr / (1 - 0.9 ** step), 0.9, 0.999,
                         (1 - 0.999 ** step) ** 0.5, 1e-8)


def scene():
    from _cases import Case
    from msplat import _backend as B
    case = Case("sh1_odd")
    g = B.DeviceGaussians(*case.scene.params(), sh_degree=case.degree)
    return case, g, B.camera_from_oracle(case.ocam), torch.as_tensor(case.gt).cuda()


def render_loss(case, g, cam, gt, rgb):
    """(loss, dL/dcolour as columns of the records) of the scene with these colours."""
    from msplat import _backend as B
    from msplat.sharding import loss_from_parts
    records, parts = torch.empty(g.n, 16, device="cuda"), torch.zeros(3, dtype=torch.float64, device="cuda")
    B.shard_forward_backward_rgb(g, cam, case.degree, case.bg, gt, 0.8, 0.0, 0.2, records, parts, rgb,
                                 rows=(0, (cam.height + 15) // 16))
    return loss_from_parts(parts.cpu(), 0.2, cam.width, cam.height), records[:, 10:13]


def plain_gradients(net, dcolour, keep, targets, weight):
    """The network's gradients by torch's differentiation in 64 bits, from the same dL/dcolour."""
    p = {k: v.double().requires_grad_() for k, v in net.p.items()}
    z1 = p["x"] @ p["w1"].T + p["b1"]
    h = torch.where(keep, z1 * torch.special.ndtr(z1) * (65536 / (65536 - 13107)), torch.zeros_like(z1))
    rgb = torch.sigmoid(h @ p["w2"].T + p["b2"])
    known = (targets >= 0) & (targets < p["table"].shape[0])
    ce = torch.nn.functional.cross_entropy((h @ p["table"].T)[known], targets[known].long()) * weight
    ((rgb * dcolour.double()).sum() + ce).backward()
    return rgb.detach(), {k: v.grad for k, v in p.items()}, float(ce.detach())


def test_learned_colours_and_labels_gradients():
    case, g, cam, gt = scene()
    net = Network(g.n, 37)
    targets = torch.randint(-10, 37, (g.n,), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(9))
    seed, step = 1234, 5
    rgb = net.forward(seed, step)
    _, dcolour = render_loss(case, g, cam, gt, rgb)
    assert dcolour.stride(0) == 16 and bool(dcolour.any())
    grads, loss = net.backward(dcolour, seed, step, targets, weight=0.5)
    keep = torch.from_numpy(R.draws(g.n * H, seed, step) >= 13107).reshape(g.n, H).cuda()
    want_rgb, want, want_loss = plain_gradients(net, dcolour, keep, targets, 0.5)
    # Each value is a few sums of at most N terms in 32 bits one after the other: against the size of the tensor, 64 steps
    # of 2^-20 (a chain of functions, R.FUN) cover them with room.
    tol = 64 * R.FUN
    assert float((rgb.double() - want_rgb).abs().max()) <= tol
    assert abs(float(loss) - want_loss) <= tol * want_loss
    for k in net.p:
        off = float((grads[k].double() - want[k]).norm() / want[k].norm())
        assert off <= tol, (k, off)


def test_learned_colours_against_differences():
    """d(render loss)/d(weights) along a direction, through the rasteriser, against a central difference."""
    case, g, cam, gt = scene()
    net = Network(g.n, 5, seed=3)
    seed, step = 7, 1
    rgb = net.forward(seed, step)
    _, dcolour = render_loss(case, g, cam, gt, rgb)
    grads, _ = net.backward(dcolour, seed, step)
    gen = torch.Generator(device="cuda").manual_seed(11)
    for k in ("w1", "b1", "w2", "b2"):
        # along the gradient, so that the difference is far above the 32-bit image's rounding
        d = grads[k] / grads[k].norm() + 0.1 * torch.randn(net.p[k].shape, generator=gen, device="cuda") / net.p[k].numel() ** 0.5
        e, base, value = 0.02, net.p[k].clone(), []
        for sign in (1, -1):
            net.p[k].copy_(base + sign * e * d)
            value.append(render_loss(case, g, cam, gt, net.forward(seed, step))[0])
        net.p[k].copy_(base)
        want = float((grads[k].double() * d.double()).sum())
        # L1 has kinks where a pixel passes its target and the step is 2% of the weights' size: 5% of the derivative
        assert abs((value[0] - value[1]) / (2 * e) - want) <= 0.05 * abs(want), (k, want, value)


def test_learned_colours_train():
    """A few steps with Adam run, with another mask each step, and leave finite weights that have moved."""
    case, g, cam, gt = scene()
    net = Network(g.n, 37)
    targets = torch.randint(0, 37, (g.n,), device="cuda", dtype=torch.int32)
    before = {k: v.clone() for k, v in net.p.items()}
    for step in range(1, 4):
        rgb = net.forward(42, step)
        loss, dcolour = render_loss(case, g, cam, gt, rgb)
        grads, label_loss = net.backward(dcolour, 42, step, targets, weight=0.1)
        net.update(grads, step)
        assert loss == loss and float(label_loss) > 0
    for k, v in net.p.items():
        assert bool(torch.isfinite(v).all()) and not torch.equal(v, before[k]), k
