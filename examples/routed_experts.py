"""A layer of routed experts, forwards and backwards, with the operators of ``nacho_b200.nacho``: a router gives every token its best experts, an
expert is a gated pair of 8-bit products, and the results come back weighted by the router.

    python -m examples.routed_experts [--tokens 1024] [--experts 16] [--best 2] [--width 512] [--hidden 1024] [--halves] [--clip 0.5]

prints the loss of a few steps of gradient descent on a fixed random target; it falls. With --halves the gated product is one call in 16 bits, forwards and
backwards, and only the way down is multiplied in 8; with --clip the gradients of the weights are scaled to that norm at most."""
import argparse

import torch

from nacho_b200 import nacho


def route(scores, best, capacity):
    """The router's decision as CSR: every token's `best` experts, softmax over their scores. An entry beyond an expert's capacity, counted
    in the tokens' order, is dropped."""
    tokens, experts = scores.shape
    top, expert = torch.topk(scores, best, dim=1)
    weight = torch.softmax(top, dim=1)
    taken = torch.nn.functional.one_hot(expert.flatten(), experts).cumsum(0).gather(1, expert.flatten()[:, None]).squeeze(1)
    expert = torch.where(taken <= capacity, expert.flatten(), -1)
    offsets = torch.arange(0, tokens * best + 1, best, dtype=torch.int32, device=scores.device)
    return nacho.CSR_gpu(offsets, expert.int(), weight.flatten(), (tokens, experts)), weight, expert


def forward(r, x, up, down):
    """y, and what the way back needs. up: (experts, 2 hidden, width), down: (experts, width, hidden), both in 8 bits."""
    order, xs = nacho.gpu_expert_sort_fp8(r, x)
    both = nacho.gpu_fp8_product(xs, up, order)
    gate, value = both.chunk(2, dim=1)
    hidden = torch.nn.functional.silu(gate) * value
    z = nacho.gpu_fp8_product(nacho.to_fp8_rows(hidden), down, order)
    return nacho.gpu_expert_unsort(r, order, z), (order, both, hidden, z)


def backward(r, x, up, down, kept, dy):
    """Gradients of the tokens, of the gate weights and of both products' weights."""
    order, both, hidden, z = kept
    dz, dgate = nacho.gpu_expert_unsort_grad(r, order, z, dy)
    dhidden, ddown = nacho.gpu_fp8_product_grad(dz, hidden, down, order)
    gate, value = both.float().chunk(2, dim=1)
    soft = torch.sigmoid(gate)
    dboth = torch.cat([dhidden * value * soft * (1 + gate * (1 - soft)), dhidden * gate * soft], dim=1).to(x.dtype)
    dxs, dup = nacho.gpu_fp8_product_grad(dboth, nacho.gpu_expert_sort(r, x)[1], up, order)
    return nacho.gpu_expert_sort_grad(order, dxs), dgate, dup, ddown


def forward_halves(r, x, up, down):
    """The same with up in 16 bits."""
    order, xs = nacho.gpu_expert_sort(r, x)
    hidden, both = nacho.gpu_gated_product(xs, up, order, keep=True)
    z = nacho.gpu_fp8_product(nacho.to_fp8_rows(hidden), down, order)
    return nacho.gpu_expert_unsort(r, order, z), (order, xs, both, hidden, z)


def backward_halves(r, up, down, kept, dy):
    order, xs, both, hidden, z = kept
    dz, dgate = nacho.gpu_expert_unsort_grad(r, order, z, dy)
    dhidden, ddown = nacho.gpu_fp8_product_grad(dz, hidden, down, order)
    dxs, dup = nacho.gpu_gated_product_grad(dhidden, both, xs, up, order)
    return nacho.gpu_expert_sort_grad(order, dxs), dgate, dup, ddown


def descend(tokens=1024, experts=16, best=2, width=512, hidden=1024, steps=5, rate=0.5, halves=False, clip=None):
    g = torch.Generator(device="cuda").manual_seed(0)
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    x, target = draw(tokens, width).bfloat16(), draw(tokens, width)
    router, up, down = draw(width, experts) * width ** -0.5, draw(experts, 2 * hidden, width) * width ** -0.5, draw(experts, width, hidden) * hidden ** -0.5
    losses = []
    for _ in range(steps):
        scores = x.float() @ router
        r, weight, expert = route(scores, best, capacity=2 * tokens * best // experts + 1)
        up8, down8 = up.bfloat16() if halves else nacho.to_fp8_tiles(up), nacho.to_fp8_tiles(down)
        y, kept = forward_halves(r, x, up8, down8) if halves else forward(r, x, up8, down8)
        off = y.float() - target
        losses.append(float((off * off).mean()))
        dy = (off * (2 / width)).bfloat16()
        dx, dgate, dup, ddown = backward_halves(r, up8, down8, kept, dy) if halves else backward(r, x, up8, down8, kept, dy)
        if clip is not None:
            nacho.gpu_clip_gradients([dup, ddown], clip)
        # the softmax over a token's best scores, then the router's matrix
        dgate = dgate.view(tokens, best)
        dtop = weight * (dgate - (dgate * weight).sum(1, keepdim=True))
        top = torch.topk(scores, best, dim=1).indices
        router -= rate / tokens * x.float().t() @ torch.zeros_like(scores).scatter_(1, top, dtop)
        up -= rate * experts / tokens * dup
        down -= rate * experts / tokens * ddown
    return losses, dx


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("tokens", 1024), ("experts", 16), ("best", 2), ("width", 512), ("hidden", 1024), ("steps", 5)):
        parser.add_argument(f"--{name}", type=int, default=value)
    parser.add_argument("--halves", action="store_true")
    parser.add_argument("--clip", type=float)
    for loss in descend(**vars(parser.parse_args()))[0]:
        print(f"loss {loss:.5f}")
