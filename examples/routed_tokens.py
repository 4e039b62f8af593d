"""Cameras to routed tokens: the layer entries (hip_layers.h) in the order in
which an actor over this library's sensor planes uses them.

  sensor planes   tb_hip_actor_inputs_device: luma [n, 4, 64, 64]
  stem            8 x 8 patches through one matrix, group norm and SiLU over
                  each camera's 64 patches: the tokens, n * 256 rows
  router          logits, two of eight experts a token, none for a patch that
                  is black throughout; the choices in the experts' order
  experts         4-bit weights: up with SiLU, down with the routing weight
  sum             token + its experts' rows

The weights are random.  The entries' buffers and workspaces are made once for a
batch; an acting step only launches, on the current stream.  What torch computes
between them (patches, planes, logits, the rows' sums) it allocates itself.

    python examples/routed_tokens.py [environments]
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from turbinator_c_amd import features, layers, synth  # noqa: E402

PATCH, PATCHES, CAMERAS = 8, 64, 4
WIDTH, HIDDEN, GROUPS, EXPERTS, TOP = 256, 512, 8, 8, 2
EPS = 1e-5
F32, BF16 = layers.DTYPES["f32"], layers.DTYPES["bf16"]
SILU, NONE = layers.ACTS["silu"], layers.ACTS["none"]
SOFTMAX = layers.SCORES["softmax"]


def done(status: int) -> None:
    if status != 1:
        raise RuntimeError("a layer entry refused its arguments")


class FourBit:
    """A matrix of `rows` rows of k, as codes and scales."""

    def __init__(self, rows: int, k: int):
        self.rows, self.k, padded = rows, k, layers.mx4_padded(k)
        self.codes = torch.empty(rows, padded // 2, dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(rows, padded // 32, dtype=torch.uint8, device="cuda")

    def take(self, x: torch.Tensor, stream) -> "FourBit":
        done(layers.mx4_quantise_device(x, x.stride(0) * x.element_size(), self.codes,
                                        self.scales, self.rows, self.k,
                                        layers.DTYPES[x.dtype], stream))
        return self

    def values(self) -> torch.Tensor:
        v = torch.empty(self.rows, self.k, device="cuda")
        done(layers.mx4_values_device(self.codes, self.scales, v, self.rows, self.k, F32,
                                      torch.cuda.current_stream()))
        return v


class RoutedTokens:
    def __init__(self, environments: int, seed: int = 1):
        self.n = environments
        self.images, self.tokens = environments * CAMERAS, environments * CAMERAS * PATCHES
        rng = torch.Generator().manual_seed(seed)

        def random(*shape, scale):
            return (torch.randn(*shape, generator=rng) * scale).cuda()

        self.stem = random(PATCH * PATCH, WIDTH, scale=0.3).bfloat16()
        self.gamma, self.beta = 1 + random(WIDTH, scale=0.1), random(WIDTH, scale=0.1)
        self.router = random(WIDTH, EXPERTS, scale=0.2).bfloat16()
        up = random(EXPERTS * HIDDEN, WIDTH, scale=WIDTH ** -0.5)
        down = random(EXPERTS * WIDTH, HIDDEN, scale=HIDDEN ** -0.5)
        self.up_bias = random(EXPERTS * HIDDEN, scale=0.1)
        stream = torch.cuda.current_stream()
        self.up = FourBit(*up.shape).take(up, stream)
        self.down = FourBit(*down.shape).take(down, stream)

        def space(*shape, dtype=torch.float32):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        rows = self.tokens * TOP
        self.proprio, self.mission = space(self.n, 91), space(self.n, 49)
        self.tactical, self.prior = space(self.n, 24), space(self.n, 15)
        self.luma = space(self.n, CAMERAS, 64, 64)
        self.token = space(self.tokens, WIDTH, dtype=torch.bfloat16)
        self.mean, self.rstd = space(self.images, GROUPS), space(self.images, GROUPS)
        self.experts = space(self.tokens, TOP, dtype=torch.int32)
        self.weights = space(self.tokens, TOP)
        self.offsets = space(EXPERTS + 1, dtype=torch.int32)
        self.row_token = space(rows, dtype=torch.int32)
        self.positions = space(self.tokens, TOP, dtype=torch.int32)
        self.row_weight = space(rows)
        self.token4, self.hidden4 = FourBit(self.tokens, WIDTH), FourBit(rows, HIDDEN)
        self.hidden = space(rows, HIDDEN, dtype=torch.bfloat16)
        self.part = space(rows, WIDTH, dtype=torch.bfloat16)
        sizes = (self.images, PATCHES, WIDTH, GROUPS, BF16)
        self.norm_space = space(layers.group_norm_workspace_bytes(*sizes), dtype=torch.uint8)
        self.grad_space = space(layers.group_norm_workspace_bytes(*sizes, backward=True),
                                dtype=torch.uint8)
        self.order_space = space(
            layers.expert_order_workspace_bytes(self.tokens, EXPERTS, TOP), dtype=torch.uint8)

    def act(self, obs, mission, cameras) -> torch.Tensor:
        """The routed tokens [tokens, WIDTH] of the environments' inputs."""
        stream = torch.cuda.current_stream()
        done(features.actor_inputs_device(obs, mission, cameras, self.proprio, self.mission,
                                          self.tactical, self.prior, None, self.luma, self.n,
                                          stream))
        side = 64 // PATCH
        patch = self.luma.view(self.images, side, PATCH, side, PATCH).transpose(2, 3)
        patch = patch.reshape(self.tokens, PATCH * PATCH)
        self.valid = (patch > -0.5).any(1)
        self.planes = patch.bfloat16() @ self.stem
        row = WIDTH * 2
        done(layers.group_norm_device(self.planes, PATCHES * row, row, self.gamma, self.beta,
                                      self.token, self.mean, self.rstd, self.norm_space,
                                      self.images, PATCHES, WIDTH, GROUPS, EPS, SILU, BF16,
                                      stream))
        self.logits = self.token @ self.router
        done(layers.route_device(self.logits, EXPERTS * 2, None, self.valid, self.experts,
                                 self.weights, self.tokens, EXPERTS, TOP, 1, 1, SOFTMAX, True,
                                 1.0, BF16, stream))
        done(layers.expert_order_device(self.experts, self.weights, self.offsets, self.row_token,
                                        self.positions, self.row_weight, self.order_space,
                                        self.tokens, EXPERTS, TOP, stream))
        self.token4.take(self.token, stream)
        rows = self.tokens * TOP
        done(layers.mx4_product_device(self.token4.codes, self.token4.scales, self.tokens,
                                       self.row_token, self.up.codes, self.up.scales,
                                       self.offsets, self.up_bias, None, self.hidden, rows,
                                       HIDDEN, WIDTH, EXPERTS, SILU, BF16, stream))
        self.hidden4.take(self.hidden, stream)
        done(layers.mx4_product_device(self.hidden4.codes, self.hidden4.scales, rows, None,
                                       self.down.codes, self.down.scales, self.offsets, None,
                                       self.row_weight, self.part, rows, WIDTH, HIDDEN, EXPERTS,
                                       NONE, BF16, stream))
        return self.token + self.summed(self.part)

    def summed(self, part) -> torch.Tensor:
        """Each token's rows added up; a choice without a row adds nothing."""
        there = (self.positions >= 0).unsqueeze(2)
        return (part[self.positions.clamp(min=0).long()] * there).sum(1)

    def learn(self, dout) -> dict:
        """Gradients of router, gamma and beta and of the stem's planes for the
        gradient of act's result, after it.  The experts are fixed, and so is
        what they read: a token's gradient comes past them and through the
        router."""
        stream = torch.cuda.current_stream()
        # What each choice's weight multiplies: the experts' rows without it.
        rows = self.tokens * TOP
        plain = torch.empty_like(self.part)
        done(layers.mx4_product_device(self.hidden4.codes, self.hidden4.scales, rows, None,
                                       self.down.codes, self.down.scales, self.offsets, None,
                                       None, plain, rows, WIDTH, HIDDEN, EXPERTS, NONE, BF16,
                                       stream))
        picked = plain[self.positions.clamp(min=0).long()].float()
        dweights = (picked * dout.float().unsqueeze(1)).sum(2)
        dlogits = torch.empty_like(self.logits)
        done(layers.route_backward_device(self.logits, EXPERTS * 2, self.experts, dweights,
                                          dlogits, self.tokens, EXPERTS, TOP, SOFTMAX, True, 1.0,
                                          BF16, stream))
        dtoken = dout + dlogits @ self.router.t().contiguous()
        dplanes = torch.empty_like(self.planes)
        dgamma, dbeta = torch.empty_like(self.gamma), torch.empty_like(self.beta)
        row = WIDTH * 2
        done(layers.group_norm_backward_device(self.planes, PATCHES * row, row, dtoken,
                                               PATCHES * row, row, self.gamma, self.beta,
                                               self.mean, self.rstd, dplanes, dgamma, dbeta,
                                               self.grad_space, self.images, PATCHES, WIDTH,
                                               GROUPS, SILU, BF16, stream))
        return {"router": self.token.t().contiguous() @ dlogits, "gamma": dgamma, "beta": dbeta,
                "planes": dplanes, "dweights": dweights, "dlogits": dlogits, "dtoken": dtoken}


def main() -> None:
    n = int(sys.argv[1]) if len(sys.argv) > 1 else 64
    batch = synth.make_batch(n)
    inputs = [torch.from_numpy(a).cuda() for a in (batch.obs, batch.mission, batch.cameras)]
    net = RoutedTokens(n)

    def time(call, times=20):
        for _ in range(3):
            call()
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        for _ in range(times):
            call()
        end.record()
        end.synchronize()
        return begin.elapsed_time(end) / times * 1e3

    out = net.act(*inputs)
    counts = net.offsets.diff().tolist()
    print(f"{n} environments, {net.tokens} tokens of {WIDTH}, {TOP} of {EXPERTS} experts")
    print(f"rows of each expert: {counts}; black patches: {int((~net.valid).sum())}")
    print(f"mean |token| {out.float().abs().mean():.4f}")
    print(f"acting   {time(lambda: net.act(*inputs)):8.1f} us")
    dout = torch.randn_like(out)
    print(f"learning {time(lambda: net.learn(dout)):8.1f} us")


if __name__ == "__main__":
    main()
