"""A network that goes along the rows of equirectangular images in both directions, next to a mapped
convolution, trained with AdamW for some steps; and a causal block of the same parts that answers token by
token from a kept state.

    python -m mappedconvolutions_amd.examples.scan_recurrence

Synthetic data: the network learns the running mean of every row up to a pixel, which a 3x3 convolution
cannot see and a recurrence can.
"""
import torch
import torch.nn as nn

from ..nn import GatedRecurrence, GroupNormActivation, MappedConvolution
from ..util import AdamW, latitude_map


class ScanBlock(nn.Module):
    """Norm and activation, one projection, the recurrence, projection: [B, L, channels] -> the same,
    added.  The channels' memories reach from a token to `longest` of them."""

    def __init__(self, channels, groups=8, longest=64, reverse=False, activation='silu'):
        super().__init__()
        self.norm = GroupNormActivation(groups, channels, activation=activation)
        self.project = nn.Linear(channels, 3 * channels)
        self.scan = GatedRecurrence(reverse)
        self.join = nn.Linear(channels, channels, bias=False)
        with torch.no_grad():
            self.project.bias.zero_()
            self.project.bias[channels:2 * channels] = torch.linspace(1, longest, channels).log()

    def forward(self, x, lengths=None):
        out, _ = self.scan(*self.project(self.norm(x)).chunk(3, -1), lengths=lengths)
        return x + self.join(out)


class CausalBlock(nn.Module):
    """The same for tokens that come one by one, each normed by itself."""

    def __init__(self, channels, groups=8, longest=64):
        super().__init__()
        self.block = ScanBlock(channels, groups, longest)

    def parts(self, x):
        b = self.block
        return b.project(b.norm(x.flatten(0, 1)).view(x.shape)).chunk(3, -1)

    def forward(self, x):
        return x + self.block.join(self.block.scan(*self.parts(x))[0])

    def step(self, x, state):
        """The next tokens [B, L, channels] from the state float32 [B, channels], changed in place."""
        return x + self.block.join(self.block.scan.step(state, *self.parts(x)))


class ScanNetwork(nn.Module):
    """A mapped 3x3 convolution, every row forward and backward, one value a pixel."""

    def __init__(self, channels=64):
        super().__init__()
        self.convolution = MappedConvolution(1, channels, 9)
        self.forward_rows = ScanBlock(channels)
        self.backward_rows = ScanBlock(channels, reverse=True)
        self.read = nn.Linear(channels, 1)

    def forward(self, images, sample_map):
        x = self.convolution(images, sample_map).permute(0, 2, 3, 1)      # B H W C
        B, H, W, C = x.shape
        x = self.backward_rows(self.forward_rows(x.reshape(B * H, W, C)))
        return self.read(x).view(B, H, W)


def running_mean(images):
    """The sum of a row up to a pixel over the root of its length: of variance one everywhere."""
    count = torch.arange(1, images.shape[-1] + 1, device=images.device)
    return images.float().cumsum(-1) / count.sqrt()


def train(steps=60, height=16, width=64, batch=4, seed=0, device='cuda', bits=32, rate=3e-3,
          dtype=torch.float32):
    """-> (the network, the loss of every step)."""
    torch.manual_seed(seed)
    net = ScanNetwork().to(device, dtype)
    sample_map = latitude_map(height, width).to(device)
    optimizer = AdamW(net.parameters(), lr=rate, bits=bits, max_norm=1.0)
    losses = []
    for _ in range(steps):
        images = torch.randn(batch, 1, height, width, device=device).to(dtype)
        optimizer.zero_grad()
        loss = (net(images, sample_map).float() - running_mean(images[:, 0])).square().mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return net, torch.stack(losses).tolist()


def serve(tokens=50, channels=128, batch=3, dtype=torch.bfloat16, seed=0, device='cuda'):
    """A causal block over a whole sequence and over the same one token by token -> both outputs."""
    torch.manual_seed(seed)
    block = CausalBlock(channels).to(device, dtype)
    x = torch.randn(batch, tokens, channels, device=device).to(dtype)
    state = torch.zeros(batch, channels, device=device)
    with torch.no_grad():
        whole = block(x)
        one_by_one = [block.step(x[:, t:t + 1], state) for t in range(tokens)]
    return whole, torch.cat(one_by_one, 1)


if __name__ == '__main__':
    for bits in (32, 8):
        _, history = train(bits=bits)
        print('moments in %d bits, loss: first %.4f, last %.4f' % (bits, history[0], history[-1]))
    a, b = serve()
    print('whole sequence against one by one: %.2g' % (a - b).abs().max().item())
