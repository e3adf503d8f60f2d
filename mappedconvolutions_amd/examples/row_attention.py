"""Attention along the rows of equirectangular images next to a mapped convolution, trained for some
steps, and a causal decoder of the same parts that answers token by token.

    python -m mappedconvolutions_amd.examples.row_attention

Synthetic data: the network learns to undo a turn of the panorama (a shift of every row by a quarter
of its columns), which a 3x3 convolution cannot see and attention on the circle can.
"""
import torch
import torch.nn as nn

from ..nn import MappedConvolution, QKNormRotation, RelativeAttention
from ..util import clip_grad_norm_, distance_buckets, latitude_map, rotation_table


class HeadsOfTokens(nn.Module):
    """Projection, norm and rotation, attention, projection: [B, L, channels] -> the same, added."""

    def __init__(self, channels, heads, key_heads, buckets, zero, num_buckets, causal=False):
        super().__init__()
        self.heads, self.key_heads, self.head_dim = heads, key_heads, channels // heads
        self.project = nn.Linear(channels, (heads + 2 * key_heads) * self.head_dim, bias=False)
        self.norm = QKNormRotation(self.head_dim)
        self.attention = RelativeAttention(heads, buckets, zero, num_buckets, causal=causal)
        self.join = nn.Linear(channels, channels, bias=False)

    def parts(self, x, cos, sin, positions=None):
        packed = self.project(x).unflatten(-1, (-1, self.head_dim))
        q, k, v = packed.split([self.heads, self.key_heads, self.key_heads], 2)
        return (*self.norm(q, k, cos, sin, positions), v)

    def forward(self, x, cos, sin):
        return x + self.join(self.attention(*self.parts(x, cos, sin)).flatten(-2))

    def step(self, x, cos, sin, cache, lengths):
        """The next token of every sequence, x [B, 1, channels], at position lengths[b] (int32); its
        key and value go into the cache [2, B, places, key heads, head_dim]."""
        at = lengths.long()
        q, k, v = self.parts(x, cos, sin, at[:, None])
        which = torch.arange(x.shape[0], device=x.device)
        cache[0, which, at], cache[1, which, at] = k[:, 0], v[:, 0]
        out = self.attention(q, cache[0], cache[1], query_start=lengths, key_lengths=lengths + 1)
        return x + self.join(out.flatten(-2))


class RowNetwork(nn.Module):
    """A mapped 3x3 convolution, attention along every row, one value a pixel."""

    def __init__(self, width, channels=64, heads=4, key_heads=2, num_buckets=32):
        super().__init__()
        self.convolution = MappedConvolution(1, channels, 9)
        buckets, zero = distance_buckets(num_buckets, circle=width)
        self.rows = HeadsOfTokens(channels, heads, key_heads, buckets, zero, num_buckets)
        self.read = nn.Linear(channels, 1)
        # (their bits as whole numbers: a network that is cast keeps its angles in float32)
        angles = torch.stack(rotation_table(width, channels // heads, circle=True))
        self.register_buffer('angles', angles.view(torch.int32))

    def forward(self, images, sample_map):
        x = self.convolution(images, sample_map).permute(0, 2, 3, 1)      # B H W C
        B, H, W, C = x.shape
        cos, sin = self.angles.view(torch.float32)
        y = self.rows(x.reshape(B * H, W, C), cos, sin)
        return self.read(y).view(B, H, W)


def train(steps=60, height=16, width=64, batch=4, seed=0, device='cuda', max_norm=1.0, rate=3e-3):
    """-> the loss of every step."""
    torch.manual_seed(seed)
    net = RowNetwork(width).to(device)
    sample_map = latitude_map(height, width).to(device)
    optimizer = torch.optim.Adam(net.parameters(), lr=rate)
    losses = []
    for _ in range(steps):
        images = torch.randn(batch, 1, height, width, device=device)
        wanted = images[:, 0].roll(width // 4, -1)
        optimizer.zero_grad()
        loss = (net(images, sample_map) - wanted).square().mean()
        loss.backward()
        clip_grad_norm_(net.parameters(), max_norm)
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def serve(tokens=50, channels=128, batch=3, dtype=torch.bfloat16, seed=0, device='cuda'):
    """A causal block over a whole sequence and over the same one token by token -> both outputs."""
    torch.manual_seed(seed)
    buckets, zero = distance_buckets(32, reach=128)
    block = HeadsOfTokens(channels, 4, 2, buckets, zero, 32, causal=True).to(device, dtype)
    nn.init.normal_(block.attention.table)
    cos, sin = rotation_table(tokens, channels // 4, device=device)
    x = torch.randn(batch, tokens, channels, device=device, dtype=dtype)
    cache = torch.zeros(2, batch, tokens, 2, channels // 4, device=device, dtype=dtype)
    with torch.no_grad():
        whole = block(x, cos, sin)
        one_by_one = []
        for t in range(tokens):
            lengths = torch.full((batch,), t, dtype=torch.int32, device=device)
            one_by_one.append(block.step(x[:, t:t + 1], cos, sin, cache, lengths))
    return whole, torch.cat(one_by_one, 1)


if __name__ == '__main__':
    history = train()
    print('loss: first %.4f, last %.4f' % (history[0], history[-1]))
    a, b = serve()
    print('whole sequence against one by one: %.2g' % (a - b).abs().max().item())
