"""Self-attention head of the CAPL model - same constructor, parameter names
(q_map/k_map/v_map.weight) and forward contract as the reference
model/attention.py:10-48.  On the GPU with the reference's head size (64) the
softmax(q^T k / sqrt(d)) v product runs as ONE fused HIP kernel (K5, gfs3d_attention_forward_f32: no (B,N,N) tensor,
dropout decisions from a counter-based hash so that the backward regenerates them); other head sizes use the torch
formulation below.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F


class SelfAttention(nn.Module):
    def __init__(self, in_channel, out_channel=None, attn_dropout=0.1):
        super().__init__()
        self.in_channel = in_channel
        self.out_channel = in_channel if out_channel is None else out_channel
        self.temperature = self.out_channel ** 0.5
        for name in ("q_map", "k_map", "v_map"):          # registration order = reference order
            setattr(self, name, nn.Conv1d(in_channel, self.out_channel, 1, bias=False))
        self.dropout = nn.Dropout(attn_dropout)
        self._forced_keep_mask = None      # tests: (B,N,N) bool, replaces the RNG draw of nn.Dropout

    def forward(self, x, cloud=None):
        """x (B, in_channel, N) -> (B, out_channel, N).  `cloud` is WindowSelfAttention's; unused here."""
        q, k, v = self.q_map(x), self.k_map(x), self.v_map(x)
        if x.is_cuda and self.out_channel == 64:
            from gfs3d import ops
            p = float(self.dropout.p) if self.training else 0.0
            mask = self._forced_keep_mask if (self.training and self._forced_keep_mask is not None) else None
            # one draw from torch's generator per call: reproducible under torch.manual_seed like nn.Dropout
            seed = int(torch.randint(0, 2 ** 62, (1,)).item()) if (p > 0.0 and mask is None) else 0
            return ops.attention(q, k, v, 1.0 / self.temperature, p, seed, mask)
        return self._attend_torch(q, k, v)

    def forward_pm(self, x_pm, cloud=None):
        """x_pm (B, N, in_channel) point-major -> (B, 64, N): the three projections as ONE HIP GEMM on the concatenated
        weights (gfs3d_linear_forward_f32, channel-first q / k / v straight from its epilogue), then the fused K5 kernel."""
        from gfs3d import ops
        if self.out_channel != 64 or not x_pm.is_cuda:
            raise NotImplementedError("SelfAttention.forward_pm: head size 64 on the GPU")
        w = torch.cat((self.q_map.weight, self.k_map.weight, self.v_map.weight), dim=0)
        q, k, v = ops.linear_cf(x_pm, w)
        p = float(self.dropout.p) if self.training else 0.0
        mask = self._forced_keep_mask if (self.training and self._forced_keep_mask is not None) else None
        seed = int(torch.randint(0, 2 ** 62, (1,)).item()) if (p > 0.0 and mask is None) else 0
        return ops.attention(q, k, v, 1.0 / self.temperature, p, seed, mask)

    def _attend_torch(self, q, k, v):
        attn = torch.bmm(q.transpose(1, 2) / self.temperature, k)
        attn = F.softmax(attn, dim=-1)
        if self._forced_keep_mask is not None and self.training:
            attn = attn * (self._forced_keep_mask.to(attn.dtype) / (1.0 - self.dropout.p))
        else:
            attn = self.dropout(attn)
        return torch.bmm(attn, v.transpose(1, 2)).transpose(1, 2)


class WindowSelfAttention(nn.Module):
    """Attention learner whose cost grows with the number of points, not with its square: the points are put in the order of a
    space-filling curve (gfs3d.morton) and pass through `layers` pre-norm layers - RMS norm of the residual stream, one projection
    to q, k, v, rotary positions along the curve, attention over `window` points to either side and the curve's first `sinks`
    points, output projection - then a last norm and a projection to out_channel.  Takes SelfAttention's place in the models
    (args.att_window > 0; no counterpart in the reference) with its call signature and the network's input cloud, whose first three
    channels are the coordinates.  GPU only.  Under gfs3d.ops.compute("bf16" / "f16") the branches are that type beside an fp32 stream."""

    def __init__(self, in_channel, out_channel=None, window=128, sinks=4, layers=1, heads=4, key_heads=2, head_dim=64):
        super().__init__()
        if layers < 1:
            raise ValueError(f"WindowSelfAttention: layers must be at least 1, got {layers} (args.att_layers)")
        self.in_channel = in_channel
        self.out_channel = in_channel if out_channel is None else out_channel
        self.window, self.sinks, self.heads, self.key_heads, self.head_dim = int(window), int(sinks), heads, key_heads, head_dim
        wide = (heads + 2 * key_heads) * head_dim
        self.norms = nn.ParameterList([nn.Parameter(torch.ones(in_channel)) for _ in range(layers + 1)])
        self.qkv_maps = nn.ModuleList([nn.Linear(in_channel, wide, bias=False) for _ in range(layers)])
        self.out_maps = nn.ModuleList([nn.Linear(heads * head_dim, in_channel, bias=False) for _ in range(layers)])
        self.head_map = nn.Linear(in_channel, self.out_channel, bias=False)
        self.register_buffer("freqs", self._frequencies(), persistent=False)

    def _apply(self, fn, *args, **kwargs):
        """Casts reach buffers too and round the frequencies (fp32: 7e-4 rad at position 65536): they are formed anew in 64 bits."""
        super()._apply(fn, *args, **kwargs)
        self.freqs = self._frequencies().to(self.freqs.device)
        return self

    def _frequencies(self):
        from gfs3d import ops
        return ops.rotary_frequencies(self.head_dim // 2)[0]

    def forward(self, x, cloud):
        """x (B, in_channel, N), cloud (B, C >= 3, N) -> (B, out_channel, N)."""
        return self.forward_pm(x.transpose(1, 2), cloud)

    def forward_pm(self, x_pm, cloud):
        """x_pm (B, N, in_channel) point-major -> (B, out_channel, N)."""
        from gfs3d import ops
        from gfs3d.morton import morton_order
        order, rank = morton_order(cloud[:, :3].detach())
        place = torch.arange(x_pm.shape[1], device=x_pm.device, dtype=torch.int32)
        dtype = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[ops.get_compute()]
        H, G, D = self.heads, self.key_heads, self.head_dim
        stream = x_pm.gather(1, order[:, :, None].expand(-1, -1, x_pm.shape[2]))
        branch = None
        for norm, qkv_map, out_map in zip(self.norms, self.qkv_maps, self.out_maps):
            if branch is None:
                y = ops.rms_norm(stream, norm).to(dtype)
            else:
                y, stream = ops.rms_norm(branch, norm, residual=stream)
            qkv = F.linear(y, qkv_map.weight.to(dtype)).unflatten(2, (H + 2 * G, D))
            q, k = ops.rotary(qkv[:, :, :H], qkv[:, :, H:H + G], place, self.freqs)
            o = ops.window_attention(q, k, qkv[:, :, H + G:], left=self.window, right=self.window, sinks=self.sinks)
            branch = F.linear(o.flatten(2), out_map.weight.to(dtype))
        y, _ = ops.rms_norm(branch, self.norms[len(self.qkv_maps)], residual=stream)
        out = F.linear(y, self.head_map.weight.to(dtype)).float()
        return out.gather(1, rank[:, :, None].expand(-1, -1, self.out_channel)).transpose(1, 2)


def attention_learner(args, in_channel, out_channel):
    """The models' attention learner: the reference's SelfAttention, or WindowSelfAttention where args.att_window is positive
    (args.att_sinks, args.att_layers: its sinks and depth)."""
    window = int(getattr(args, "att_window", 0) or 0)
    if window <= 0:
        return SelfAttention(in_channel, out_channel)
    return WindowSelfAttention(in_channel, out_channel, window, int(getattr(args, "att_sinks", 4)), int(getattr(args, "att_layers", 1)))
