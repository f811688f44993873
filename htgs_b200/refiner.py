"""A small network over the Gaussians of a scene, from the sequence operators: it reads the raw parameters in the order of a space-filling curve and
returns refined ones, which go on into `glue.activate` and the rasterizer.

    refiner = GaussianRefiner(width=256, layers=4).cuda()
    refined = refiner(raw)                                            # in training: differentiable in its weights and in raw
    scales, rotations, opacities = glue.activate(refined["scales"], refined["rotations"], refined["opacities"])
    image = diff_rasterize(refined["positions"], scales, rotations, opacities, refined["sh_0"], sh_rest, densification_info, settings, False)

Each layer adds to a residual stream what a gated recurrence along the curve makes of it: norm, projection to values and gates, recurrence (forwards and
backwards in turn), projection back.  The raw parameters go into the first projection in 32 bits: with the three bits of an 8-bit code neighbours
along the curve would be one number to the network.  The others are 8-bit products: in training the norm is 16-bit and they code their operands themselves; `freeze()` codes their weights
once, and from then on `infer` has the norm leave 8-bit codes and the projections take them.  (No counterpart in the reference.)
"""
from __future__ import annotations

from typing import Dict, Optional

import torch

from .sequence import add_rms_norm, add_rms_norm_fp8, fp8_linear, fp8_matmul, gated_scan, quantize_fp8

# raw parameters per Gaussian that the network reads and refines
PARAMETERS = (("positions", 3), ("scales", 3), ("rotations", 4), ("opacities", 1), ("sh_0", 3))
CHANNELS = sum(width for _, width in PARAMETERS)


def curve_order(positions: torch.Tensor, offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Indices that sort Gaussians along the Morton curve through cubic cells, 2^20 along the longest side of the bounding box of their finite positions (others
    lie at its faces).  With the `offsets` at which packed scenes begin, each scene has its own box and its own curve: it gets the order that it has alone."""
    if positions.shape[0] == 0:
        return torch.empty(0, dtype=torch.long, device=positions.device)
    finite = positions.isfinite()
    least, most = positions.masked_fill(~finite, float("inf")), positions.masked_fill(~finite, float("-inf"))
    if offsets is None:
        low, high = least.amin(dim=0), most.amax(dim=0)
    else:
        row = torch.arange(positions.shape[0], device=positions.device)
        scene = torch.bucketize(row, offsets[1:-1].long(), right=True)
        scenes = offsets.numel() - 1
        parts = max(1, 4096 // scenes)                       # of a scene's rows, so that few of them meet at one value (1 M rows in two scenes: 5.2 ms in one part each)
        at = (scene * parts + row % parts)[:, None].expand(-1, 3)
        low, high = (torch.full((scenes * parts, 3), none, dtype=positions.dtype, device=positions.device).scatter_reduce_(0, at, ends, reduce).view(scenes, parts, 3)
                     for none, ends, reduce in ((float("inf"), least, "amin"), (float("-inf"), most, "amax")))
        low, high = low.amin(dim=1)[scene], high.amax(dim=1)[scene]
    most_cell = 2 ** 20 - 1            # so many, and cubes, that a few Gaussians far from the others leave these enough of them in each direction
    side = (high - low).amax(dim=-1, keepdim=True).clamp(min=1e-12)
    cell = ((positions.float() - low) / side * most_cell).nan_to_num().clamp(0, most_cell).long()
    for shift, mask in ((32, 0x1F00000000FFFF), (16, 0x1F0000FF0000FF), (8, 0x100F00F00F00F00F), (4, 0x10C30C30C30C30C3), (2, 0x1249249249249249)):
        cell = (cell | cell << shift) & mask                     # bit i goes to bit 3 i
    order = torch.argsort(cell[:, 0] | cell[:, 1] << 1 | cell[:, 2] << 2, stable=True)
    return order if offsets is None else order[torch.argsort(scene[order], stable=True)]


class GaussianRefiner(torch.nn.Module):
    def __init__(self, width: int = 256, layers: int = 4, dtype: torch.dtype = torch.bfloat16, step: float = 0.01):
        super().__init__()
        self.width, self.layers, self.step = width, layers, step

        def weight(rows, columns, scale=1.0):
            return torch.nn.Parameter((torch.randn(rows, columns) * scale * columns ** -0.5).to(dtype))

        self.embed = weight(width, CHANNELS)
        self.norms = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(width, dtype=dtype)) for _ in range(layers + 1)])
        self.enter = torch.nn.ParameterList([weight(2 * width, width) for _ in range(layers)])       # values, then gates
        self.leave = torch.nn.ParameterList([weight(width, width, 0.5) for _ in range(layers)])
        self.head = weight(CHANNELS, width)
        self._frozen = None

    def freeze(self) -> "GaussianRefiner":
        """Codes the weights for `infer`; to be called again when they have changed."""
        with torch.no_grad():
            self._frozen = {"embed": self.embed.detach().to(torch.float32, copy=True), "head": quantize_fp8(self.head, 128), "enter": [quantize_fp8(w, 128) for w in self.enter],
                            "leave": [quantize_fp8(w, 128) for w in self.leave]}
        return self

    def _read(self, raw: Dict[str, torch.Tensor], offsets, embed):
        flat = torch.cat([raw[name].reshape(-1, width) for name, width in PARAMETERS], dim=1)
        order = curve_order(raw["positions"].detach(), offsets)
        return flat, order, torch.nn.functional.linear(flat[order].float(), embed.float()).to(self.embed.dtype)

    def _write(self, raw, flat, order, change):
        refined = flat.index_add(0, order, change.to(flat.dtype) * self.step)
        parts = torch.split(refined, [width for _, width in PARAMETERS], dim=1)
        return {**raw, **{name: part.reshape(raw[name].shape) for (name, _), part in zip(PARAMETERS, parts)}}

    def forward(self, raw: Dict[str, torch.Tensor], offsets: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """Refined copies of the parameters named in PARAMETERS; `offsets` (int32) where packed scenes begin.  Differentiable."""
        flat, order, update = self._read(raw, offsets, self.embed)
        stream = None
        for layer in range(self.layers):
            y, stream = add_rms_norm(update, self.norms[layer], stream)
            both = fp8_linear(y, self.enter[layer])
            h, _ = gated_scan(both[:, :self.width], both[:, self.width:], offsets=offsets, reverse=layer % 2 == 1)
            update = fp8_linear(h, self.leave[layer])
        y, _ = add_rms_norm(update, self.norms[-1], stream)
        return self._write(raw, flat, order, fp8_linear(y, self.head))

    @torch.no_grad()
    def infer(self, raw: Dict[str, torch.Tensor], offsets: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """`forward` without gradients, on the weights of the last `freeze()`."""
        if self._frozen is None:
            raise RuntimeError("call freeze() before infer()")
        f = self._frozen
        flat, order, update = self._read(raw, offsets, f["embed"])
        stream = None
        for layer in range(self.layers):
            q, stream = add_rms_norm_fp8(update, self.norms[layer], stream)
            both = fp8_matmul(q, f["enter"][layer], update.dtype)
            h, _ = gated_scan(both[:, :self.width], both[:, self.width:], offsets=offsets, reverse=layer % 2 == 1)
            update = fp8_matmul(h, f["leave"][layer])
        q, _ = add_rms_norm_fp8(update, self.norms[-1], stream)
        return self._write(raw, flat, order, fp8_matmul(q, f["head"], update.dtype))
