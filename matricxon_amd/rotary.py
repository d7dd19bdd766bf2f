"""Rotary positions of q and k on the device, in one launch (`mxa_rope`): the step between the q | k | v projections
(`matricxon_amd.fused_ops.project_shared`) and attention.

Pair i of the rotary part (d = `rotary_dim` values) of a head turns by the angle p * f_i at position p, the pair being
elements (i, i + d / 2), or (2 i, 2 i + 1) when `interleaved` (GGUF's order of attn_q and attn_k rows before the
loader's reordering). f_i = base^(-2 i / d), scaled for contexts longer than the model was trained on:

* `linear`: f_i / factor.
* `ntk`: base * factor^(d / (d - 2)) in place of base.
* `yarn`: pairs that turn at least `beta_fast` times within `original_context` keep f_i, those that turn at most
  `beta_slow` times take f_i / factor, with a ramp over i between them; the turned values are multiplied by
  `attention_factor` (0.1 ln(factor) + 1 unless given).
* `llama3`: pairs that turn at least `high_freq_factor` times within `original_context` keep f_i, those that turn at
  most `low_freq_factor` times take f_i / factor, linearly between them in the number of turns.

`freq_factors` (GGUF's rope_freqs.weight) divides the f_i besides. The table is made in float64 on the host, and the
kernel reduces the angles in float64, so positions of millions lose nothing.
"""

import math

import torch

from matricxon_amd.gemm import HipGemm

# a scaling's keys and their defaults (None: has to be given)
_SCALINGS = {
    "linear": {"factor": None},
    "ntk": {"factor": None},
    "yarn": {"factor": None, "original_context": None, "beta_fast": 32.0, "beta_slow": 1.0, "attention_factor": 0.0},
    "llama3": {"factor": None, "original_context": None, "low_freq_factor": 1.0, "high_freq_factor": 4.0},
}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                       freq_factors: torch.Tensor | None = None) -> tuple[torch.Tensor, float]:
    """(f (rotary_dim / 2) float64 on the CPU, the factor on the turned values)."""
    d = int(rotary_dim)
    if d < 2 or d % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 0:
        raise ValueError(f"base must be positive, got {base}")
    kind, opt = None, {}
    if scaling is not None:
        kind = scaling.get("type")
        if kind not in _SCALINGS:
            raise ValueError(f"scaling type must be one of {sorted(_SCALINGS)}, got {kind!r}")
        opt = dict(_SCALINGS[kind])
        for key, value in scaling.items():
            if key == "type":
                continue
            if key not in opt and key != "original_context":  # a context may be named beside any scaling
                raise ValueError(f"{kind} scaling takes {sorted(opt)}, got {key!r}")
            opt[key] = value
        missing = [key for key, value in opt.items() if value is None]
        if missing:
            raise ValueError(f"{kind} scaling needs {missing}")
        if not opt["factor"] > 0 or not opt.get("original_context", 1) > 0:
            raise ValueError("factor and original_context must be positive")
        if kind == "ntk" and d == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        if kind == "llama3" and not 0 < opt["low_freq_factor"] < opt["high_freq_factor"]:
            raise ValueError("llama3 scaling needs 0 < low_freq_factor < high_freq_factor")
        if kind == "yarn" and (base == 1 or not 0 < opt["beta_slow"] < opt["beta_fast"]):
            raise ValueError("yarn scaling needs 0 < beta_slow < beta_fast and a base other than 1")
    i = torch.arange(d // 2, dtype=torch.float64, device="cpu")
    if kind == "ntk":
        base = base * opt["factor"] ** (d / (d - 2))
    f = float(base) ** (-2 * i / d)
    mscale = 1.0
    if kind == "linear":
        f = f / opt["factor"]
    elif kind == "yarn":
        def place(turns: float) -> float:  # the (real) pair index that turns so often within the context
            return d * math.log(opt["original_context"] / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(place(opt["beta_fast"])), 0), min(math.ceil(place(opt["beta_slow"])), d - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / opt["factor"] * ramp + f * (1 - ramp)
        mscale = float(opt["attention_factor"]) or 0.1 * math.log(opt["factor"]) + 1
    elif kind == "llama3":
        low, high = opt["low_freq_factor"], opt["high_freq_factor"]
        kept = ((opt["original_context"] * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = kept * f + (1 - kept) * f / opt["factor"]
    if freq_factors is not None:
        ff = freq_factors.detach().to("cpu", torch.float64).reshape(-1)
        if ff.shape != f.shape:
            raise ValueError(f"freq_factors must have {d // 2} values, got {ff.numel()}")
        f = f / ff
    return f, mscale


class HipRotary:
    """`rot = HipRotary(head_dim, ...)`, then `q, k = rot(q, k, positions)`."""

    def __init__(self, head_dim: int, *, rotary_dim: int | None = None, base: float = 10000.0,
                 interleaved: bool = False, scaling: dict | None = None, freq_factors: torch.Tensor | None = None,
                 device: torch.device | str = "cuda") -> None:
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if not 2 <= self.rotary_dim <= self.head_dim <= HipGemm.ROPE_MAX_DIM or self.head_dim % 2:
            raise ValueError(f"head_dim must be even, at most {HipGemm.ROPE_MAX_DIM} and at least rotary_dim, got "
                             f"{head_dim} and {rotary_dim}")
        self.interleaved = bool(interleaved)
        self.frequencies, self.scale = rotary_frequencies(self.rotary_dim, base, scaling, freq_factors)
        self._gemm = HipGemm.get()
        self._turns: dict[torch.device, torch.Tensor] = {}
        device = torch.device(device)
        if device.type == "cuda" and torch.cuda.is_available():
            self._table(torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index))

    def _table(self, device: torch.device) -> torch.Tensor:
        """Turns per position of each pair, on `device` (laid out at the first use of a device)."""
        table = self._turns.get(device)
        if table is None:
            if device.type != "cuda":
                raise ValueError(f"q and k must be tensors on a HIP device, got {device}")
            table = self._turns[device] = (self.frequencies / (2 * math.pi)).to(device)
        return table

    def __call__(self, q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor
                 ) -> tuple[torch.Tensor, torch.Tensor | None]:
        """q (T, heads, head_dim) or (B, T, heads, head_dim) and k likewise, of its own number of heads (or None), of
        any strides with adjacent values in a head, as the columns of a q | k | v buffer; positions int32 or int64
        (T,), or (B, T) for a batch. Returns new contiguous tensors of those shapes and that dtype, float32 or
        bfloat16. Any position, negative ones turning back."""
        return self._gemm._rope(q, k, positions, self._table(q.device), self.rotary_dim, self.interleaved, self.scale)

    def shift(self, k: torch.Tensor, delta: torch.Tensor) -> torch.Tensor:
        """Keys that were turned for their positions, turned on by `delta` positions (a tensor as `positions`;
        negative: back), as a cache needs whose start moves. The scaling's factor on the values is already in them."""
        return self._gemm._rope(k, None, delta, self._table(k.device), self.rotary_dim, self.interleaved, 1.0)[0]
