"""Decoder architectures of the benchmark configurations.

Llama (SmolLM2) and Qwen2 decoder layers as mlx-lm builds them: RMSNorm,
q/k/v projections (Qwen2 with bias), rotary embedding, by default over the full
head dimension in the non-interleaved ("rotate half") form, its frequencies
scaled for long contexts where the architecture says so, causal grouped-query
attention with scale ``head_dim ** -0.5``, output projection, residual,
RMSNorm, SwiGLU MLP, residual.  The reference runs the mlx-lm layer inside
``block_output`` (mround/pipeline/blocks.py:578-606); its math is restated in
:mod:`mround_b200.pipeline.block`.
"""

from __future__ import annotations

import dataclasses

__all__ = ["ARCHITECTURES", "Arch", "RopeScaling", "get_arch"]

ROPE_SCALINGS = ("linear", "llama3", "yarn")


@dataclasses.dataclass(frozen=True, slots=True)
class RopeScaling:
    """How rotary frequencies are scaled for contexts longer than trained on.

    ``kind`` "linear": every frequency divided by ``factor``.  "llama3":
    wavelengths above ``original_max_position / low_freq_factor`` divided by
    ``factor``, those below ``original_max_position / high_freq_factor`` kept,
    a ramp in between.  "yarn": frequencies that turn fewer than ``beta_slow``
    times in ``original_max_position`` positions divided, more than
    ``beta_fast`` kept, a ramp over the columns in between, and cosines and
    sines multiplied by ``attention_factor`` (0.1 ln(factor) + 1 when None)."""

    kind: str
    factor: float
    original_max_position: int | None = None
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self) -> None:
        from mround_b200.exceptions import ArchitectureError

        if self.kind not in ROPE_SCALINGS:
            raise ArchitectureError(f"rope scaling {self.kind!r} is not one of "
                                    f"{', '.join(ROPE_SCALINGS)}")
        if not self.factor >= 1.0:
            raise ArchitectureError(f"rope scaling factor must be at least 1, got {self.factor}")
        if self.kind != "linear" and not (self.original_max_position or 0) > 0:
            raise ArchitectureError(f"{self.kind} rope scaling needs the original number of "
                                    "positions")
        if self.kind == "llama3" and not 0 < self.low_freq_factor < self.high_freq_factor:
            raise ArchitectureError("llama3 rope scaling needs 0 < low_freq_factor < "
                                    "high_freq_factor")
        if self.kind == "yarn" and not 0 < self.beta_slow < self.beta_fast:
            raise ArchitectureError("yarn rope scaling needs 0 < beta_slow < beta_fast")


@dataclasses.dataclass(frozen=True, slots=True)
class Arch:
    name: str
    family: str  # "llama" or "qwen2"
    hidden: int
    layers: int
    heads: int
    kv_heads: int
    head_dim: int
    intermediate: int
    vocab: int
    rms_eps: float
    rope_theta: float
    qkv_bias: bool
    tied: bool
    rope_scaling: RopeScaling | None = None
    rope_interleaved: bool = False  # pairs (2j, 2j + 1) instead of halves
    rotary_dim: int | None = None  # rotated columns of a head; all of them when None

    def __post_init__(self) -> None:
        r = self.rotary_dim
        if r is not None and (r % 2 or not 2 <= r <= self.head_dim):
            from mround_b200.exceptions import ArchitectureError

            raise ArchitectureError(f"rotary_dim must be even and at most the head dimension "
                                    f"{self.head_dim}, got {r}")

    @property
    def rope_layout(self) -> str:
        return "interleaved" if self.rope_interleaved else "half"

    @property
    def q_dim(self) -> int:
        return self.heads * self.head_dim

    @property
    def kv_dim(self) -> int:
        return self.kv_heads * self.head_dim

    def linear_shapes(self) -> dict[str, tuple[int, int]]:
        """(out_features, in_features) of each block linear, by mlx-lm module path."""
        h, i = self.hidden, self.intermediate
        return {
            "self_attn.q_proj": (self.q_dim, h),
            "self_attn.k_proj": (self.kv_dim, h),
            "self_attn.v_proj": (self.kv_dim, h),
            "self_attn.o_proj": (h, self.q_dim),
            "mlp.gate_proj": (i, h),
            "mlp.up_proj": (i, h),
            "mlp.down_proj": (h, i),
        }

    def block_weights(self) -> int:
        """Weights in the linears of one block."""
        return sum(o * i for o, i in self.linear_shapes().values())


ARCHITECTURES: dict[str, Arch] = {
    "smollm2-135m": Arch("smollm2-135m", "llama", 576, 30, 9, 3, 64, 1536, 49152, 1e-5, 1e5,
                         False, True),
    "qwen2.5-0.5b": Arch("qwen2.5-0.5b", "qwen2", 896, 24, 14, 2, 64, 4864, 151936, 1e-6, 1e6,
                         True, True),
    "qwen2.5-3b": Arch("qwen2.5-3b", "qwen2", 2048, 36, 16, 2, 128, 11008, 151936, 1e-6, 1e6,
                       True, True),
    "qwen2.5-7b": Arch("qwen2.5-7b", "qwen2", 3584, 28, 28, 4, 128, 18944, 152064, 1e-6, 1e6,
                       True, False),
    # test-sized architectures (not benchmark configurations)
    "tiny-llama": Arch("tiny-llama", "llama", 128, 2, 4, 2, 32, 256, 512, 1e-5, 1e4, False, True),
    "tiny-qwen2": Arch("tiny-qwen2", "qwen2", 128, 2, 4, 2, 32, 384, 512, 1e-6, 1e6, True, True),
}


def get_arch(name: str) -> Arch:
    try:
        return ARCHITECTURES[name]
    except KeyError as exc:
        from mround_b200.exceptions import ArchitectureError

        raise ArchitectureError(
            f"unknown architecture {name!r}; known: {', '.join(sorted(ARCHITECTURES))}"
        ) from exc
