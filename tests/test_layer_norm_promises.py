"""Promises of the layer norm entry points that can be read from their source.  No GPU."""
import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parent.parent / "monet_amd" / "csrc" / "layernorm.hip"


def _parameters(kernel):
    """{name: declaration} of a kernel's parameters."""
    text = re.search(r"void[^;{]*?\b%s\((.*?)\) \{" % kernel, SOURCE.read_text(), re.S).group(1)
    return {re.search(r"(\w+)$", p.strip()).group(1): p for p in text.split(",")}


def test_in_place_calls_are_defined():
    """`y may alias x` and `dx may alias grad`: neither side may be declared free of aliases."""
    for kernel, pair in (("ln_fwd_kernel", "xy"), ("ln_fwd_long_kernel", "xy"),
                         ("ln_bwd_kernel", ("g", "dx")), ("ln_bwd_long_kernel", ("g", "dx"))):
        decl = _parameters(kernel)
        for name in pair:
            assert "*" in decl[name] and "restrict" not in decl[name], (kernel, decl[name])
