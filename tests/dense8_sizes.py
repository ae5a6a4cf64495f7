"""Layers that take a certain form of the 8-bit product (test infrastructure): algebra, filter layout, type, samples, features in and out."""
import ctypes

from phoenix_core_b200 import _lib
from phoenix_core_b200.ops import _ALGEBRAS
from phoenix_core_b200.descriptors import Algebra

# Tiles of 256 x 256 on pairs of SMs in all three products: rows of results on 16 bytes and not, ragged in every direction, up to three tiles for a pair, every algebra, layout and type
PAIRS = [("real", "io", "f16", 4103, 904, 2904), ("real", "oi", "bf16", 4103, 904, 2904), ("real", "oi", "f32", 4103, 904, 2904), ("real", "oi", "f16", 2905, 901, 4103),
         ("real", "io", "f32", 2905, 901, 4103), ("complex", "io", "bf16", 701, 1703, 2101), ("complex", "oi", "f16", 2101, 1703, 701), ("quaternion", "io", "f16", 709, 900, 904),
         ("quaternion", "oi", "bf16", 701, 905, 901), ("quaternion", "oi", "f32", 709, 900, 904), ("ga300", "io", "bf16", 503, 701, 707), ("ga300", "oi", "f16", 900, 300, 901)]
# The same beside an SM margin (each of whose SMs counts as a pair: beside larger ones single SMs are the faster)
MARGINS = [(5, ("real", "io", "f16", 4103, 904, 2904)), (2, ("quaternion", "oi", "bf16", 901, 903, 907)), (5, ("ga300", "oi", "f16", 900, 300, 901))]
# Up to four tokens, quantised by the product itself: several tiles to a CTA, several groups of blocks to a reduction, every algebra
FEW_TOKENS = [("real", "io", "bf16", 1, 4096, 20000), ("real", "oi", "f16", 4, 1100, 300), ("real", "io", "f32", 4, 513, 19100), ("real", "oi", "bf16", 3, 515, 19103),
              ("complex", "io", "f16", 2, 1100, 200), ("complex", "oi", "f32", 4, 700, 10001), ("quaternion", "oi", "bf16", 4, 300, 200), ("quaternion", "io", "f16", 3, 1025, 200),
              ("quaternion", "io", "f32", 1, 600, 5003), ("ga300", "io", "bf16", 2, 530, 200), ("ga300", "oi", "f16", 4, 1100, 200), ("ga300", "io", "f32", 3, 77, 2600)]
# Both gradients in one launch
BOTH = [("quaternion", "io", "f16", 777, 500, 1001), ("real", "oi", "bf16", 1500, 1030, 1100), ("ga300", "io", "f32", 130, 200, 140)]


def sizes_of(case):
    algebra, layout, dtype, n, i, o = case
    d = _lib.DenseDesc()
    d.dtype = {"f32": _lib.PCB_F32, "f16": _lib.PCB_F16, "bf16": _lib.PCB_BF16}[dtype]
    d.algebra = _ALGEBRAS[{"real": Algebra.REAL, "complex": Algebra.COMPLEX, "quaternion": Algebra.QUATERNION, "ga300": Algebra.GA_300}[algebra]]
    d.batch, d.in_features, d.out_features, d.filter_oi, d.require_input_grad = n, i, o, int(layout == "oi"), 1
    return d


def form(case, product):
    """1: tokens quantised by the product, 2: the filter as the first operand, 3: tiles, 4: pairs, 5: both gradients at once (pcb_dense8_form)."""
    return _lib.lib().pcb_qdense8_form_for(ctypes.byref(sizes_of(case)), product)
