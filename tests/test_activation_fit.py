"""The gelu's polynomial, as the source has it, against the scaled complementary error function in 64 bits."""
import os
import re

import torch

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "approxtrain_amd", "csrc", "amsim_norm.hip")


def test_the_tail_s_polynomial():
    with open(SOURCE) as f:
        gelu = re.search(r"struct Gelu \{(.*?)\n\};", f.read(), re.S).group(1)
    slope = float(re.search(r"__builtin_fmaf\(([\d.]+)f, t, 1\.0f\)", gelu).group(1))
    first = re.search(r"float q = (-?[\d.e-]+)f;", gelu).group(1)
    coefficients = [float(first)] + [float(c) for c in re.findall(r"q = __builtin_fmaf\(q, w, (-?[\d.e-]+)f\);", gelu)]
    assert len(coefficients) == 9 and all(torch.tensor(c, dtype=torch.float64).float().double().item() == c for c in coefficients + [slope])
    t = torch.cat([torch.linspace(0, 1, 100001, dtype=torch.float64) ** 2, torch.linspace(1, 14.5, 200001, dtype=torch.float64)])
    w, q = t / (1 + slope * t), torch.zeros_like(t)
    for c in coefficients:
        q = q * w + c
    r = 0.5 * torch.special.erfcx(t / 2 ** 0.5)
    assert ((0.5 + w * q) / r - 1).abs().max() <= 2.1e-8
