"""Which quotients and tanh of mods may be computed to less than the last bit: those of a score that stay one."""
import pytest
import torch

from flaxattention_b200.modtrace import lower_mods


def quick(score, mask=None):
    """Names of the forms that kernels may replace, in the value of score_mod and in the mask."""
    source = lower_mods(score, mask).source
    body = source[source.index("float fa_score_mod("):]
    body = body[: body.index("fa_score_mod_grad")]
    rest = source[source.index("bool fa_mask_mod("):]
    assert "FA_QUOTIENT" not in rest and "FA_TANH" not in rest
    return [name for name in ("FA_QUOTIENT(", "FA_QUOTIENT_BY(", "FA_TANH(") if name in body], [name for name in (" / ", "tanhf(") if name in body]


@pytest.mark.parametrize("score,names", [
    (lambda s, b, h, q, kv: 30.0 * torch.tanh(s / 30.0), (["FA_QUOTIENT_BY(", "FA_TANH("], [])),
    (lambda s, b, h, q, kv: torch.tanh(s * 0.1) + torch.exp(s / (h + 1)), (["FA_QUOTIENT(", "FA_TANH("], [])),
    (lambda s, b, h, q, kv: torch.where(q >= kv, s / (h + 2), -s) * s, (["FA_QUOTIENT("], [])),
    (lambda s, b, h, q, kv: torch.maximum(s / (h + 2), s * s), (["FA_QUOTIENT("], [])),
    # nothing of the score in it
    (lambda s, b, h, q, kv: s * s + (q - kv) / 3.0 + torch.tanh(kv * 0.1), ([], [" / ", "tanhf("])),
    (lambda s, b, h, q, kv: s * s - (q - kv) / (h + 1), ([], [" / "])),
    # something is decided by it
    (lambda s, b, h, q, kv: torch.where(s / 3.0 > 1.0, s * s, s), ([], [" / "])),
    (lambda s, b, h, q, kv: torch.where(torch.tanh(s) > 0.5, s * s, s), ([], ["tanhf("])),
    (lambda s, b, h, q, kv: torch.floor(s / 3.0) * s, ([], [" / "])),
    (lambda s, b, h, q, kv: (s * s) // 3.0, ([], [" / "])),
    (lambda s, b, h, q, kv: s + (s / 3.0) % 2.0, ([], [" / "])),
    # both: a value that is used in two ways
    (lambda s, b, h, q, kv: (lambda x: torch.where(x > 1.0, x * x, x))(s / 3.0), ([], [" / "])),
    (lambda s, b, h, q, kv: (lambda x: torch.ceil(torch.exp(x)) + x)(s / (h + 1)), ([], [" / "])),
    # a divisor whose reciprocal is out of range
    (lambda s, b, h, q, kv: torch.tanh(s / 1e-35), (["FA_QUOTIENT(", "FA_TANH("], [])),
])
def test_what_stays_exact(score, names):
    assert quick(score, lambda b, h, q, kv: torch.floor(q / 7.0) == torch.tanh(kv / 7.0)) == names


def test_mods_without_such_forms_keep_their_text():
    assert "FA_QUOTIENT" not in lower_mods(lambda s, b, h, q, kv: s - (q - kv) / 3.0, lambda b, h, q, kv: q / 3 >= kv / 3).source
