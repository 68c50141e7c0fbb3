"""The 8-bit mixture-of-experts example on the GPU: every run checks itself against a dense evaluation."""

import pytest

from nanoep_amd.examples import fp8_moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize(
    "arguments",
    [
        [],
        ["--tokens", "1", "--topk", "1", "--alignment", "1"],
        ["--tokens", "300", "--hidden", "512", "--intermediate", "208", "--experts", "3", "--topk", "2", "--alignment", "128"],
        ["--tokens", "64", "--hidden", "768", "--intermediate", "1040", "--experts", "40", "--topk", "8"],
        ["--train"],
        ["--train", "--tokens", "1", "--topk", "1"],
        ["--train", "--tokens", "500", "--hidden", "2816", "--experts", "60", "--topk", "6"],
    ],
)
def test_fp8_moe_example(device, arguments):
    print("fp8_moe", *arguments, flush=True)
    fp8_moe.run(fp8_moe.parse_args(arguments))
