"""The status word, in which the kernels OR their errors (include/chia_paged.h), by its names."""

import re

import pytest

import chia_proj_b200 as cp


@pytest.mark.parametrize("code,names", [(8, {"BAD_INDEX"}), (16, {"NO_PAGES"}), (24, {"BAD_INDEX", "NO_PAGES"}),
                                        (13, {"DEVICE_TIMEOUT", "BAD_INDEX"}), (12, {"LAUNCH", "BAD_INDEX"}),
                                        (21, {"DEVICE_TIMEOUT", "NO_PAGES"}),
                                        (29, {"DEVICE_TIMEOUT", "BAD_INDEX", "NO_PAGES"}), (5, {"DEVICE_TIMEOUT"})])
def test_every_error_in_a_status_word_is_named(code, names):
    e = cp.ChiaError(code, "x")
    assert e.code == code and set(re.findall(r"CHIA_ERR_(\w+)", str(e))) == names


@pytest.mark.parametrize("code", [7, 32, 40, 15])
def test_unknown_bits_stay_a_number(code):
    assert str(cp.ChiaError(code)) == f"status {code}"
