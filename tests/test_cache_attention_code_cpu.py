"""The code of the kernels that attend over caches, in the built library, without a GPU."""
from tests.test_attention_code_cpu import kernels  # noqa: F401  (a fixture)


def test_no_load_is_flat(kernels):  # noqa: F811
    """A flat load counts as a load of LDS too, and both must then have arrived for either:
    a pointer that may lead to another address space than the caches' would make the
    kernels' loads ahead wait at their first use."""
    names = [name for name in kernels if "cache_kernel" in name]
    assert names
    for name in names:
        flat = [code for code in kernels[name] if code.startswith("flat_load")]
        assert not flat, (name, flat[:3])
