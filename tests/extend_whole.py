"""The error of a chunk attention's result as a whole, whatever its size."""
import shared_cache_ref as R


def check_whole(got, want, dtype):
    """At scores of order one: four roundings of 0.42 u each make 0.84 u in the root mean square (see
    ``shared_cache_ref.check_extend``); 2 u leaves room for what 128 values scatter, and a lost or doubled share of the keys is
    tens of u at least."""
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel <= 2 * R.unit(dtype), f"relative error {rel:.3g}, allowed {2 * R.unit(dtype):.3g}"
