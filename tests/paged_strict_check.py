"""The bounds of ``paged_scores_reference``, under which a NaN is a difference
like any other."""


def check(got, want, ordinary=True):
    """``paged_scores_reference.check``, which compares with ``>``: a NaN in the
    output alone, or in a bound, passes there.  Here a NaN is due exactly where the
    restatement has one, and everything else has to be shown to be near."""
    out, tol, l2 = want
    got = got.double()
    nan = got.isnan()
    if bool((nan != out.isnan()).any()):
        return f"{int((nan & ~out.isnan()).sum())} elements are NaN and {int((~nan & out.isnan()).sum())} are not, wrongly"
    near = ((got - out).abs() <= tol) | (got == out) | nan
    if not bool(near.all()):
        i = int((~near).flatten().nonzero()[0])
        return f"{int((~near).sum())} elements off, one {(got - out).flatten()[i]:.3g} of {tol.flatten()[i]:.3g}"
    if ordinary:
        rows = out.isfinite().all(-1)
        near = ((got - out).norm(dim=-1) <= l2) | ~rows
        if not bool(near.all()):
            return f"{int((~near).sum())} rows off in L2"
    return ""
