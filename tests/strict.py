"""A comparison that a NaN or an infinity does not pass: |NaN - x| > tol is false."""


def strictly(close):
    """`close(got, want, ...)`, and every value of `got` finite whose `want` is."""
    def compare(got, want, *rest):
        lost = ~got.detach().cpu().isfinite() & want.detach().cpu().isfinite()
        assert not lost.any(), (rest[-1], int(lost.sum()), lost.nonzero()[:4].tolist())
        close(got, want, *rest)
    return compare
