"""Numbers for the paged cache's tests at their edges."""
from decimal import Decimal, localcontext


def pi_of(digits):
    """By Gauss and Legendre's means."""
    with localcontext() as c:
        c.prec = digits + 10
        a, b, t, p = Decimal(1), Decimal(2).sqrt() / 2, Decimal(1) / 4, 1
        while abs(a - b) > Decimal(10) ** -(digits + 5):
            a, b, t, p = (a + b) / 2, (a * b).sqrt(), t - p * ((a - b) / 2) ** 2, 2 * p
        return (a + b) ** 2 / (4 * t)
