"""What the operators' modules share."""


def check_probability(p):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be between 0 and 1, got {p}")
