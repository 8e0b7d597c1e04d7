from lqg_amd.belief import kf, ssm  # noqa: F401
