"""Small programs that use the package as a user would."""
